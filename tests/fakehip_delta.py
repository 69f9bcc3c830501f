"""fakehip.py's steps with the gated delta rule's calls beside them: run(fake, steps)."""
import json
import os
import subprocess
import sys

import fakehip


def run(fake, steps, **env):
    r = subprocess.run([sys.executable, os.path.abspath(__file__), fake], input=json.dumps(steps), text=True,
                       capture_output=True, env=dict(os.environ, **env), timeout=120)
    assert r.returncode == 0, r.stderr
    return json.loads(r.stdout.splitlines()[-1])


class Child(fakehip._Child):
    def delta(self, form, t, n, seqs, k_heads, v_heads, k_dim, v_dim):
        call = self.enc.delta_step if form == "step" else self.enc.delta_prompt
        P = self.P
        call(P, P, P, P, P, P << 32, P, seqs, n, k_heads, v_heads, k_dim, v_dim, type=self.ok.BY_NAME[t])

    def conv(self, t, n, seqs, channels, width):
        P = self.P
        self.enc.conv(P, P, P << 32, P, seqs, n, channels, width, type=self.ok.BY_NAME[t])

    def delta_reserve(self, t, n, seqs, k_heads, v_heads, k_dim, v_dim):
        self.enc.delta_reserve(n, seqs, k_heads, v_heads, k_dim, v_dim, self.ok.BY_NAME[t])

    def attn_reserve(self, *args):
        self.enc.attn_reserve(*args)


if __name__ == "__main__":
    steps = json.load(sys.stdin)
    child = Child(sys.argv[1])
    print(json.dumps([child.step(*s) for s in steps]))
