"""fakehip.py's steps with the attention calls beside them: run(fake, steps)."""
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
    def decode(self, seqs, stride, heads, kv_heads, dim, tokens, weights, window=0, over=False):
        cache = self.ok.KVCache(self.P, self.P, self.P, self.P, 100, kv_heads, dim)
        w = self.P if weights else None
        o = self.P if over else self.P << 32  # (over the queries, or far from them)
        self.enc.attn_decode(cache, self.ok.KVSeqs(self.P, self.P, seqs, stride), self.P, o, tokens, heads, 1.0, window=window,
                             w_in=w, w_out=w, w_stride=64 * stride)

    def attn_reserve(self, seqs, stride, heads, kv_heads, dim, tokens, weights):
        self.enc.attn_reserve(seqs, stride, heads, kv_heads, dim, tokens, bool(weights))

    def prompt(self, t, seqs, n_q, n_k, heads, kv_heads, dim, window=0):
        self.enc.attn_prompt(self.P, self.P, self.P, self.P, self.P, self.P, seqs, n_q, n_k, heads, kv_heads, dim,
                             type=self.ok.BY_NAME[t], window=window)


if __name__ == "__main__":
    steps = json.load(sys.stdin)
    child = Child(sys.argv[1])
    print(json.dumps([child.step(*s) for s in steps]))
