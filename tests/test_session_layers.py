"""The layers of chatokf_amd/session.py as their calls run behind each other: a chat whose queries and
keys have norms and positions, through eviction; and the gated delta rule's layer over packed chats, from
its projections' values to its output's input, in 64 bits."""
import numpy as np
import pytest

import attn_oracle as ao
import layer_oracle as lo

torch = pytest.importorskip("torch")
import chatokf_amd as ok  # noqa: E402
from test_attn import U, dev, gpu, host  # noqa: E402


@gpu
@pytest.mark.parametrize("pairs,rot,norms", [(False, 64, True), (True, 32, True), (False, 64, False), (False, 0, True)])
def test_chat_with_positions(enc, pairs, rot, norms):
    """Every token's queries and keys stand at its own position, also those behind an eviction; kept keys stay as they were."""
    from chatokf_amd.session import Chat, Layer
    K, H, KV, D = 256, 4, 2, 64
    rng = np.random.default_rng(11)
    qn, kn = (1 + 0.3 * rng.standard_normal((2, D))).astype(np.float32) if norms else (None, None)
    plain = Layer(enc, K, H, KV, D)
    layer = Layer(enc, K, H, KV, D, rope=ok.Rope(rot, pairs=pairs) if rot else None, q_norm=dev(qn) if norms else None,
                  k_norm=dev(kn) if norms else None, eps=1e-5)
    chat = Chat(layer, limit=200, keep=96, sink=2, recent=16)
    f, mag = lo.freqs(rot, 1e4)
    seen, out = {}, layer.output
    layer.output = lambda a: out(seen.setdefault("a", a))
    keys = np.zeros((0, KV, D))  # what the cache should hold, before its 8 bits
    total = 0
    for turn, (call, n) in enumerate(((chat.prompt, 90), (chat.prompt, 70), (chat.step, 1), (chat.step, 3), (chat.prompt, 60), (chat.step, 1), (chat.step, 1))):
        x = torch.from_numpy(rng.standard_normal((n, K)).astype(np.float32)).cuda()
        seen.clear()
        pos, first = np.arange(total, total + n), chat.n == 0
        call(x)
        total += n
        assert chat.pos == total
        raw, mine = plain.project(x), layer.project(x, int(pos[0]))
        held = chat.values()
        enc.sync()
        q, k, v = (host(t) for t in mine)
        for y, r, w in ((q, raw[0], qn), (k, raw[1], kn)):
            ref, size = lo.norm_rope(host(r), pos, w, 1e-5, rot, pairs, f, mag)
            # (24 u as in test_rope.py; these positions' angles in 64 bits add less than one)
            assert np.abs(y - ref).max() <= 25 * U * size.max()
        assert np.array_equal(host(raw[2]), v)
        if chat.n < total and len(keys) + n > 200:
            kept = host(chat.kept).astype(int)
            keys = np.stack([keys[kept[h], h] for h in range(KV)], 1)
        keys = np.concatenate([keys, k])
        ck, cv = host(held[0]), host(held[1])
        assert ck.shape == keys.shape
        # 8 bits a value: each call, and the eviction, may round a page's codes anew, by half a step of its scale,
        # which is at most 1/127 of the head's largest value
        assert (np.abs(ck - keys) <= np.abs(keys).max((0, 2))[:, None] / 127 * (turn + 2) / 2).all()
        if first:
            ck, cv = k, v
        a, at = host(seen["a"]), np.arange(chat.n - n, chat.n)
        big = np.sqrt((q ** 2).sum(-1)).max() * np.sqrt((ck ** 2).sum(-1)).max() * D ** -0.5
        bound = (2 * (D + 4) * big + 2 * chat.n + 16) * 2.0 ** -24 * np.abs(cv).max()  # (as in test_attn.py)
        for h in range(H):
            ref, _ = ao.attend(q[:, h], ck[:, h // 2], cv[:, h // 2], at, 0, D ** -0.5)
            assert np.abs(a[:, h] - ref).max() <= bound
    assert total == 226 and chat.n == 96 + 62


class Delta64:
    """The layer from its projections' values to its output projection's input, in 64 bits, with what a
    result may be off by (u = 2^-24): the convolution (W + 4) u of its terms' absolute values (the activation's slope is at
    most 1.1); lengths (k_dim / 2 + 8) u and the same relative error as their rows, twice; decays 4 u (|g| e^g < 1/2, g within 8 u), the
    shares of new values 4 u; a token of the rule as in test_delta.py with those on top, each at most M, a column's or value's
    length, four times its keys' error (and each token's decay is that of the errors before it); an output's norm (v_dim / 2 + 8) u of itself, 1 + sqrt(v_dim) of its input's error over its
    root mean square; the gate 8 u."""

    def __init__(self, layer, chats):
        self.l, self.conv, self.state = layer, [np.zeros((layer.width - 1, layer.channels))] * chats, \
            [np.zeros((layer.v_heads, layer.k_dim, layer.v_dim))] * chats
        self.off = [np.zeros(layer.v_heads)] * chats  # of the states, each head's

    def run(self, i, u, z, ab, keep):
        """Chat i's rows: the rows and their bounds."""
        L, m = self.l, len(u)
        KH, VH, DK, DV, nk = L.k_heads, L.v_heads, L.k_dim, L.v_dim, L.keys
        y, size, conv = lo.conv(u, host(L.conv), None, self.conv[i], True)
        ey = (L.width + 4) * U * size + 4 * U * np.abs(y)
        q, k, v = (y[:, a:b].reshape(m, h, -1) for a, b, h in ((0, nk, KH), (nk, 2 * nk, KH), (2 * nk, L.channels, VH)))
        length = [np.sqrt((x ** 2).sum(-1, keepdims=True) + L.eps) for x in (q, k)]
        ek = max(2 * np.sqrt((e.reshape(m, KH, DK) ** 2).sum(-1) / n[..., 0] ** 2).max() for e, n in
                 zip((ey[:, :nk], ey[:, nk:2 * nk]), length)) + (DK / 2 + 8) * U
        g = -host(L.decay) * np.logaddexp(0, ab[:, :VH])
        beta = 1 / (1 + np.exp(-ab[:, VH:]))
        o, S = lo.delta(q / length[0], k / length[1], v, g, beta, self.state[i], DK ** -0.5)
        M = np.sqrt((self.state[i] ** 2).sum(1)).max(-1) + 2 * np.abs(v).max((0, 2))
        s, eo = self.off[i], np.zeros((m, VH, 1))
        for t in range(m):  # (a token's decay is its error's)
            s = s * np.exp(g[t]) + ((DK + 2 * 64 + 8 + 12) * U + 4 * ek) * M + ey[:, 2 * nk:].max()
            eo[t, :, 0] = DK ** -0.5 * (s + (DK * U + 2 * ek) * M)
        if keep:
            self.conv[i], self.state[i], self.off[i] = conv, S, s
        rms = np.sqrt((o ** 2).mean(-1, keepdims=True) + L.eps)
        n = o / rms
        en = (1 + np.sqrt(DV)) * eo / rms + (DV / 2 + 8) * U * np.abs(n)
        gate = (z / (1 + np.exp(-z))).reshape(m, VH, DV)
        return (gate * n).reshape(m, -1), (np.abs(gate) * en + 8 * U * np.abs(gate * n)).reshape(m, -1)


@gpu
@pytest.mark.parametrize("KH,VH,DK,DV,width", [(2, 4, 64, 64, 4), (1, 2, 80, 48, 2), (2, 2, 32, 128, 8)])
def test_delta_chats(enc, KH, VH, DK, DV, width):
    from chatokf_amd.session import DeltaChats, DeltaLayer
    K = 256
    layer = DeltaLayer(enc, K, KH, VH, DK, DV, width)
    chats, ref = DeltaChats(layer, 3), Delta64(layer, 3)
    rng = np.random.default_rng(7)
    gemm, seen, share = enc.gemm, [], []

    def watch(w, x, y, n):
        gemm(w, x, y, n)
        seen.append((w, x if w is layer.o else y))
    enc.gemm = watch
    try:
        for call, lens, keep in ((chats.prompt, [40, 1, 33], True), (chats.prompt, [0, 35, 2], True), (chats.step, [1, 1, 1], True),
                                 (chats.verify, [4, 0, 2], False), (chats.step, [2, 0, 1], True), (chats.prompt, [1, 50, 0], True),
                                 (chats.step, [1, 1, 1], True)):
            x = torch.from_numpy(rng.standard_normal((sum(lens), K)).astype(np.float32)).cuda()
            seen.clear()
            before = chats.state.clone(), chats.conv.clone()
            out = call(x, lens)
            enc.sync()
            assert out.shape == (sum(lens), K) and torch.isfinite(out).all()
            (_, u), (_, z), (_, ab), (_, got) = [(w, host(t)) for w, t in seen]
            at = 0
            # (the gate is written over z, and what the projection takes is that)
            z = host(projected(enc, gemm, layer.z, x))
            for i, m in enumerate(lens):
                if m:
                    y, b = ref.run(i, u[at:at + m], z[at:at + m], ab[at:at + m], keep)
                    assert (np.abs(got[at:at + m] - y) <= b).all(), (lens, i)
                    share.append(np.median(b) / np.sqrt((y ** 2).mean()))
                same = torch.equal(before[0][i], chats.state[i]) and torch.equal(before[1][i], chats.conv[i])
                assert same == (not keep or m == 0)
                assert (np.abs(host(chats.state[i]) - ref.state[i]).max((1, 2)) <= ref.off[i]).all()
                at += m
    finally:
        del enc.gemm
    assert np.median(share) < 0.25  # (of the outputs: the bounds see something)


def projected(enc, gemm, w, x):
    y = torch.empty((x.shape[0], w.M), device="cuda")
    gemm(w, x, y, x.shape[0])
    enc.sync()
    return y


def test_delta_rows_that_do_not_fit():
    from chatokf_amd.session import DeltaChats
    chats = DeltaChats.__new__(DeltaChats)
    chats.layer, chats.chats = None, 2
    for lens, n in (([3], 3), ([1, 1, 1], 3), ([2, 2], 3), ([4, -1], 3), ([0, 0], 0), (None, 0)):
        with pytest.raises(ValueError):
            chats.prompt(torch.zeros(n, 64), lens)
