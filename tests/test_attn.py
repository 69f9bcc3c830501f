"""Attention over prompts and over the paged 8-bit KV cache, and the cache's own
operators, against the 64-bit oracle (attn_oracle.py).

Tolerances, from the roundings: u = 2^-24.  A score, sum of D products in fp32,
is off by at most (D + 4) u times the sum of their absolute values (call the
largest B, times the scale), so a softmax weight by twice that in relative terms
plus the sum's and the exponential's few u; an output by that times max |v|.
The decode kernel's 23-bit queries and weights are off by 2^-23 of the largest
of a row each: (D + 4) and the number of keys n cover them with the factors
below.  f16 / bf16: half a step for each weight and for the output.  Codes,
scales, kept tokens and values read back as fp32 are equal, bit for bit."""
import ctypes
import sys

import numpy as np
import pytest

import attn_oracle as ao

torch = pytest.importorskip("torch")
import chatokf_amd as ok  # noqa: E402

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
gpu = pytest.mark.gpu


def dev(a, t=None):
    x = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return x if t is None else x.to(t)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def host(t):
    torch.cuda.synchronize()
    return t.double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def starts(lens):
    return [0, *np.cumsum(lens).tolist()]


def tol(q, k, v, scale, n, D, t="f32"):
    fin = lambda x: x[np.isfinite(x)]  # noqa: E731
    b = np.sqrt((np.where(np.isfinite(q), q, 0) ** 2).sum(-1)).max() * np.sqrt((np.where(np.isfinite(k), k, 0) ** 2).sum(-1)).max() * scale
    rel = 2 * (D + 4) * U * b + (2 * n + 16) * U
    if t != "f32":
        rel += torch.finfo(TYPES[t]).eps  # a weight's and the output's half step
    return rel * np.abs(fin(v)).max() + 1e-30


# ------------------------------------------------------------------ refusals
FAKE = 0x10000


@pytest.fixture()
def detached():
    e = ok.Enc(-1)
    yield e
    e.close()


def fails(call, status):
    with pytest.raises(ok.OkfError) as e:
        call()
    assert e.value.status == status


def attn(e, **over):
    a = dict(q=FAKE, k=FAKE, v=FAKE, out=FAKE, q_start=FAKE, k_start=FAKE, seqs=1, n_q=4, n_k=4, heads=8, kv_heads=2,
             dim=64)
    e.attn_prompt(**{**a, **over})


@pytest.mark.parametrize("over,status", [
    ({}, ok.OKF_E_NODEV), ({"type": ok.F16}, ok.OKF_E_NODEV), ({"window": 5}, ok.OKF_E_NODEV),
    ({"q": 0}, ok.OKF_E_ARG), ({"k_start": 0}, ok.OKF_E_ARG), ({"type": ok.Q8_0}, ok.OKF_E_TYPE),
    ({"heads": 7}, ok.OKF_E_SHAPE), ({"kv_heads": 0}, ok.OKF_E_SHAPE), ({"dim": 8}, ok.OKF_E_SHAPE),
    ({"dim": 72}, ok.OKF_E_SHAPE), ({"dim": 272}, ok.OKF_E_SHAPE), ({"n_q": 0}, ok.OKF_E_SHAPE),
    ({"seqs": 0}, ok.OKF_E_SHAPE), ({"v": FAKE + 8}, ok.OKF_E_SHAPE), ({"q_start": FAKE + 2}, ok.OKF_E_SHAPE),
    ({"strides": (32, 0, 0, 0)}, ok.OKF_E_SHAPE), ({"strides": (513, 0, 0, 0)}, ok.OKF_E_SHAPE),
    ({"strides": (516, 0, 0, 0)}, ok.OKF_E_NODEV), ({"strides": (516, 0, 0, 0), "type": ok.BF16}, ok.OKF_E_SHAPE),
    ({"head_strides": (0, 63, 0, 0)}, ok.OKF_E_SHAPE)])
def test_prompt_refusals(detached, over, status):
    fails(lambda: attn(detached, **over), status)


def fake_cache(**over):
    return ok.KVCache(**{**dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, pages=4, heads=2, dim=64), **over})


def fake_seqs(**over):
    return ok.KVSeqs(**{**dict(pages=FAKE, lens=FAKE, count=3, stride=2), **over})


@pytest.mark.parametrize("cache,seqs,status", [
    ({}, {}, ok.OKF_E_NODEV), ({"k": 0}, {}, ok.OKF_E_ARG), ({"v_scale": 0}, {}, ok.OKF_E_ARG),
    ({"dim": 24}, {}, ok.OKF_E_SHAPE), ({"dim": 320}, {}, ok.OKF_E_SHAPE), ({"pages": 0}, {}, ok.OKF_E_SHAPE),
    ({"heads": 0}, {}, ok.OKF_E_SHAPE), ({"v": FAKE + 4}, {}, ok.OKF_E_SHAPE), ({}, {"pages": 0}, ok.OKF_E_ARG),
    ({}, {"lens": 0}, ok.OKF_E_ARG), ({}, {"count": 0}, ok.OKF_E_SHAPE), ({}, {"stride": 0}, ok.OKF_E_SHAPE),
    ({}, {"lens": FAKE + 1}, ok.OKF_E_SHAPE)])
def test_cache_refusals(detached, cache, seqs, status):
    c, s = fake_cache(**cache), fake_seqs(**seqs)
    fails(lambda: detached.attn_decode(c, s, FAKE, FAKE, 1, 8, 1.0), status)
    fails(lambda: detached.kv_append(c, s, FAKE, FAKE, FAKE, 5), status)
    fails(lambda: detached.kv_read(c, s, FAKE, FAKE, FAKE, 5), status)
    fails(lambda: detached.kv_evict(c, s, fake_cache(), fake_seqs(), 100, 4, 10, FAKE, 128, FAKE, 128, FAKE), status)
    fails(lambda: detached.kv_evict(fake_cache(), fake_seqs(), c, s, 100, 4, 10, FAKE, 128, FAKE, 128, FAKE), status)


def test_call_refusals(detached):
    c, s, e = fake_cache(), fake_seqs(), detached
    for args, st in (((FAKE, FAKE, 1, 7, 1.0), ok.OKF_E_SHAPE), ((FAKE, FAKE, 0, 8, 1.0), ok.OKF_E_SHAPE),
                     ((0, FAKE, 1, 8, 1.0), ok.OKF_E_ARG), ((FAKE + 4, FAKE, 1, 8, 1.0), ok.OKF_E_SHAPE)):
        fails(lambda: e.attn_decode(c, s, *args), st)
    fails(lambda: e.attn_decode(c, s, FAKE, FAKE, 1, 8, 1.0, w_in=FAKE, w_stride=128), ok.OKF_E_ARG)
    fails(lambda: e.attn_decode(c, s, FAKE, FAKE, 1, 8, 1.0, w_out=FAKE, w_stride=127), ok.OKF_E_SHAPE)
    fails(lambda: e.attn_decode(c, s, FAKE, FAKE, 1, 8, 1.0, w_out=FAKE, w_stride=128), ok.OKF_E_NODEV)
    for call in (e.kv_append, e.kv_read):
        fails(lambda: call(c, s, FAKE, FAKE, FAKE, 0), ok.OKF_E_SHAPE)
        fails(lambda: call(c, s, FAKE, FAKE, 0, 5), ok.OKF_E_ARG)
        fails(lambda: call(c, s, FAKE, FAKE, FAKE, 5, type=ok.Q4_K), ok.OKF_E_TYPE)
        fails(lambda: call(c, s, FAKE, FAKE, FAKE, 5, k_stride=127), ok.OKF_E_SHAPE)
        fails(lambda: call(c, s, FAKE, FAKE, FAKE, 5, v_stride=130), ok.OKF_E_SHAPE)
        fails(lambda: call(c, s, FAKE + 8, FAKE, FAKE, 5), ok.OKF_E_SHAPE)
    fails(lambda: e.kv_append(c, s, 0, FAKE, FAKE, 5), ok.OKF_E_ARG)
    fails(lambda: e.kv_read(c, s, 0, 0, FAKE, 5), ok.OKF_E_ARG)
    fails(lambda: e.kv_read(c, s, 0, FAKE, FAKE, 5), ok.OKF_E_NODEV)

    def evict(keep=100, sink=4, recent=10, w=FAKE, ws=128, wo=FAKE, wos=128, kept=FAKE, dst=c, to=s):
        e.kv_evict(c, s, dst, to, keep, sink, recent, w, ws, wo, wos, kept)
    fails(lambda: evict(wo=0, wos=0), ok.OKF_E_NODEV)
    fails(lambda: evict(w=0), ok.OKF_E_ARG)
    fails(lambda: evict(kept=0), ok.OKF_E_ARG)
    for bad in (dict(keep=0), dict(keep=129), dict(sink=91), dict(ws=127), dict(wos=99), dict(dst=fake_cache(heads=1)),
                dict(dst=fake_cache(dim=128)), dict(to=fake_seqs(count=2))):
        fails(lambda: evict(**bad), ok.OKF_E_SHAPE)


# -------------------------------------------------------------------- prompt
def run_prompt(enc, q, k, v, qs, ks, t, window, scale, H, KV, D, **kw):
    """q, k, v on the GPU in the type; the output as float64."""
    o = torch.full((q.shape[0], H, D), float("nan"), dtype=TYPES[t], device="cuda")
    enc.attn_prompt(q, k, v, o, ints(qs), ints(ks), len(qs) - 1, qs[-1], ks[-1], H, KV, D, type=ok.BY_NAME[t],
                    scale=scale, window=window, **kw)
    enc.sync()
    return host(o)


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,KV,D,qlens,klens,window", [
    (1, 1, 16, [1], [1], 0),
    (4, 4, 64, [1, 1, 1], [1, 64, 65], 0),                 # one token behind a prefix
    (6, 2, 128, [63, 64, 65, 0, 1, 200], None, 0),         # ragged, an empty sequence
    (5, 1, 80, [130, 3], None, 0),
    (8, 1, 256, [70, 129], [300, 129], 0),
    (3, 3, 48, [257], None, 33),
    (4, 2, 128, [150, 40], [400, 40], 100),
    (2, 1, 128, [100, 20], [30, 0], 0),                    # more queries than keys, and no key at all
    (2, 2, 64, [300], [300], 1),                           # every row sees itself
    (2, 1, 192, [129], [140], 64),
    (16, 8, 128, [333], None, 0),
])
def test_prompt(enc, t, H, KV, D, qlens, klens, window):
    rng = np.random.default_rng(len(qlens) * 1000 + D + window)
    klens = klens or qlens
    qs, ks = starts(qlens), starts(klens)
    nk = max(ks[-1], 1)
    q, k, v = (dev(rng.standard_normal(s).astype(np.float32) * f, TYPES[t]) for s, f in
               (((qs[-1], H, D), 2.0), ((nk, KV, D), 1.0), ((nk, KV, D), 1.0)))
    got = run_prompt(enc, q, k, v, qs, ks[:-1] + [nk] if ks[-1] == nk else ks, t, window, D ** -0.5, H, KV, D)
    q, k, v = host(q), host(k), host(v)
    ref = ao.prompt(q, k, v, qs, ks, window, D ** -0.5)
    err = np.abs(got - ref).max()
    print("prompt", t, D, err, tol(q, k, v, D ** -0.5, max(klens), D, t), file=sys.stderr)
    assert err <= tol(q, k, v, D ** -0.5, max(klens), D, t)


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,KV,D,qlens,klens,window", [
    (2, 1, 128, [70], [1500], 0),                               # few rows, many keys: the keys over four groups
    (3, 1, 64, [33, 100], [900, 1200], 0),
    (2, 2, 80, [129], [1000], 900),
    (2, 1, 96, [65], [1024], 0),
    (2, 1, 256, [100], [800], 0),
    (48, 4, 64, [300, 1, 513], None, 0),                        # many rows: 128 a workgroup
    (48, 4, 128, [300, 1, 513], None, 77),
    (32, 8, 96, [700, 400], [700, 900], 0),
    (130, 2, 256, [290], None, 0),
    (16, 2, 64, [i * 7 % 13 for i in range(80)], None, 0),      # more sequences than a wavefront has lanes
    (2, 2, 64, [5, 0, 300, 64, 1, 129], [5, 7, 900, 1000, 1, 500], 0),  # tiles of the most keys first
])
def test_prompt_workgroups(enc, t, H, KV, D, qlens, klens, window):
    """The shapes of workgroups that the sizes choose, and the orders of their tiles."""
    test_prompt(enc, t, H, KV, D, qlens, klens, window)


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,n,before", [(2, 60, 1000), (40, 900, 0), (2, 100, 50)])
def test_prompt_unseen_by_workgroups(enc, t, H, n, before):
    """A NaN value and an infinite key half way: rows before them are as ever, all others show it."""
    rng = np.random.default_rng(16)
    D, m = 64, n + before
    at = before + n // 2
    q, k, v = (rng.standard_normal((r, h, D)).astype(np.float32) for r, h in ((n, H), (m, 1), (m, 1)))
    q_, k_, v_ = (dev(x, TYPES[t]) for x in (q, k, v))
    ref = ao.prompt(host(q_), host(k_), host(v_), [0, n], [0, m], 0, 0.1)
    v_[at, 0, 9], k_[at + 1, 0, 3] = float("nan"), float("inf")
    got = run_prompt(enc, q_, k_, v_, [0, n], [0, m], t, 0, 0.1, H, 1, D)
    assert np.abs(got[:n // 2] - ref[:n // 2]).max() <= tol(host(dev(q, TYPES[t])), k, v, 0.1, m, D, t)
    assert not np.isfinite(got[n // 2:, :, 9]).any()


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_prompt_strides(enc, t):
    """Rows of a fused projection, and a head-major layout; the gaps are left alone."""
    rng = np.random.default_rng(5)
    H, KV, D, n = 4, 2, 64, 150
    x = dev(rng.standard_normal((n, H + 2 * KV, D)).astype(np.float32), TYPES[t])
    q, k, v = x[:, :H], x[:, H:H + KV], x[:, H + KV:]
    ref = ao.prompt(host(q), host(k), host(v), [0, n], [0, n], 0, 0.2)
    bound = tol(host(q), host(k), host(v), 0.2, n, D, t)
    got = run_prompt(enc, q, k, v, [0, n], [0, n], t, 0, 0.2, H, KV, D, strides=(x.stride(0),) * 3 + (0,))
    assert np.abs(got - ref).max() <= bound
    qh, kh, vh = (y.transpose(0, 1).contiguous() for y in (q, k, v))
    o = torch.full((H, n + 3, D), 7.0, dtype=TYPES[t], device="cuda")
    enc.attn_prompt(qh, kh, vh, o, ints([0, n]), ints([0, n]), 1, n, n, H, KV, D, type=ok.BY_NAME[t], scale=0.2,
                    strides=(D,) * 4, head_strides=(n * D, n * D, n * D, (n + 3) * D))
    enc.sync()
    assert np.abs(host(o)[:, :n].transpose(1, 0, 2) - ref).max() <= bound
    assert np.all(host(o)[:, n:] == 7.0)


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_prompt_unseen_places(enc, t, bad):
    """NaN and infinities in keys and values that a row does not see: later ones, other
    sequences', ones the window leaves behind.  Rows that see them are not compared."""
    rng = np.random.default_rng(6)
    H, KV, D, lens = 4, 1, 128, [90, 70, 200]
    s = starts(lens)
    q, k, v = (rng.standard_normal((s[-1], h, D)).astype(np.float32) for h in (H, KV, KV))
    ref, clean = ao.prompt(q, k, v, s, s, 0, 0.1), None
    k, v = k.copy(), v.copy()
    k[s[1] + 40, 0, 5] = v[s[1] + 40, 0, 7] = bad      # seen by rows 40.. of the second sequence
    v[s[2] - 1, 0, :] = bad                            # its last row
    v[s[2] + 3, 0, 0] = bad                            # with window 50: by rows 3..52 of the third
    for window in (0, 50):
        q_, k_, v_ = (dev(x, TYPES[t]) for x in (q, k, v))
        got = run_prompt(enc, q_, k_, v_, s, s, t, window, 0.1, H, KV, D)
        with np.errstate(invalid="ignore"):
            clean = ao.prompt(host(q_), np.nan_to_num(host(k_), nan=0, posinf=0, neginf=0),
                              np.nan_to_num(host(v_), nan=0, posinf=0, neginf=0), s, s, window, 0.1)
        rows = np.ones(s[-1], bool)
        rows[s[1] + 40:s[2]] = False
        rows[s[2] + 3:s[2] + 53 if window else s[3]] = False
        bound = tol(q, np.nan_to_num(k, nan=0, posinf=0, neginf=0), np.nan_to_num(v, nan=0, posinf=0, neginf=0), 0.1,
                    200, D, t) + (0 if t == "f32" else 0)
        assert np.abs(got[rows] - clean[rows]).max() <= bound
        assert not np.isfinite(got[s[1] + 40:s[2]]).all(axis=2).any()  # (and those that see it show it)
    del ref


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_prompt_extremes(enc, t):
    """Scores of hundreds (one key takes all), equal scores, scores of -inf, a scale of 0."""
    rng = np.random.default_rng(7)
    n, H, KV, D = 130, 2, 1, 64
    q, k, v = (rng.standard_normal((n, h, D)).astype(np.float32) for h in (H, KV, KV))
    for f, scale in ((12.0, 1.0), (1.0, 0.0)):
        q_, k_, v_ = (dev(x, TYPES[t]) for x in (q * f, k, v))
        got = run_prompt(enc, q_, k_, v_, [0, n], [0, n], t, 0, scale, H, KV, D)
        ref = ao.prompt(host(q_), host(k_), host(v_), [0, n], [0, n], 0, scale)
        assert np.abs(got - ref).max() <= tol(host(q_), host(k_), host(v_), scale, n, D, t)
    k2 = np.zeros_like(k)
    k2[0], q2 = -np.inf, np.abs(q)   # key 0 scores -inf: row 0 sees nothing else
    q_, k_, v_ = (dev(x, TYPES[t]) for x in (q2, k2, v))
    got = run_prompt(enc, q_, k_, v_, [0, n], [0, n], t, 0, 1.0, H, KV, D)
    assert np.all(got[0] == 0)
    mean = np.cumsum(host(v_)[1:], 0) / np.arange(1, n)[:, None, None]
    assert np.abs(got[1:] - mean).max() <= tol(q, np.zeros_like(k), v, 1.0, n, D, t)


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_prompt_one_key_takes_nearly_all(enc, t):
    """The other 5999 keys, 2^-20.5 of the first each, keep their part of the output (whose
    value at the first key is 0): a weight's and the output's half step, and the sums' u."""
    n, D = 6000, 64
    q, k, v = torch.zeros(1, 1, D), torch.zeros(n, 1, D), torch.ones(n, 1, D)
    q[..., 0], k[0, 0, 0], v[0] = 4.0, 8.0, 0.0
    scale = 20.5 * np.log(2) / 32
    got = run_prompt(enc, *(x.to(TYPES[t]).cuda() for x in (q, k, v)), [0, 1], [0, n], t, 0, scale, 1, 1, D)
    w = (n - 1) * 2.0 ** -20.5
    ref = w / (1 + w)
    assert np.abs(got / ref - 1).max() <= (2 * n + 100) * U + (0 if t == "f32" else torch.finfo(TYPES[t]).eps)


@gpu
def test_prompt_bad_starts(enc):
    """Starts that leave the rows or decrease are clamped: nothing outside is read or written."""
    n, D = 70, 64
    x = torch.randn(n, 1, D, device="cuda")
    o = torch.full((n + 64, 1, D), 3.0, device="cuda")
    for qs, ks in (([-5, 40, 1000], [0, 2000, 30]), ([50, 20, 70], [-1, -1, 100])):
        enc.attn_prompt(x, x, x, o, ints(qs), ints(ks), 2, n, n, 1, 1, D)
        enc.sync()
        assert np.all(host(o)[n:] == 3.0)


# --------------------------------------------------------------------- cache
class Dev:
    """An oracle cache and its copy on the GPU, with sequences on pages in random order."""

    def __init__(self, lens, heads, D, seed, spare=0, more=0):
        self.rng = np.random.default_rng(seed)
        need = [max(1, (n + 63) // 64) for n in lens]
        self.stride = max(need) + more
        pages = sum(need) + spare + 1
        self.c = ao.Cache(pages, heads, D, self.rng)
        order = self.rng.permutation(pages).tolist()
        self.table = np.full((len(lens), self.stride), -1, np.int32)
        for i, n in enumerate(need):
            self.table[i, :n] = [order.pop() for _ in range(n)]
        self.free, self.lens, self.heads, self.D = order, list(lens), heads, D
        self.push()

    def push(self):
        self.k, self.v, self.ks, self.vs = dev(self.c.k), dev(self.c.device_v()), dev(self.c.ks), dev(self.c.vs)
        self.cache = ok.KVCache(self.k, self.v, self.ks, self.vs, len(self.c.k), self.heads, self.D)
        self.dtable, self.dlen = dev(self.table), ints(self.lens)
        self.seqs = ok.KVSeqs(self.dtable, self.dlen, len(self.lens), self.stride)

    def same(self, pages=None):
        pages = slice(None) if pages is None else pages
        assert np.array_equal(host(self.ks)[pages], self.c.ks[pages].astype(np.float64), equal_nan=True)
        assert np.array_equal(host(self.vs)[pages], self.c.vs[pages].astype(np.float64), equal_nan=True)


def held(d, s, n):
    """For each page of sequence s the tokens held of its first n: (page, count)."""
    return [(d.table[s, b], min(64, n - 64 * b)) for b in range((n + 63) // 64)
            if b < d.stride and 0 <= d.table[s, b] < len(d.c.k)]


def same_codes(d):
    gk, gv = host(d.k), ao.Cache.tokens_of(host(d.v))
    for s, n in enumerate(d.lens):
        for p, m in held(d, s, n):
            assert np.array_equal(gk[p, :, :m], d.c.k[p, :, :m]), ("k", s, p)
            assert np.array_equal(gv[p, :, :m], d.c.v[p, :, :m]), ("v", s, p)


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,heads,before,new", [
    (64, 2, [0, 0, 0], [1, 64, 65]), (128, 3, [63, 64, 10, 100], [1, 1, 3, 0]), (16, 1, [0], [1]),
    (256, 2, [5, 127, 0], [200, 2, 130]), (80, 8, [30, 31], [40, 0]), (48, 1, [0, 62], [128, 3])])
def test_append(enc, t, D, heads, before, new):
    lens = [a + b for a, b in zip(before, new)]
    d = Dev(lens, heads, D, D + len(new))
    st = starts(new)
    for f in (0.5, 4.0, 1e-3):   # scales that grow and that stay
        k, v = (dev(d.rng.standard_normal((st[-1], heads, D)).astype(np.float32) * f, TYPES[t]) for _ in range(2))
        enc.kv_append(d.cache, d.seqs, k, v, ints(st), st[-1], type=ok.BY_NAME[t])
        enc.sync()
        for s, n in enumerate(lens):
            d.c.append(d.table[s], n, host(k)[st[s]:st[s + 1]], host(v)[st[s]:st[s + 1]])
        d.same()
        same_codes(d)


@gpu
def test_append_rounds_ties_to_even(enc):
    """x / scale at and next to halves, under scales that are and are not powers of two."""
    d = Dev([64], 1, 128, 3)
    for top in (127.0, 127 * 0.7310585):
        s = np.float32(top) / np.float32(127)
        h = (np.arange(64 * 128) % 253 - 126.5).astype(np.float32) * s
        x = np.nextafter(h, np.where(np.arange(h.size) % 3 == 0, np.inf, np.where(np.arange(h.size) % 3 == 1, -np.inf, h)).astype(np.float32))
        x[0] = top
        x = x.reshape(64, 1, 128)
        enc.kv_append(d.cache, d.seqs, dev(x), dev(x), ints([0, 64]), 64)
        enc.sync()
        d.c.append(d.table[0], 64, x, x)
        d.same()
        same_codes(d)


@gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_append_not_finite(enc, bad):
    """The page's head reads as NaN, the others are as ever; a page begun anew is well again."""
    d = Dev([70, 70], 2, 64, 4)
    k, v = (d.rng.standard_normal((20, 2, 64)).astype(np.float32) for _ in range(2))
    k[3, 1, 5] = v[12, 0, 9] = bad
    for kk, vv in ((k, v), (np.nan_to_num(k, nan=1, posinf=1), np.nan_to_num(v, nan=1, posinf=1))):
        enc.kv_append(d.cache, d.seqs, dev(kk), dev(vv), ints([0, 10, 20]), 20)
        enc.sync()
        for s in range(2):
            d.c.append(d.table[s], 70, kk[10 * s:10 * s + 10], vv[10 * s:10 * s + 10])
        d.same()
        same_codes(d)
        assert np.isnan(host(d.ks)).any()  # (the first page's scale stays NaN)
    whole = d.rng.standard_normal((140, 2, 64)).astype(np.float32)
    enc.kv_append(d.cache, d.seqs, dev(whole), dev(whole), ints([0, 70, 140]), 140)
    enc.sync()
    for s in range(2):
        d.c.append(d.table[s], 70, whole[70 * s:70 * s + 70], whole[70 * s:70 * s + 70])
    d.same()
    same_codes(d)
    assert not np.isnan(host(d.ks)).any()


@gpu
def test_append_drops_what_has_no_page(enc):
    """Bad pages, lengths past the table, more new tokens than the length, strided rows."""
    d = Dev([200, 128, 5], 2, 64, 8)
    d.table[0, 1], d.table[1, 0] = len(d.c.k), -7
    d.lens = [400, 128, 5]      # the first past its table
    d.push()
    x = torch.randn(390 + 128 + 9, 6, 64, device="cuda")
    k, v = x[:, :2], x[:, 3:5]
    st = [0, 390, 390 + 128, 390 + 128 + 9]
    enc.kv_append(d.cache, d.seqs, k, v, ints(st), st[-1], k_stride=x.stride(0), v_stride=x.stride(0))
    enc.sync()
    for s, n in enumerate(d.lens):
        d.c.append(d.table[s], n, host(k)[st[s]:st[s + 1]], host(v)[st[s]:st[s + 1]])
    d.same()
    same_codes(d)


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,heads,lens,rows", [
    (64, 2, [70, 1, 0, 200], [70, 1, 0, 3]), (128, 1, [64], [64]), (256, 3, [130, 65], [100, 70]),
    (80, 2, [5, 300], [9, 299]), (16, 4, [1000], [1000])])
def test_read(enc, t, D, heads, lens, rows):
    d = Dev(lens, heads, D, D)
    if len(lens) == 4:
        d.table[3, 3] = 10 ** 6
        d.push()
    st = starts(rows)
    k, v = (torch.full((st[-1] + 1, heads + 1, D), 9.0, dtype=TYPES[t], device="cuda") for _ in range(2))
    kw = dict(type=ok.BY_NAME[t], k_stride=(heads + 1) * D, v_stride=(heads + 1) * D)
    enc.kv_read(d.cache, d.seqs, k, v, ints(st), st[-1], **kw)
    enc.sync()
    for x, i in ((k, 0), (v, 1)):
        got = host(x)
        assert np.all(got[-1] == 9.0) and np.all(got[:, heads] == 9.0)
        for s, n in enumerate(lens):
            ref = d.c.values(d.table[s], n)[i]
            ref = np.concatenate([np.zeros((max(0, rows[s] - n), heads, D)), ref[max(0, n - rows[s]):]])
            ref = torch.from_numpy(ref.astype(np.float32)).to(TYPES[t]).double().numpy()
            assert np.array_equal(got[st[s]:st[s + 1], :heads], ref), (i, s)
    only = torch.full_like(v, 9.0)
    enc.kv_read(d.cache, d.seqs, None, only, ints(st), st[-1], **kw)
    enc.sync()
    assert np.array_equal(host(only), host(v))


@gpu
def test_append_and_read_many_sequences(enc):
    """More sequences than a wavefront has lanes, some with no new token."""
    rng = np.random.default_rng(23)
    new = [int(x) for x in rng.integers(0, 4, 150)]
    new[149] = 70
    lens = [int(x) + m for x, m in zip(rng.integers(0, 130, 150), new)]
    d = Dev(lens, 1, 16, 24)
    st = starts(new)
    k, v = (rng.standard_normal((st[-1], 1, 16)).astype(np.float32) for _ in range(2))
    enc.kv_append(d.cache, d.seqs, dev(k), dev(v), ints(st), st[-1])
    ko, vo = (torch.empty(st[-1], 1, 16, device="cuda") for _ in range(2))
    enc.kv_read(d.cache, d.seqs, ko, vo, ints(st), st[-1])
    enc.sync()
    for s, n in enumerate(lens):
        d.c.append(d.table[s], n, k[st[s]:st[s + 1]], v[st[s]:st[s + 1]])
    d.same()
    same_codes(d)
    for s, n in enumerate(lens):
        for got, ref in zip((ko, vo), d.c.values(d.table[s], n)):
            assert np.array_equal(host(got)[st[s]:st[s + 1]], ref[n - new[s]:].astype(np.float32).astype(np.float64))


def decode_ref(d, q, window, scale):
    """Outputs [B][T][H][D] and weights [B][KV][tokens] of the oracle."""
    Bn, T, H, D = q.shape
    G = H // d.heads
    o, w = np.zeros(q.shape), np.zeros((Bn, d.heads, d.stride * 64))
    for s, n in enumerate(d.lens):
        k, v, have = d.c.values(d.table[s], max(n, 0))
        idx = np.nonzero(have)[0]
        for h in range(H):
            for t in range(T):
                at = n - T + t
                see = idx[(idx <= at) & ((idx > at - window) if window else True)]
                if len(see):
                    o[s, t, h:h + 1], p = ao.attend(q[s, t, h:h + 1], k[see, h // G], v[see, h // G], [len(see)], 0, scale)
                    w[s, h // G, see] += p[0]
    return o, w


@gpu
@pytest.mark.parametrize("H,KV,D,T,lens,window", [
    (1, 1, 16, 1, [1], 0), (2, 1, 64, 1, [1, 63, 64, 65, 0], 0), (8, 8, 128, 1, [300], 0), (5, 1, 128, 4, [129, 7, 2, 0], 0),
    (40, 8, 128, 1, [500, 77], 0), (16, 2, 64, 5, [200, 333], 0), (6, 2, 80, 3, [1000], 0), (4, 4, 256, 2, [64, 1500], 0),
    (20, 4, 256, 4, [700], 100), (8, 1, 48, 1, [2000, 10], 33), (3, 1, 192, 7, [90, 3000], 0), (4, 1, 128, 20, [100], 10),
    (2, 2, 128, 1, [9000], 0), (2, 1, 112, 2, [513], 1)])
def test_decode(enc, H, KV, D, T, lens, window):
    d = Dev(lens, KV, D, H + D + T, more=1)
    q = d.rng.standard_normal((len(lens), T, H, D)).astype(np.float32) * 2
    scale = D ** -0.5 / 2
    w = d.rng.random((len(lens), KV, d.stride * 64 + 5)).astype(np.float32)
    o, plain = (torch.full(q.shape, float("nan"), device="cuda") for _ in range(2))
    wi, wo = dev(w), torch.full(w.shape, 5.0, device="cuda")
    enc.attn_decode(d.cache, d.seqs, dev(q), plain, T, H, scale, window=window)
    enc.attn_decode(d.cache, d.seqs, dev(q), o, T, H, scale, window=window, w_in=wi, w_out=wo, w_stride=w.shape[2])
    enc.attn_decode(d.cache, d.seqs, dev(q), plain, T, H, scale, window=window, w_in=wi, w_out=wi, w_stride=w.shape[2])
    enc.sync()
    ref, add = decode_ref(d, q, window, scale)
    n, big = max(lens), max((np.abs(d.c.values(d.table[s], m)[i]).max() for s, m in enumerate(lens) for i in (0, 1) if m), default=1)
    kb = np.full((1, D), big)
    bound = tol(np.abs(q), kb, kb, scale, n, D)
    print("decode", D, T, np.abs(host(o) - ref).max(), bound, file=sys.stderr)
    assert np.abs(host(o) - ref).max() <= bound and np.abs(host(plain) - ref).max() <= bound
    rel = bound / big
    got, inplace = host(wo), host(wi)
    for s, m in enumerate(lens):
        want = w[s, :, :m] + add[s, :, :m]
        assert np.abs(got[s, :, :m] - want).max(initial=0) <= rel * T * (H // KV) + 4 * U * T * (H // KV)
        assert np.array_equal(got[s, :, :m], inplace[s, :, :m])
        assert np.all(got[s, :, m:] == 5.0) and np.array_equal(inplace[s, :, m:], w[s, :, m:].astype(np.float64))


@gpu
def test_decode_no_weights_before(enc):
    d = Dev([100], 2, 64, 1)
    q = d.rng.standard_normal((1, 1, 4, 64)).astype(np.float32)
    o, wo = torch.empty(q.shape, device="cuda"), torch.full((1, 2, 128), 9.0, device="cuda")
    enc.attn_decode(d.cache, d.seqs, dev(q), o, 1, 4, 0.1, w_out=wo, w_stride=128)
    enc.sync()
    assert np.abs(host(wo)[0, :, :100].sum(1) - 2).max() <= 200 * U * 2


@gpu
def test_decode_bad_pages_and_lengths(enc):
    """Page ids out of range, lengths past the table and below zero, NaN in pages that are not seen."""
    d = Dev([300, 200, 64, 100], 2, 64, 11)
    d.table[0, 2], d.table[1, 0], d.table[1, 3] = -5, len(d.c.k), 2 ** 30
    d.table[2, 0] = 2 ** 31 - 1      # a sequence without a single token
    d.lens = [300, 10 ** 6, 64, -3]
    free = d.free[0]
    d.c.ks[free] = d.c.vs[free] = np.nan
    d.push()
    q = d.rng.standard_normal((4, 2, 4, 64)).astype(np.float32)
    o, wo = torch.full(q.shape, 7.0, device="cuda"), torch.zeros((4, 2, d.stride * 64), device="cuda")
    enc.attn_decode(d.cache, d.seqs, dev(q), o, 2, 4, 0.1, w_out=wo, w_stride=d.stride * 64)
    enc.sync()
    d.lens[1], d.lens[3] = d.stride * 64 + 2, 0   # (both queries behind everything that the table has)
    ref, add = decode_ref(d, q, 0, 0.1)
    bound = tol(q, np.full((1, 64), 5.2), np.full(1, 5.2), 0.1, 320, 64)
    assert np.abs(host(o) - ref).max() <= bound
    assert np.all(host(o)[2:] == 0)
    got = host(wo)
    assert np.abs(got - add).max() <= bound * 4
    # an empty page's NaN scale shows where its tokens are seen
    d.table[0, 0] = free
    d.push()
    enc.attn_decode(d.cache, d.seqs, dev(q), o, 2, 4, 0.1, window=100)
    enc.sync()
    assert np.isfinite(host(o)[0]).all()     # (the window leaves the page behind)
    enc.attn_decode(d.cache, d.seqs, dev(q), o, 2, 4, 0.1)
    enc.sync()
    assert np.isnan(host(o)[0]).all() and np.isfinite(host(o)[1]).all()


@gpu
def test_decode_extreme_queries(enc):
    """Queries of zero, of very different sizes in one row, huge ones, NaN."""
    d = Dev([200], 1, 64, 12)
    q = d.rng.standard_normal((1, 1, 8, 64)).astype(np.float32)
    q[0, 0, 0] = 0
    q[0, 0, 1, 0] = 300
    q[0, 0, 2] *= 1e-30
    q[0, 0, 3] *= 1e-42
    q[0, 0, 4] *= 50
    q[0, 0, 6, 3] = np.nan
    q[0, 0, 7, 3] = np.inf
    o = torch.empty(q.shape, device="cuda")
    enc.attn_decode(d.cache, d.seqs, dev(q), o, 1, 8, 0.1)
    enc.sync()
    got = host(o)
    ref, _ = decode_ref(d, np.nan_to_num(q, nan=0, posinf=0), 0, 0.1)
    for h in range(6):
        bound = tol(q[0, 0, h:h + 1] * 8, np.full((1, 64), 5.2), np.full(1, 5.2), 0.1, 200, 64)
        assert np.abs(got[0, 0, h] - ref[0, 0, h]).max() <= bound, h
    assert np.isnan(got[0, 0, 6]).all() and not np.isfinite(got[0, 0, 7]).any()


@gpu
def test_decode_one_token_takes_nearly_all(enc):
    """The other tokens, 2^-27.5 of the first each, keep their part of the output (whose values
    in the first page are 0): the sums' u, 2^-23 of each page's weights, a score's few u times 19."""
    d = Dev([6400], 1, 64, 14)
    d.c.k[:], d.c.v[:], d.c.ks[:], d.c.vs[:] = 0, 100, 1, 0.01
    first = d.table[0, 0]
    d.c.k[first, 0, 0, 0], d.c.v[first] = 127, 0
    d.push()
    q = np.zeros((1, 1, 1, 64), np.float32)
    q[..., 0] = 1
    o = torch.empty(q.shape, device="cuda")
    enc.attn_decode(d.cache, d.seqs, dev(q), o, 1, 1, 27.5 * np.log(2) / 127)
    enc.sync()
    w = 2.0 ** -27.5
    ref = 6336 * w / (1 + 6399 * w) * 100 * np.float64(np.float32(0.01))
    assert np.abs(host(o) / ref - 1).max() <= (2 * 6400 + 200) * U


@gpu
def test_long_cache_offsets(enc):
    """Codes past 4 GiB: the last pages of a cache of 5 GB a side."""
    pages, heads, D = 80000, 8, 128
    c = ok.KVCache.new(pages, heads, D)
    rng = np.random.default_rng(13)
    table = np.array([[pages - 1, 3, pages - 2]], np.int32)
    x = rng.standard_normal((150, heads, D)).astype(np.float32)
    lens = ints([150])
    t = dev(table)
    seqs = ok.KVSeqs(t, lens, 1, 3)
    enc.kv_append(c, seqs, dev(x), dev(x), ints([0, 150]), 150)
    k, v = torch.empty(150, heads, D, device="cuda"), torch.empty(150, heads, D, device="cuda")
    enc.kv_read(c, seqs, k, v, ints([0, 150]), 150)
    enc.sync()
    assert np.abs(host(k) - x).max() <= np.abs(x).max() / 127 * 0.501 and np.array_equal(host(k), host(v))
    q = rng.standard_normal((1, 1, heads, D)).astype(np.float32)
    o = torch.empty(q.shape, device="cuda")
    enc.attn_decode(c, seqs, dev(q), o, 1, heads, 0.1)
    enc.sync()
    kk = host(k)
    ref = np.stack([ao.attend(q[0, :, h], kk[:, h], kk[:, h], [149], 0, 0.1)[0][0] for h in range(heads)])
    assert np.abs(host(o)[0, 0] - ref).max() <= tol(q, kk, kk, 0.1, 150, D)


# --------------------------------------------------------------------- evict
@gpu
@pytest.mark.parametrize("D,heads,lens,keep,sink,recent", [
    (64, 2, [300, 100, 0], 100, 4, 20), (128, 1, [129], 128, 0, 0), (16, 3, [1000, 64], 1, 0, 1), (256, 2, [200], 65, 65, 0),
    (80, 1, [5000], 700, 3, 64), (48, 2, [64, 63, 65], 64, 1, 1), (64, 1, [9000], 4000, 0, 0)])
def test_evict(enc, D, heads, lens, keep, sink, recent):
    nb = (keep + 63) // 64
    d = Dev(lens, heads, D, D + keep, spare=nb * len(lens))
    w = (d.rng.integers(0, 40, (len(lens), heads, d.stride * 64)) / 8).astype(np.float32)  # many ties
    w[:, :, 7::50] = -0.0
    w[:, :, 11::90] = np.nan
    w[:, :, 13::90] = -1.5
    w[:, :, 17::190] = np.inf
    w[:, :, 19::190] = -np.inf
    to = np.array([[d.free.pop() for _ in range(nb)] for _ in lens], np.int32)
    dto, new_len, kept = dev(to), torch.full((len(lens),), -9, dtype=torch.int32, device="cuda"), \
        torch.full((len(lens), heads, keep), -9, dtype=torch.int32, device="cuda")
    wo = torch.full((len(lens), heads, nb * 64), 77.0, device="cuda")
    enc.kv_evict(d.cache, d.seqs, d.cache, ok.KVSeqs(dto, new_len, len(lens), nb), keep, sink, recent, dev(w),
                 w.shape[2], wo, nb * 64, kept)
    enc.sync()
    gk, gv, gks, gvs = host(d.k), ao.Cache.tokens_of(host(d.v)), host(d.ks), host(d.vs)
    for s, n in enumerate(lens):
        m = min(n, keep)
        assert host(new_len)[s] == m
        for h, (tok, ck, tk, cv, tv) in enumerate(d.c.evict(d.table[s], n, w[s], keep, sink, recent)):
            assert host(kept)[s, h].tolist() == tok + [-1] * (keep - m)
            assert np.array_equal(host(wo)[s, h, :m], w[s, h, tok].astype(np.float64), equal_nan=True)
            assert np.all(host(wo)[s, h, m:] == 77.0)
            for b in range((m + 63) // 64):
                p, e = to[s, b], min(64, m - 64 * b)
                assert gks[p, h] == tk[b] and gvs[p, h] == tv[b]
                assert np.array_equal(gk[p, h, :e], ck[64 * b:64 * b + e]) and np.array_equal(gv[p, h, :e], cv[64 * b:64 * b + e])


@gpu
@pytest.mark.parametrize("kind", ["steps", "equal", "nan", "some nan", "tiny"])
@pytest.mark.parametrize("keep,sink,recent", [(700, 3, 64), (64, 64, 0), (1000, 0, 0)])
def test_evict_selects(enc, kind, keep, sink, recent):
    """Which tokens stay, of up to 33000: steps, equal weights, NaN (all, and more than may go), denormals."""
    lens = [33000, 16385, 16384, 1001, 1000]
    d = Dev(lens, 1, 16, keep, spare=16)
    n = d.stride * 64
    w = {"steps": d.rng.integers(0, 300, (5, 1, n)) / 8, "equal": np.full((5, 1, n), 0.25), "nan": np.full((5, 1, n), np.nan),
         "some nan": np.where(d.rng.random((5, 1, n)) < 0.99, np.nan, d.rng.random((5, 1, n))),
         "tiny": d.rng.integers(-5, 9, (5, 1, n)) * 1e-45}[kind].astype(np.float32)
    nb = (keep + 63) // 64
    dto, new_len = torch.full((5, nb), -1, dtype=torch.int32, device="cuda"), ints([0] * 5)   # (no pages: the list is what counts)
    kept, wo = torch.full((5, 1, keep), -9, dtype=torch.int32, device="cuda"), torch.full((5, 1, keep), 7.0, device="cuda")
    enc.kv_evict(d.cache, d.seqs, d.cache, ok.KVSeqs(dto, new_len, 5, nb), keep, sink, recent, dev(w), n, wo, keep, kept)
    enc.sync()
    for s, m in enumerate(lens):
        x = np.nan_to_num(w[s, 0, :m].astype(np.float64), nan=-np.inf)
        inner = sorted(range(sink, m - recent), key=lambda i: (-x[i], i))[:keep - sink - recent] if m > keep else []
        want = sorted([*range(sink), *inner, *range(m - recent, m)]) if m > keep else list(range(m))
        assert host(kept)[s, 0].tolist() == want + [-1] * (keep - len(want)), (s, m)
        assert np.array_equal(host(wo)[s, 0, :len(want)], w[s, 0, want].astype(np.float64), equal_nan=True)
        assert host(new_len)[s] == min(m, keep)


@gpu
def test_evict_bad_pages(enc):
    """Tokens without a page move as zeros; a NaN scale moves on; pages that do not exist get nothing."""
    d = Dev([200, 130], 1, 64, 21, spare=6)
    d.table[0, 1] = -1
    d.c.ks[d.table[1, 2]] = np.nan
    d.push()
    w = d.rng.random((2, 1, d.stride * 64)).astype(np.float32)
    to = np.array([[d.free.pop(), 10 ** 7], [d.free.pop(), d.free.pop()]], np.int32)
    new_len, kept = ints([0, 0]), torch.empty((2, 1, 100), dtype=torch.int32, device="cuda")
    dto = dev(to)
    enc.kv_evict(d.cache, d.seqs, d.cache, ok.KVSeqs(dto, new_len, 2, 2), 100, 2, 5, dev(w), w.shape[2], None, 0, kept)
    enc.sync()
    gk, gv, gks = host(d.k), ao.Cache.tokens_of(host(d.v)), host(d.ks)
    for s in range(2):
        (tok, ck, tk, cv, _), = d.c.evict(d.table[s], d.lens[s], w[s], 100, 2, 5)
        assert host(kept)[s, 0].tolist() == tok
        for b in range(2):
            if to[s, b] < len(d.c.k):
                e = min(64, 100 - 64 * b)
                assert np.array_equal(gks[to[s, b], 0], tk[b], equal_nan=True)
                assert np.array_equal(gk[to[s, b], 0, :e], ck[64 * b:64 * b + e])
                assert np.array_equal(gv[to[s, b], 0, :e], cv[64 * b:64 * b + e])


# -------------------------------------------------------------------- graphs
@gpu
def test_graph_step(enc):
    """Append, attend with weights, evict and a prompt captured into one graph; replayed with new
    inputs and lengths, with eager calls between the replays, each replay against the eager result."""
    hip, vp = ctypes.CDLL("libamdhip64.so"), ctypes.c_void_p
    H, KV, D = 8, 2, 128
    mine = ok.Enc(0)
    try:
        a, b = Dev([500, 90], KV, D, 31, spare=8), Dev([500, 90], KV, D, 31, spare=8)
        x = [torch.empty(2, KV, D, device="cuda") for _ in range(2)]
        q, st = torch.empty(2, 1, H, D, device="cuda"), ints([0, 1, 2])
        to = ints(np.array([a.free[:2], a.free[2:4]]).tolist())
        res = [{"o": torch.empty(2, 1, H, D, device="cuda"), "w": torch.zeros(2, KV, a.stride * 64, device="cuda"),
                "kept": torch.empty(2, KV, 100, dtype=torch.int32, device="cuda"), "len": ints([0, 0]),
                "p": torch.empty(2, H, D, device="cuda")} for _ in range(2)]

        def step(d, r):
            mine.kv_append(d.cache, d.seqs, x[0], x[1], st, 2)
            mine.attn_decode(d.cache, d.seqs, q, r["o"], 1, H, 0.1, w_in=r["w"], w_out=r["w"], w_stride=r["w"].shape[2])
            mine.kv_evict(d.cache, d.seqs, d.cache, ok.KVSeqs(to, r["len"], 2, 2), 100, 4, 10, r["w"], r["w"].shape[2],
                          None, 0, r["kept"])
            mine.attn_prompt(q, x[0], x[1], r["p"], st, st, 2, 2, 2, H, KV, D, scale=0.1)

        def fresh(i):
            g = torch.Generator(device="cuda").manual_seed(i)
            for y in (*x, q):
                y.normal_(0, 1 + i, generator=g)
            for d in (a, b):
                d.dlen.copy_(ints([401 + i, 64 + i]))
            torch.cuda.synchronize()
        fresh(0)
        step(b, res[1])
        mine.sync()
        b.push()
        b2, res[1]["w"] = b, torch.zeros_like(res[1]["w"])
        graph, exe, stream = vp(), vp(), vp(mine.stream)
        assert hip.hipStreamBeginCapture(stream, 0) == 0
        step(a, res[0])
        assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
        assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0) == 0
        try:
            for i in range(4):
                print("graph step", i, file=sys.stderr, flush=True)
                fresh(i)
                step(b2, res[1])
                mine.sync()
                assert hip.hipGraphLaunch(exe, stream) == 0
                mine.sync()
                for name in res[0]:
                    assert np.array_equal(host(res[0][name]), host(res[1][name])), name
        finally:
            hip.hipGraphExecDestroy(exe)
            hip.hipGraphDestroy(graph)
    finally:
        mine.close()
