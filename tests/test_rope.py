"""Norms of queries and keys with the rotation by positions (okf_norm_rope_rows) against 64 bits.

Tolerance, from the roundings (u = 2^-24): a norm's sum of D <= 256 squares goes over 16 a lane and
5 steps between lanes, 21 u, half of it after the root; 3 u for the division, the root and the
reciprocal, 2 u for the products: 16 u.  A cosine is off by 3 u (its argument, its
series, mag), the rotation by 2 u of each product: 24 u of |y0| + |y1| together.  The
frequencies are off by 4 2^-53 of themselves, an angle by that times the position.  16-bit
types: half a step of the result."""
import numpy as np
import pytest

import layer_oracle as lo

torch = pytest.importorskip("torch")
import chatokf_amd as ok  # noqa: E402
from test_attn import FAKE, TYPES, U, dev, fails, gpu, host, ints  # noqa: E402


@pytest.fixture()
def detached():
    e = ok.Enc(-1)
    yield e
    e.close()


def call(e, rope=None, **over):
    a = dict(pos=FAKE, n=4, q=FAKE, q_out=FAKE, heads=8, k=FAKE * 2, k_out=FAKE * 2, kv_heads=2, dim=64)
    e.norm_rope(rope or ok.Rope(64), **{**a, **over})


FAR = FAKE << 8
NAN = float("nan")


@pytest.mark.parametrize("over,status", [
    ({}, ok.OKF_E_NODEV), ({"type": ok.BF16, "q_norm": FAKE + 4}, ok.OKF_E_NODEV), ({"k": 0, "k_out": 0, "kv_heads": 0}, ok.OKF_E_NODEV),
    ({"q": 0}, ok.OKF_E_ARG), ({"q_out": 0}, ok.OKF_E_ARG), ({"k": 0}, ok.OKF_E_ARG), ({"k_out": 0}, ok.OKF_E_ARG), ({"pos": 0}, ok.OKF_E_ARG),
    ({"pos": 0, "rope": ok.Rope(0)}, ok.OKF_E_NODEV), ({"type": ok.Q8_0}, ok.OKF_E_TYPE), ({"heads": 0}, ok.OKF_E_SHAPE),
    ({"heads": 65536}, ok.OKF_E_SHAPE), ({"kv_heads": 0}, ok.OKF_E_SHAPE), ({"dim": 72}, ok.OKF_E_SHAPE), ({"dim": 272}, ok.OKF_E_SHAPE),
    ({"dim": 0}, ok.OKF_E_SHAPE), ({"n": 0}, ok.OKF_E_SHAPE), ({"n": 2 ** 31 - 1}, ok.OKF_E_SHAPE), ({"rope": ok.Rope(63)}, ok.OKF_E_SHAPE),
    ({"rope": ok.Rope(66)}, ok.OKF_E_SHAPE), ({"q": FAR + 8}, ok.OKF_E_SHAPE), ({"k_norm": FAKE + 2}, ok.OKF_E_SHAPE), ({"pos": FAKE + 1}, ok.OKF_E_SHAPE),
    ({"rope": ok.Rope(64, div=FAKE + 2)}, ok.OKF_E_SHAPE), ({"strides": (63, 0, 0, 0)}, ok.OKF_E_SHAPE), ({"strides": (0, 130, 0, 0)}, ok.OKF_E_SHAPE),
    ({"strides": (0, 0, 0, 2 ** 41)}, ok.OKF_E_SHAPE), ({"head_strides": (0, 0, 63, 0)}, ok.OKF_E_SHAPE),
    ({"rope": ok.Rope(64, base=0.0)}, ok.OKF_E_ARG), ({"rope": ok.Rope(64, base=-2.0)}, ok.OKF_E_ARG), ({"rope": ok.Rope(64, base=NAN)}, ok.OKF_E_ARG),
    ({"rope": ok.Rope(64, factor=0.0)}, ok.OKF_E_ARG), ({"rope": ok.Rope(64, factor=float("inf"))}, ok.OKF_E_ARG), ({"rope": ok.Rope(64, mag=NAN)}, ok.OKF_E_ARG),
    ({"rope": ok.Rope(64, original=100, base=1.0)}, ok.OKF_E_ARG), ({"rope": ok.Rope(64, original=100, beta_slow=0.0)}, ok.OKF_E_ARG),
    ({"rope": ok.Rope(64, original=100, beta_fast=-1.0)}, ok.OKF_E_ARG), ({"rope": ok.Rope(64, beta_fast=0.0)}, ok.OKF_E_NODEV),
    # overlaps: in place with other strides, half in place, outputs over each other or over the other input
    ({"strides": (512, 0, 1024, 0)}, ok.OKF_E_ARG), ({"q_out": FAKE + 64}, ok.OKF_E_ARG), ({"k_out": FAKE + 1024}, ok.OKF_E_ARG),
    ({"q_out": FAR, "k_out": FAR + 4096}, ok.OKF_E_ARG), ({"q_out": FAR, "k_out": FAR + 8192}, ok.OKF_E_NODEV),
    # columns of the same rows: apart, and one value into each other
    ({"k": FAKE + 2048, "k_out": FAKE + 2048, "strides": (768,) * 4}, ok.OKF_E_NODEV), ({"k": FAKE + 2032, "k_out": FAKE + 2032, "strides": (768,) * 4}, ok.OKF_E_ARG),
    ({"k": FAKE + 2048, "k_out": FAKE + 2048, "strides": (768, 1024, 768, 1024)}, ok.OKF_E_ARG)])
def test_refusals(detached, over, status):
    fails(lambda: call(detached, **over), status)


def bound(y, size, pos, f, t, rot, pairs):
    far = np.zeros(y.shape)
    if rot:
        a = np.abs(np.asarray(pos, np.float64))[:, None, None] * np.asarray(f, np.float64) * 4 * 2.0 ** -53
        far[..., 0:rot:2 if pairs else 1][..., :rot // 2] = a
        far[..., slice(1, rot, 2) if pairs else slice(rot // 2, rot)] = a
    b = (24 * U + far) * size
    return b + (0 if t == "f32" else torch.finfo(TYPES[t]).eps / 2 * (np.abs(y) + b) + 2.0 ** -25)


def check(enc, t, H, KV, D, pos, rot, pairs=False, norm=True, seed=0, **kw):
    rng = np.random.default_rng(seed + D + 7 * H)
    n = len(pos)
    q, k = (dev(rng.standard_normal((n, h, D)).astype(np.float32) * np.float32(3), TYPES[t]) for h in (H, KV))
    qn, kn = ((1 + 0.3 * rng.standard_normal((2, D))).astype(np.float32)) if norm else (None, None)
    div = (1 + 7 * rng.random(rot // 2)).astype(np.float32) if kw.pop("div", False) else None
    base = kw.pop("base", 1e4)
    f, mag = lo.freqs(rot, base, kw.get("factor", 1.0), kw.get("original", 0), kw.get("beta_fast", 32.0), kw.get("beta_slow", 1.0),
                      kw.get("mag", 0.0), div)
    qo, ko = (torch.full(x.shape, NAN, dtype=TYPES[t], device="cuda") for x in (q, k))
    r = ok.Rope(rot, pairs=pairs, base=base, div=None if div is None else dev(div), **kw)
    enc.norm_rope(r, ints(pos), n, q, qo, H, k, ko, KV, D, type=ok.BY_NAME[t], q_norm=dev(qn) if norm else None,
                  k_norm=dev(kn) if norm else None, eps=1e-5)
    enc.sync()
    for x, got, w in ((q, qo, qn), (k, ko, kn)):
        y, size = lo.norm_rope(host(x), pos, w, 1e-5, rot, pairs, f, mag)
        err = np.abs(host(got) - y) - bound(y, size, pos, f, t, rot, pairs)
        assert err.max() <= 0, (t, H, KV, D, rot, pairs, err.max())


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D", [16, 32, 48, 64, 80, 96, 112, 128, 144, 160, 192, 208, 240, 256])
def test_widths(enc, t, D):
    """Whole heads, parts of them, halves that do not break at 16 bytes, pairs, and none at all."""
    for rot in (D, D // 2, D // 4, 2, D - 2, 10, 0):
        for pairs in (False, True):
            check(enc, t, 3, 1, D, [0, 1, 77], rot, pairs, norm=rot % 4 == 0, seed=rot)


@gpu
@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("H,KV,n", [(1, 1, 1), (16, 8, 1), (40, 8, 300), (7, 7, 65), (5, 1, 1500), (65, 5, 9)])
def test_heads_and_rows(enc, t, H, KV, n):
    check(enc, t, H, KV, 128, list(range(1000, 1000 + n)), 128)
    check(enc, t, H, KV, 80, list(range(n)), 40, True)


@gpu
@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("kw", [
    dict(factor=8.0), dict(factor=0.5), dict(div=True), dict(div=True, factor=3.0), dict(mag=1.5), dict(original=4096, factor=16.0),
    dict(original=32768, factor=4.0, base=1e6), dict(original=2048, factor=40.0, mag=0.7), dict(original=100, factor=2.0),
    dict(original=8192, factor=0.5), dict(original=4096, factor=4.0, beta_fast=1.0, beta_slow=32.0), dict(original=4096, factor=4.0, div=True),
    dict(base=1.5), dict(base=1.0)])
@pytest.mark.parametrize("pairs", [False, True])
def test_scaling(enc, t, kw, pairs):
    check(enc, t, 4, 2, 128, [0, 5, 4095, 131071, 999983], 128, pairs, **kw)
    check(enc, t, 4, 2, 96, [3, 60000], 24, pairs, **kw)


@gpu
@pytest.mark.parametrize("pairs", [False, True])
def test_far_and_negative_positions(enc, pairs):
    check(enc, "f32", 2, 1, 128, [2 ** 31 - 1, 2 ** 31 - 2, -1, -2 ** 31, 123456789], 128, pairs)
    check(enc, "f32", 2, 1, 256, [2 ** 30 + 1, -77], 256, pairs, base=5e6)


@gpu
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_in_place_strides_and_one_kind(enc, t):
    """Queries and keys of fused rows in place, values beside them left alone; a head-major layout; queries alone."""
    rng = np.random.default_rng(1)
    n, H, KV, D, rot = 70, 6, 2, 64, 32
    x = dev(rng.standard_normal((n, H + 2 * KV, D)).astype(np.float32), TYPES[t])
    was, pos, w = host(x), list(range(n)), (1 + rng.random(D)).astype(np.float32)
    f, mag = lo.freqs(rot, 1e4)
    r, q, k = ok.Rope(rot), x[:, :H], x[:, H:H + KV]
    ref, size = lo.norm_rope(was[:, :H + KV], pos, w, 1e-6, rot, False, f, mag)
    b = bound(ref, size, pos, f, t, rot, False)
    enc.norm_rope(r, ints(pos), n, q, q, H, k, k, KV, D, type=ok.BY_NAME[t], q_norm=dev(w), k_norm=dev(w), eps=1e-6, strides=(x.stride(0),) * 4)
    enc.sync()
    got = host(x)
    assert (np.abs(got[:, :H + KV] - ref) <= b).all() and np.array_equal(got[:, H + KV:], was[:, H + KV:])
    planes = dev(was[:, :H].transpose(1, 0, 2).astype(np.float32), TYPES[t])
    out = torch.full((H, n + 3, D), 7.0, dtype=TYPES[t], device="cuda")
    enc.norm_rope(r, ints(pos), n, planes, out, H, dim=D, type=ok.BY_NAME[t], q_norm=dev(w), eps=1e-6, strides=(D, 0, D, 0),
                  head_strides=(n * D, 0, (n + 3) * D, 0))
    enc.sync()
    got = host(out).transpose(1, 0, 2)
    assert (np.abs(got[:n] - ref[:, :H]) <= b[:, :H]).all() and (got[n:] == 7).all()


@gpu
def test_unit_vectors(enc):
    """Norms of dim^-0.5 and eps / dim: x / sqrt(sum x^2 + eps), also of a row of zeros."""
    rng = np.random.default_rng(2)
    x = rng.standard_normal((5, 4, 96)).astype(np.float32)
    x[2, 1] = 0
    y, w = torch.empty(5, 4, 96, device="cuda"), np.full(96, 96 ** -0.5, np.float32)
    enc.norm_rope(ok.Rope(0), None, 5, dev(x), y, 4, dim=96, q_norm=dev(w), eps=1e-6 / 96)
    enc.sync()
    ref = x / np.sqrt((x.astype(np.float64) ** 2).sum(-1, keepdims=True) + 1e-6)
    assert np.abs(host(y) - ref).max() <= 26 * U and (host(y)[2, 1] == 0).all()


@gpu
@pytest.mark.parametrize("pairs,rot,D", [(False, 64, 128), (True, 64, 128), (False, 20, 80), (True, 20, 80)])
def test_what_is_not_finite_stays_in_its_pair(enc, pairs, rot, D):
    """Without a norm a NaN or an infinity reaches its own pair, and none where it does not turn."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((3, 2, D)).astype(np.float32)
    x[0, 0, 1], x[1, 1, rot + 1], x[2, 0, D - 1] = NAN, np.inf, NAN
    y = torch.empty(3, 2, D, device="cuda")
    enc.norm_rope(ok.Rope(rot, pairs=pairs), ints([1, 2, 3]), 3, dev(x), y, 2, dim=D)
    enc.sync()
    bad = ~np.isfinite(host(y))
    want = np.zeros(x.shape, bool)
    want[0, 0, [0, 1] if pairs else [1, 1 + rot // 2]] = True
    want[1, 1, rot + 1] = want[2, 0, D - 1] = True
    assert np.array_equal(bad, want) and host(y)[1, 1, rot + 1] == np.inf


@gpu
def test_offsets_past_32_bits(enc):
    """Rows so far apart that their values' offsets pass 2^32."""
    n, D, st = 5, 64, 1 << 30
    x = torch.empty(4 * st + 2 * D, dtype=torch.bfloat16, device="cuda")
    rng = np.random.default_rng(4)
    rows = rng.standard_normal((n, 1, D)).astype(np.float32)
    view = torch.as_strided(x, (n, 2, D), (st, D, 1))
    view[:, :1] = dev(rows, torch.bfloat16)
    pos, (f, mag) = list(range(n)), lo.freqs(D, 1e4)
    y, size = lo.norm_rope(host(view[:, :1].contiguous()), pos, None, 0, D, False, f, mag)
    enc.norm_rope(ok.Rope(D), ints(pos), n, x, x[D:], 1, dim=D, type=ok.BF16, strides=(st, 0, st, 0))
    enc.sync()
    assert (np.abs(host(view[:, 1:].contiguous()) - y) <= bound(y, size, pos, f, "bf16", D, False)).all()
