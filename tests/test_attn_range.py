"""Attention at the ends of its arguments' ranges: windows as large as the type, scales and
queries of any finite size.  Bounds as in test_attn.py; scaling by a power of two is exact, so
that an input scaled one way and its scale the other leave the bound as it was."""
import numpy as np
import pytest

import attn_oracle as ao

torch = pytest.importorskip("torch")
import chatokf_amd as ok  # noqa: E402
from test_attn import TYPES, Dev, attn, decode_ref, dev, fails, gpu, host, run_prompt, starts, tol  # noqa: E402


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("window", [0xFFFFFFFF, 0x80000000, 0x7FFFFFFF, 0x7FFFFFFE, 0x7FFFFFC0, 200, 25])
@pytest.mark.parametrize("H,KV,D,qlens,klens", [(2, 1, 128, [100, 20, 70], [30, 0, 70]),   # positions from -70 on
                                                (40, 2, 64, [700, 330], [200, 301])])     # 128 rows a workgroup
def test_prompt_window_larger_than_the_keys(enc, t, window, H, KV, D, qlens, klens):
    """More queries than keys: the first tile's positions are below zero, whatever the window."""
    rng = np.random.default_rng(D + len(qlens))
    qs, ks = starts(qlens), starts(klens)
    q, k, v = (dev(rng.standard_normal((s[-1], h, D)).astype(np.float32), TYPES[t]) for s, h in ((qs, H), (ks, KV), (ks, KV)))
    got = run_prompt(enc, q, k, v, qs, ks, t, window, D ** -0.5, H, KV, D)
    q, k, v = host(q), host(k), host(v)
    ref = ao.prompt(q, k, v, qs, ks, window, D ** -0.5)
    assert np.abs(got - ref).max() <= tol(q, k, v, D ** -0.5, max(klens), D, t)


@gpu
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_prompt_scale_of_any_size(enc, t):
    """Large inputs under a scale as small: a power of two more here and less there changes nothing;
    a scale of 0 weighs all keys alike, whatever the products."""
    rng = np.random.default_rng(17)
    n, H, KV, D = 150, 2, 1, 64
    q, k, v = (rng.standard_normal((n, h, D)).astype(np.float32) for h in (H, KV, KV))
    for e, scale in ((56, 2.0 ** -115), (60, 0.0), (-40, 2.0 ** 77)):
        q_, k_, v_ = dev(np.ldexp(q, e), TYPES[t]), dev(np.ldexp(k, e), TYPES[t]), dev(v, TYPES[t])
        got = run_prompt(enc, q_, k_, v_, [0, n], [0, n], t, 0, scale, H, KV, D)
        ref = ao.prompt(host(q_), host(k_), host(v_), [0, n], [0, n], 0, scale)
        assert np.abs(got - ref).max() <= tol(q, k, v, scale * 4.0 ** e, n, D, t), e


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [1.0, -1.0, 0.5, 0.125])
@pytest.mark.parametrize("H,n,before", [(2, 70, 100), (2, 60, 1000), (40, 900, 0)])
def test_prompt_scores_at_the_types_ends(enc, t, scale, H, n, before):
    """Keys whose scores are the type's lowest or highest value, as a mask or a bias within the keys
    has them: alone they share the weight, beside others they take none or all of it."""
    rng = np.random.default_rng(19)
    D, m, top = 64, n + before, float(torch.finfo(TYPES[t]).max if t == "f16" else torch.finfo(torch.bfloat16).max)
    q, k, v = np.zeros((n, H, D), np.float32), np.zeros((m, 1, D), np.float32), rng.standard_normal((m, 1, D)).astype(np.float32)
    q[..., 0] = 1
    usual = rng.standard_normal(m) * 3
    for kind in ("lowest", "highest", "lowest and usual", "lowest first", "highest here and there", "both"):
        k[:, 0, 0] = {"lowest": -top, "highest": top, "lowest and usual": np.where(rng.random(m) < 0.3, -top, usual),
                      "lowest first": np.where(np.arange(m) < m // 2 + 3, -top, usual),
                      "highest here and there": np.where(np.arange(m) % 97 == 50, top, usual),
                      "both": np.where(np.arange(m) % 97 == 50, top, -top)}[kind]
        q_, k_, v_ = (dev(x, TYPES[t]) for x in (q, k, v))
        got = run_prompt(enc, q_, k_, v_, [0, n], [0, m], t, 0, scale, H, 1, D)
        ref = ao.prompt(host(q_)[:, :1], host(k_), host(v_), [0, n], [0, m], 0, scale)  # (all heads alike)
        small = np.where(np.abs(k) < 100, k, 0)
        assert np.abs(got - ref).max() <= tol(q, small, v, abs(scale), m, D, t), kind


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("scale", [2.0 ** -4, 2.0 ** -2, 16.0, 256.0, 2.0 ** 12, 2.0 ** 30, 2.0 ** 90])
@pytest.mark.parametrize("H,n,before", [(2, 70, 100), (2, 60, 1000), (40, 900, 0)])
def test_prompt_large_scores(enc, t, sign, scale, H, n, before):
    """Scores of sign 2^25 + 4 j, j < 16, which fp32 holds exactly, under scales that leave neighbours
    some or no weight: exponents of up to 2^117.  Bound: the sums' u, a few u of the exponents that
    still count (up to 30), and for f16 / bf16 a weight's and the output's half step."""
    rng = np.random.default_rng(20)
    D, m = 64, n + before
    q, k, v = np.zeros((n, H, D), np.float32), np.zeros((m, 1, D), np.float32), rng.standard_normal((m, 1, D)).astype(np.float32)
    q[..., 0], q[..., 1], k[..., 0] = 2048, 4, sign * 16384
    k[:, 0, 1] = rng.integers(0, 16, m)
    q_, k_, v_ = (dev(x, TYPES[t]) for x in (q, k, v))
    got = run_prompt(enc, q_, k_, v_, [0, n], [0, m], t, 0, scale, H, 1, D)
    ref = ao.prompt(host(q_)[:, :1], host(k_), host(v_), [0, n], [0, m], 0, scale)  # (all heads alike)
    bound = (2 * m + 100) * 2.0 ** -24 + (0 if t == "f32" else torch.finfo(TYPES[t]).eps)
    assert np.abs(got - ref).max() <= bound * np.abs(v).max()


@pytest.mark.parametrize("over,status", [({"n_q": 0x7FFFFF00}, ok.OKF_E_NODEV), ({"n_q": 0x7FFFFF01}, ok.OKF_E_SHAPE),
                                         ({"n_k": 0x7FFFFF00}, ok.OKF_E_NODEV), ({"n_k": 0x7FFFFF01}, ok.OKF_E_SHAPE)])
def test_prompt_rows_that_32_bits_hold(over, status):
    """A tile's rows and keys are numbered past the last one."""
    e = ok.Enc(-1)
    fails(lambda: attn(e, **over), status)
    e.close()


@gpu
@pytest.mark.parametrize("H", [8, 40])     # (with weights from the scores that are kept, and made again)
@pytest.mark.parametrize("qe,se,ke", [(127, -127, 0), (126, -126, 0), (-126, 126, 0), (-140, 120, 20), (0, -120, 120),
                                      (0, 100, -100), (100, 0, -100)])
def test_decode_sizes(enc, H, qe, se, ke):
    """Queries, scale and key scales 2^qe, 2^se and 2^ke of the usual: from the largest numbers to denormal ones."""
    d = Dev([333, 70], 1, 64, 15)
    d.c.ks[:] = np.ldexp(d.c.ks, ke)
    d.push()
    q = d.rng.standard_normal((2, 1, H, 64)).astype(np.float32)
    q = np.ldexp(np.float32(1.99) * q / np.abs(q).max(-1, keepdims=True), qe)
    assert np.isfinite(q).all()
    scale = 2.0 ** (se - 3)
    o, wo = torch.empty(q.shape, device="cuda"), torch.zeros((2, 1, d.stride * 64), device="cuda")
    enc.attn_decode(d.cache, d.seqs, dev(q), o, 1, H, scale, w_out=wo, w_stride=d.stride * 64)
    enc.sync()
    ref, add = decode_ref(d, q, 0, scale)
    bound = tol(np.ldexp(q.astype(np.float64), -qe), np.full((1, 64), 5.2), np.full(1, 5.2), 0.125, 333, 64)
    assert np.abs(host(o) - ref).max() <= bound
    assert np.abs(host(wo) - add).max() <= bound / 5.2 * H + 4 * 2.0 ** -24 * H
