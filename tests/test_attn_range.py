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
