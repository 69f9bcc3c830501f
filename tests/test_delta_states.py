"""States and outputs of the gated delta rule in chunks as root mean squares, at the narrowest and the widest keys and for 16-bit inputs,
whose outputs' rounding hides what a state shows.

Bounds as test_delta_precision.py derives them, 4 u sqrt(K / 4 + 38) of the root mean square, u = 2^-24; a state is
S' = e^G S + K^T U, of the same sums as an output, and may be smaller than its two parts, by the factor that
the 64-bit result shows.  16-bit outputs: half a step on top.  Fewer parts are made of 16-bit inputs, and no more."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
import chatokf_amd as ok  # noqa: E402
from test_attn import TYPES, dev, gpu, host, ints  # noqa: E402
from test_delta_precision import C, U, inputs, rms  # noqa: E402

SIZES = [(16, 32, 400), (128, 48, 130), (208, 32, 107), (240, 64, 150), (256, 48, 200)]
PAIRS = ((0, 0), (0, 1), (1, 0), (1, 1), (0, 2), (2, 0))


def parts(x):
    x, out = x.astype(np.float32), []
    for _ in range(3):
        u = x.view(np.uint32)
        y = (u + (0x7FFF + (u >> np.uint32(16) & np.uint32(1))).astype(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)
        out.append(y.astype(np.float64))
        x = x - y
    return out


def rule(q, k, v, g, beta, S, pairs=None):
    """One head in 64 bits, in chunks: outputs, the state left, and by how much the parts of either are larger; K^T U made of these
    pairs of parts alone."""
    o, sizes = np.zeros(v.shape), []
    for at in range(0, len(v), C):
        r = slice(at, at + C)
        qc, kc, vc, G, b = q[r], k[r], v[r], np.cumsum(g[r]), beta[r]
        e = np.exp(G[:, None] - G[None])
        T = np.linalg.solve(np.eye(len(vc)) + np.tril(kc @ kc.T * e * b[:, None], -1), np.diag(b))
        u = T @ (vc - np.exp(G)[:, None] * (kc @ S))
        x, y = np.exp(G)[:, None] * (qc @ S), np.tril(qc @ kc.T * e) @ u
        o[r] = x + y
        sizes.append((x ** 2).sum() + (y ** 2).sum())
        w, old = np.exp(G[-1] - G)[:, None] * u, np.exp(G[-1]) * S
        p, t = (parts(kc.T), parts(w)) if pairs else ((kc.T,), (w,))
        new = sum(p[i] @ t[j] for i, j in pairs or ((0, 0),))
        S = old + new
    return o, S, max(np.sqrt(sum(sizes) / o.size) / rms(o), 1), max(np.sqrt(rms(old) ** 2 + rms(new) ** 2) / rms(S), 1)


def bound(K):
    return 4 * U * np.sqrt(K / 4 + 38)


@pytest.mark.parametrize("K,V,n", SIZES)
def test_bound_sees_a_part_left_out(K, V, n):
    """Of K^T U: the six products keep the bound, without one of the first two that hold a second part they do not."""
    x = [t.astype(np.float64) for t in inputs(K, V, n)]
    _, S, _, size = rule(*x)
    assert rms(rule(*x, PAIRS)[1] - S) <= bound(K) * size * rms(S) / 4
    for less in ((0, 1), (1, 0)):
        assert rms(rule(*x, [p for p in PAIRS if p != less])[1] - S) > 16 * bound(K) * size * rms(S)


@gpu
@pytest.mark.parametrize("form", ["step", "prompt"])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("K,V,n", SIZES)
def test_states(enc, form, t, K, V, n):
    q, k, v, g, beta, S = (dev(x) for x in inputs(K, V, n))
    q, k, v = (x.to(TYPES[t]) for x in (q, k, v))
    ref, after, so, ss = rule(*(host(x).astype(np.float64) for x in (q, k, v, g, beta, S)))
    o, out = torch.empty_like(v), torch.empty_like(S)
    call = enc.delta_step if form == "step" else enc.delta_prompt
    call(q, k, v, g, beta, o, ints([0, n]), 1, n, 1, 1, K, V, type=ok.BY_NAME[t], state_in=S, state_out=out)
    enc.sync()
    assert rms(host(out) - after) <= bound(K) * ss * rms(after)
    assert rms(host(o) - ref) <= (bound(K) * so + (0 if t == "f32" else torch.finfo(TYPES[t]).eps / 2)) * rms(ref)
