"""Head norms with rotation, the short convolution and the gated delta rule in 64 bits, row by row (numpy)."""
import numpy as np

LD = np.longdouble


def freqs(rot, base, factor=1.0, original=0, fast=32.0, slow=1.0, mag=0.0, div=None):
    """Radians a position (80 bits) and the factor of sines and cosines."""
    i = np.arange(rot // 2).astype(LD)
    f = LD(np.float32(base)) ** (-2 * i / LD(rot))
    if div is not None:
        f = f / np.asarray(div, LD)
    if not original:
        return f / LD(np.float32(factor)), mag or 1.0

    def dim(turns):
        return rot * np.log(original / (turns * 2 * np.pi)) / (2 * np.log(np.float64(np.float32(base))))
    low, high = max(np.floor(dim(fast)), 0.0), min(np.ceil(dim(slow)), rot - 1.0)
    ramp = np.clip((i - LD(low)) / LD(max(high - low, 0.001)), 0, 1)
    return f * (ramp / LD(np.float32(factor)) + 1 - ramp), mag or (0.1 * np.log(np.float32(factor)) + 1 if factor > 1 else 1.0)


def norm_rope(x, pos, norm, eps, rot, pairs, f, mag):
    """x [n][heads][D]: the result, and for each value the sizes that its roundings are relative to."""
    y = x.astype(np.float64).copy()
    if norm is not None:
        y *= norm / np.sqrt((y ** 2).mean(-1, keepdims=True) + eps)
    size = np.abs(y)
    if rot:
        a = np.asarray(pos).astype(LD)[:, None] * f
        c, s = (np.asarray(t * LD(mag), np.float64)[:, None] for t in (np.cos(a), np.sin(a)))
        lo, hi = (slice(0, rot, 2), slice(1, rot, 2)) if pairs else (slice(0, rot // 2), slice(rot // 2, rot))
        y0, y1 = y[..., lo].copy(), y[..., hi].copy()
        y[..., lo], y[..., hi] = y0 * c - y1 * s, y0 * s + y1 * c
        size[..., lo] = size[..., hi] = (np.abs(y0) + np.abs(y1)) * mag
    return y, size


def conv(x, w, b, state, silu):
    """One sequence: x [m][C], state [W - 1][C]: y, the sums' absolute values, the state left."""
    W = w.shape[1]
    h = np.concatenate([state, x]).astype(np.float64)
    y, size = np.zeros(x.shape), np.zeros(x.shape)
    if b is not None:
        y, size = y + b, size + np.abs(b)
    for j in range(W):
        y = y + h[j:j + len(x)] * w[:, j]
        size = size + np.abs(h[j:j + len(x)] * w[:, j])
    if silu:
        y = y / (1 + np.exp(-y))
    return y, size, h[len(x):]


def delta(q, k, v, g, beta, state, scale):
    """One sequence: q, k [m][KH][DK], v [m][VH][DV], g, beta [m][VH], state [VH][DK][DV]: o, the state left."""
    G = v.shape[1] // k.shape[1]
    S, o = state.astype(np.float64).copy(), np.zeros(v.shape)
    with np.errstate(invalid="ignore", over="ignore"):
        for t in range(len(v)):
            for h in range(v.shape[1]):
                kt, qt, e = k[t, h // G].astype(np.float64), q[t, h // G].astype(np.float64), np.exp(np.float64(g[t, h]))
                S[h] = S[h] * e if e else np.zeros_like(S[h])
                S[h] += np.outer(kt, beta[t, h] * (v[t, h] - kt @ S[h]))
                o[t, h] = qt @ S[h] * scale
    return o, S
