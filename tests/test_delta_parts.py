"""Each product of the gated delta rule in chunks (okf_delta_prompt), one factor times one other: keys that lie on a dimension
of their own make every sum of the chunk a single product, for every place where the matrix cores make one from bf16 parts.

Bounds, in units of u = 2^-24 of the exact product.  A value: the parts' products that are left out, below 1 u (|x1| <=
2^-8 and |x2| <= 2^-17 of the power of two below |x|, so x1 y2 + x2 y1 is at most 2^-24), and up to five sums of the
products that are made, each within a step of the last place, 2 u: 11 u.  Passing through a product with 1 is exact,
the parts' sum is the value.  16-bit outputs: half a step.
The mean of N signed errors: roundings to nearest have none, a value's error is no more than 1 u (left out) and five independent
roundings of 1 u / sqrt(3), together 1.7 u as a root mean square, so 5 x 1.7 u / sqrt(N) for N values that are not copies of each
other; the sums' own mean, 0.01 u each, 0.05 u.  Parts that are cut off, not rounded, leave out 0.6 u on average.
(test_bounds_see: both on the CPU; a part that is left out moves some values by far more than 11 u.)"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
import chatokf_amd as ok  # noqa: E402
from test_attn import TYPES, dev, gpu, host, ints  # noqa: E402

U = 2.0 ** -24
VALUE, SEQS, KH, VH, V = 11 * U, 256, 2, 6, 16
PLACES = ["QS", "KU", "QK", "PU", "TR", "KS", "KK", "KK across", "solve"]


def mean_bound(n):
    return (5 * 1.7 / np.sqrt(n) + 0.05) * U


def numbers(rng, shape, t):
    x = (rng.uniform(1, 2, shape) * 2.0 ** rng.integers(-2, 3, shape) * rng.choice((-1, 1), shape)).astype(np.float32)
    return torch.from_numpy(x).to(TYPES[t]).float().numpy()


class Products:
    """Inputs, and what they come to: (sequence, token) rows of the output, or (sequence, dimension) rows of the state,
    [..][VH][V]; samples: how many of them are different."""

    def __init__(self, place, K, t, seed=0):
        rng = np.random.default_rng(seed + K)
        G, M = VH // KH, K // 2
        items = {"KK": min(M, 16), "KK across": min(M, 16), "solve": min(K // 3, 8), "KS": min(M, 40)}.get(place, min(K, 40))
        m = {"KK": 2 * items, "KK across": 32, "solve": 32}.get(place, items)
        self.m, i = m, np.arange(items)
        self.q, self.k = np.zeros((SEQS, m, KH, K), np.float32), np.zeros((SEQS, m, KH, K), np.float32)
        self.v, self.beta = np.zeros((SEQS, m, VH, V), np.float32), np.ones((SEQS, m, VH), np.float32)
        self.S = np.zeros((SEQS, VH, K, V), np.float32)
        self.o, self.after = [], []
        one = lambda: numbers(rng, (items, KH), t)  # noqa: E731
        wide = lambda kind=t: numbers(rng, (items, VH, V), kind)  # noqa: E731
        group = lambda x: np.repeat(x.astype(np.float64), G, -1)[..., None] * np.ones(V)  # noqa: E731
        for s in range(SEQS):
            d = rng.permutation(K)  # dimensions of the items, and of what marks them
            a, b, e, f, g = one(), one(), d[:items], d[items:2 * items], d[2 * items:3 * items]
            if place == "QS":
                self.q[s, i, :, e], x = a, wide("f32")
                self.S[s][:, e], self.beta[s] = x.transpose(1, 0, 2), 0
                self.o.append((s, i, group(a) * x))
            elif place == "KU":
                self.k[s, i, :, e], self.v[s] = a, wide()
                self.after.append((s, e, group(a) * self.v[s]))
            elif place == "QK":
                self.q[s, i, :, e], self.k[s, i, :, e], self.v[s] = a, b, 1
                self.o.append((s, i, group(a * b.astype(np.float64))))
            elif place == "PU":
                self.q[s, i, :, e], self.k[s, i, :, e], self.v[s] = a, 1, wide()
                self.o.append((s, i, group(a) * self.v[s]))
            elif place == "TR":
                self.k[s, i, :, e], self.v[s], self.beta[s] = 1, wide(), numbers(rng, (items, VH), "f32")
                self.after.append((s, e, self.beta[s].astype(np.float64)[..., None] * self.v[s]))
            elif place == "KS":
                self.k[s, i, :, e], self.k[s, i, :, f], x = a, 1, wide("f32")
                self.S[s][:, e] = x.transpose(1, 0, 2)
                self.after.append((s, f, -group(a) * x))
            elif place in ("KK", "KK across"):
                early, late = (2 * i, 2 * i + 1) if place == "KK" else (i, 16 + i)
                self.k[s, early, :, e], self.k[s, late, :, e], self.k[s, late, :, f], self.v[s, early] = a, b, 1, 1
                self.after.append((s, f, -group(a * b.astype(np.float64))))
            else:
                self.k[s, 2 * i, :, e], self.k[s, 2 * i + 1, :, e], self.k[s, 2 * i + 1, :, f] = 1, a, 1
                self.k[s, 16 + i, :, f], self.k[s, 16 + i, :, g], self.v[s, 2 * i] = b, 1, 1
                self.after.append((s, g, group(a * b.astype(np.float64))))
        self.samples = SEQS * items * (KH if place in ("QK", "KK", "KK across", "solve") else VH if place == "TR" else VH * V)

    def errors(self, o, S):
        """Relative to the exact products."""
        out = [(o[s, i] - x) / x for s, i, x in self.o] + [(S[s][:, d].transpose(1, 0, 2) - x) / x for s, d, x in self.after]
        return np.stack(out)


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("K", [16, 32, 64, 80, 128, 160, 192, 208, 240, 256])
@pytest.mark.parametrize("place", PLACES)
def test_single_products(enc, place, K, t):
    p = Products(place, K, t)
    n = SEQS * p.m
    q, k, v = (dev(x.reshape(n, -1), TYPES[t]) for x in (p.q, p.k, p.v))
    o, S, out = torch.empty_like(v), dev(p.S), torch.empty(p.S.shape, device="cuda")
    enc.delta_prompt(q, k, v, dev(np.zeros((n, VH), np.float32)), dev(p.beta.reshape(n, VH)), o, ints(np.arange(SEQS + 1) * p.m), SEQS, n, KH, VH, K, V,
                     type=ok.BY_NAME[t], state_in=S, state_out=out)
    enc.sync()
    e = p.errors(host(o).reshape(SEQS, p.m, VH, V).astype(np.float64), host(out).astype(np.float64))
    if p.o and t != "f32":
        assert np.abs(e).max() <= VALUE + torch.finfo(TYPES[t]).eps / 2 * (1 + VALUE)
    else:
        assert np.abs(e).max() <= VALUE and abs(e.mean()) <= mean_bound(p.samples), (np.abs(e).max() / U, e.mean() / U, mean_bound(p.samples) / U)


def parts(x, cut):
    x, out = x.astype(np.float32), []
    for _ in range(3):
        u = x.view(np.uint32)
        if not cut:
            u = u + (0x7FFF + (u >> np.uint32(16) & np.uint32(1))).astype(np.uint32)
        y = (u & np.uint32(0xFFFF0000)).view(np.float32)
        out.append(y.astype(np.float64))
        x = x - y
    assert (x == 0).all()
    return out


def test_bounds_see():
    """The six products keep both bounds; cut parts do not keep the mean's, and without any of the five smaller products some value
    does not keep its own."""
    rng = np.random.default_rng(1)
    a, b = (numbers(rng, 2560, "f32") for _ in range(2))
    x = a.astype(np.float64) * b

    def error(cut=False, less=None):
        p, q = parts(a, cut), parts(b, cut)
        return (sum(p[i] * q[j] for i in range(3) for j in range(3) if i + j <= 2 and (i, j) != less) - x) / x
    e = error()
    assert np.abs(e).max() <= U and abs(e.mean()) <= mean_bound(2560) / 3
    assert abs(error(cut=True).mean()) > 2 * mean_bound(2560)
    for less in ((0, 1), (1, 0), (1, 1), (0, 2), (2, 0)):
        assert np.abs(error(less=less)).max() > 2 * VALUE


@gpu
@pytest.mark.parametrize("place", ["v", "S", "q", "k"])
def test_next_to_the_largest_number(enc, place):
    """Numbers that as bf16 would round to infinity: what comes of them is finite, and right, in every row and column."""
    K, n, big = 64, 40, np.float32(3.4e38)
    q, k, v, S = (np.zeros(s, np.float32) for s in ((n, K), (n, K), (n, V), (K, V)))
    beta, t = np.ones((n, 1), np.float32), np.arange(n)
    q[t, t], k[t, t], v[:] = 1, 1, 0.5
    if place == "v":
        v[7, 3] = v[39, 5] = big
    elif place == "S":
        S[7, 3] = S[39, 5] = big
        beta[:] = 0
    elif place == "q":
        q[7, 7] = q[39, 39] = big
    else:
        k[7, 7] = k[39, 39] = big
        q[7, 7] = q[39, 39] = 0.25
    o, out = torch.empty(n, V, device="cuda"), torch.empty(1, 1, K, V, device="cuda")
    enc.delta_prompt(dev(q), dev(k), dev(v), dev(np.zeros((n, 1), np.float32)), dev(beta), o, ints([0, n]), 1, n, 1, 1, K, V, state_in=dev(S), state_out=out)
    enc.sync()
    want = S + k.T.astype(np.float64) @ (v * beta)
    assert np.isfinite(host(o)).all()
    ref = q.astype(np.float64) @ want
    assert (np.abs(host(o) - ref) <= 2 * VALUE * np.abs(ref)).all() and (np.abs(host(out)[0, 0] - want) <= VALUE * np.abs(want)).all()
