"""fp32 precision of the gated delta rule in chunks, as root mean squares: what the worst-case bounds of
test_delta.py are too wide to see, such as a part of a number left out of a product.

Bounds, in units of u = 2^-24, relative to the root mean square of the outputs; a rounding is a uniform
error of up to u, u / sqrt(3), and independent ones add up in squares.  Heads here forget within some
tokens and write little of each, so that errors of a state's few last tokens are all there are.
A sum of K terms in 32-term steps of six products: 6 K / 32 partial sums rounded, each of at most the
whole's size, sqrt(K / 16); K S, Q S, and K K^T and Q K^T inside T and P: K / 4 in all; three sums over a chunk's
32 tokens: 6; splits, decays, factors and the substitution: 16; the four products' left out parts, below 2^-23 of
the whole: 16.  A matrix instruction may round each of its products' sums: all that times sqrt(16) = 4; and
an output o = Q S + P U may be smaller than its two parts: by the factor that the 64-bit result shows.
Models of the arithmetic that leave out any one part fail these bounds (the tests on the CPU)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
from test_attn import dev, gpu, host, ints  # noqa: E402

U = 2.0 ** -24
PAIRS = ((0, 0), (0, 1), (1, 0), (1, 1), (0, 2), (2, 0))   # of three bf16 parts: the products that are made
C = 32


def rms(x):
    return np.sqrt(np.mean(np.square(x)))


def parts(x):
    x, out = x.astype(np.float32), []
    for _ in range(3):
        y = (x.view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)
        out.append(y.astype(np.float64))
        x = x - y
    return out


def product(a, b, pairs):
    """a b from bf16 parts, rounded to fp32; in 64 bits without pairs."""
    if pairs is None:
        return a @ b
    a, b = parts(a), parts(b)
    return sum(a[i] @ b[j] for i, j in pairs).astype(np.float32).astype(np.float64)


def chunks(q, k, v, g, beta, S, what=None, pairs=None):
    """One head's outputs; the product `what` ("all" for each) made of the given pairs of parts, the others in 64 bits.
    Also the sizes of the outputs' two parts."""
    o, size = np.zeros(v.shape), 0.0
    use = lambda name: pairs if what in (name, "all") else None  # noqa: E731
    for at in range(0, len(v), C):
        r = slice(at, at + C)
        qc, kc, vc, G, b = q[r], k[r], v[r], np.cumsum(g[r]), beta[r]
        n = len(vc)
        e = np.exp(G[:, None] - G[None])
        A = np.tril(product(kc, kc.T, use("T")) * e * b[:, None], -1)
        T = np.linalg.solve(np.eye(n) + A, np.diag(b))
        P = np.tril(product(qc, kc.T, use("P")) * e)
        X = vc - np.exp(G)[:, None] * product(kc, S, use("KS"))
        Uc = product(T, X, use("TX"))
        a, c = np.exp(G)[:, None] * product(qc, S, use("QS")), product(P, Uc, use("PU"))
        o[r] = a + c
        size += np.sum(a ** 2) + np.sum(c ** 2)
        S = np.exp(G[-1]) * S + product(kc.T, np.exp(G[-1] - G)[:, None] * Uc, use("KU"))
    return o, np.sqrt(size / o.size)


def inputs(K, V, n):
    rng = np.random.default_rng(K + n)
    q, k = (x / np.sqrt((x ** 2).sum(-1, keepdims=True)) for x in rng.standard_normal((2, n, K)))
    return [x.astype(np.float32) for x in (q, k, rng.standard_normal((n, V)), -rng.uniform(0.2, 0.6, n), rng.uniform(0.2, 0.4, n),
                                           rng.standard_normal((K, V)))]


def bound(K, o, size):
    return 4 * U * np.sqrt(K / 4 + 6 + 16 + 16) * max(size / rms(o), 1)


SIZES = [(64, 64, 300), (128, 128, 200), (32, 64, 400)]


@pytest.mark.parametrize("K,V,n", SIZES)
def test_bound_sees_a_product_left_out(K, V, n):
    """All six products are well within the bound; without any one of them it is not kept, in all products or in one of
    those that outputs are made of (of T and K S, which change new values by a fraction, without the largest two)."""
    x = [t.astype(np.float64) for t in inputs(K, V, n)]
    ref, size = chunks(*x)
    b = bound(K, ref, size)

    def err(what, less):
        return rms(chunks(*x, what, [p for p in PAIRS if p != less])[0] - ref) / rms(ref)
    assert err("all", None) <= b / 2
    for what in ("all", "P", "TX", "QS", "PU"):
        for less in PAIRS[1:]:
            assert err(what, less) > b, (what, less)
    for what in ("T", "KS"):
        assert err(what, (0, 1)) > b and err(what, (1, 0)) > b, what


@gpu
@pytest.mark.parametrize("form", ["step", "prompt"])
@pytest.mark.parametrize("K,V,n", SIZES)
def test_precision(enc, form, K, V, n):
    x = inputs(K, V, n)
    ref, size = chunks(*(t.astype(np.float64) for t in x))
    q, k, v, g, beta, S = (dev(t) for t in x)
    o = torch.empty_like(v)
    call = enc.delta_step if form == "step" else enc.delta_prompt
    call(q, k, v, g, beta, o, ints([0, n]), 1, n, 1, 1, K, V, state_in=S)
    enc.sync()
    assert rms(host(o) - ref) / rms(ref) <= bound(K, ref, size)
