"""fp32 precision of attention, as root mean squares: what the worst-case bounds of test_attn.py are
too wide to see, such as a part of a number left out of a product.

Bounds, in units of u = 2^-24, relative to the root mean square of the outputs.  A rounding is
a uniform error of up to u, so u / sqrt(3); independent ones add up in squares.  An error e of the
scores (in nats) changes an output, a weighted sum of independent values, by e in relative terms.
With s the scores' root mean square:
  prompt, scores: 6 D / 16 partial sums rounded, each of at most the whole sum's size:
    s sqrt(D / 8); products of parts left out, below 2^-23 of the whole each way: 2 s; the factor,
    the maximum's and the exponent's roundings: 2 s;
  prompt, values: 6 n / 16 partial sums over n keys: sqrt(n / 8); the exponential, the sum of
    weights and the quotient: 4;
  decode, scores: queries rounded to whole numbers, 2^22 or more for the largest of a row, which is
    up to 4.5 times its root mean square: 4.5 * 2^-22 / sqrt(12) = 5.2 u: 5.2 s; products'
    conversions and factors: 2 s; values: weights rounded to 2^-23 of a page's largest, 64 of
    them: 8 * 2^-23 / sqrt(12) = 4.6; n / 64 pages' sums: sqrt(n / 192); 4 as above.
A matrix instruction may round each of its sixteen products' sums: all that times sqrt(16) = 4.
Models of the arithmetic that leave out any one part fail these bounds (the tests on the CPU)."""
import numpy as np
import pytest

import attn_oracle as ao

torch = pytest.importorskip("torch")
from test_attn import Dev, decode_ref, dev, gpu, host, run_prompt  # noqa: E402

U = 2.0 ** -24
PAIRS = ((0, 0), (0, 1), (1, 0), (1, 1), (0, 2), (2, 0))   # of three bf16 parts: the products that are made


def rms(x):
    return np.sqrt(np.mean(np.square(x)))


def prompt_bound(s, D, n):
    return 4 * U * np.sqrt(s * s * (D / 8 + 4 + 4) + n / 8 + 16)


def decode_bound(s, n):
    return 4 * U * np.sqrt(s * s * (5.2 ** 2 + 4) + 4.6 ** 2 + n / 192 + 16)


def scores_rms(q, k, scale, before):
    """q [n][H][D] behind `before` keys of k [before + n][KV][D]: the seen scores' root mean square."""
    G, total, count = q.shape[1] // k.shape[1], 0.0, 0
    for h in range(q.shape[1]):
        sc = q[:, h] @ k[:, h // G].T * scale
        seen = np.tri(len(q), len(k), before, dtype=bool)
        total, count = total + np.square(sc[seen]).sum(), count + seen.sum()
    return np.sqrt(total / count)


def prompt_inputs(H, KV, D, n, before):
    rng = np.random.default_rng(H * 1000 + D + n)
    return [(rng.standard_normal((m, h, D)) * f).astype(np.float32) for m, h, f in ((n, H, 2), (n + before, KV, 1), (n + before, KV, 1))]


PROMPTS = [(2, 1, 128, 200, 0), (1, 1, 64, 100, 900), (2, 2, 80, 130, 20), (2, 1, 256, 150, 100), (1, 1, 16, 300, 0)]


# ------------------------------------------------------------- the arithmetic's models
def parts(x):
    x, out = x.astype(np.float32), []
    for _ in range(3):
        y = (x.view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)
        out.append(y.astype(np.float64))
        x = x - y
    return out


def model_prompt(q, k, v, scale, before, score_pairs=PAIRS, value_pairs=PAIRS):
    out, G = np.zeros(q.shape), q.shape[1] // k.shape[1]
    for h in range(q.shape[1]):
        a, b, c = parts(q[:, h]), parts(k[:, h // G]), parts(v[:, h // G])
        sc = np.where(np.tri(len(q), len(k), before, dtype=bool), sum(a[i] @ b[j].T for i, j in score_pairs) * scale, -np.inf)
        p = np.exp(sc - sc.max(1, keepdims=True))
        w = parts(p)
        out[:, h] = sum(w[i] @ c[j] for i, j in value_pairs) / p.sum(1, keepdims=True)
    return out


def digits(x, keep):
    """Whole numbers of three signed byte digits, of which the `keep` highest stay."""
    x = x.astype(np.int64)
    for d in range(3 - keep):
        x = (x + (128 << 8 * d)) >> 8 * (d + 1) << 8 * (d + 1)
    return x.astype(np.float64)


def model_decode(d, q, scale, q_digits=3, p_digits=3):
    out, G = np.zeros(q.shape), q.shape[2] // d.heads
    for s, n in enumerate(d.lens):
        k, v, _ = d.c.values(d.table[s], n)
        for t in range(q.shape[1]):
            end = n - q.shape[1] + t + 1
            for h in range(q.shape[2]):
                x = q[s, t, h].astype(np.float64)
                f = 2.0 ** (np.frexp(np.abs(x).max())[1] - 23 + (np.abs(x).max() / 2.0 ** (np.frexp(np.abs(x).max())[1] - 23) > 0x7F7F7F))
                sc = k[:end, h // G] @ digits(np.rint(x / f), q_digits) * f * scale
                top = sc.max()
                num, den = 0.0, 0.0
                for j in range(0, end, 64):
                    own = sc[j:j + 64].max()
                    p = np.exp(sc[j:j + 64] - own)
                    num = num + digits(np.rint(p * 0x7F7F7F), p_digits) @ v[j:j + 64, h // G][:len(p)] / 0x7F7F7F * np.exp(own - top)
                    den += p.sum() * np.exp(own - top)
                out[s, t, h] = num / den
    return out


@pytest.mark.parametrize("H,KV,D,n,before", PROMPTS)
def test_prompt_bound_sees_a_product_left_out(H, KV, D, n, before):
    q, k, v = prompt_inputs(H, KV, D, n, before)
    scale = D ** -0.5
    ref = ao.prompt(q, k, v, [0, n], [0, n + before], 0, scale)
    bound = prompt_bound(scores_rms(q.astype(np.float64), k.astype(np.float64), scale, before), D, n + before)
    assert rms(model_prompt(q, k, v, scale, before) - ref) / rms(ref) <= bound / 2
    for i in range(1, 6):
        less = PAIRS[:i] + PAIRS[i + 1:]
        for a, b in ((less, PAIRS), (PAIRS, less)):
            err = rms(model_prompt(q, k, v, scale, before, a, b) - ref) / rms(ref)
            assert err > bound, (PAIRS[i], a is less, err, bound)


DECODES = [(4, 2, 128, 1, [900, 130], 64), (5, 1, 80, 4, [700], 64), (20, 4, 256, 4, [500], 64), (2, 1, 16, 2, [3000], 64),
           (40, 1, 64, 1, [400, 65, 200], 64)]


def decode_inputs(H, KV, D, T, lens):
    d = Cpu(lens, KV, D, H + D)
    return d, d.rng.standard_normal((len(lens), T, H, D)).astype(np.float32) * 2, D ** -0.5 / 2


class Cpu(Dev):
    """test_attn.Dev without its copy on the GPU."""

    def push(self):
        if torch.cuda.is_available():
            super().push()


def decode_scores_rms(d, q, scale):
    G, total, count = q.shape[2] // d.heads, 0.0, 0
    for s, n in enumerate(d.lens):
        k = d.c.values(d.table[s], n)[0]
        for h in range(q.shape[2]):
            sc = q[s, :, h].astype(np.float64) @ k[:, h // G].T * scale
            seen = np.tri(q.shape[1], n, n - q.shape[1], dtype=bool)
            total, count = total + np.square(sc[seen]).sum(), count + seen.sum()
    return np.sqrt(total / count)


@pytest.mark.parametrize("H,KV,D,T,lens,seed", DECODES)
def test_decode_bound_sees_a_digit_left_out(H, KV, D, T, lens, seed):
    d, q, scale = decode_inputs(H, KV, D, T, lens)
    ref, bound = decode_ref(d, q, 0, scale)[0], decode_bound(decode_scores_rms(d, q, scale), max(lens))
    assert rms(model_decode(d, q, scale) - ref) / rms(ref) <= bound / 2
    for keep in ((2, 3), (3, 2)):
        assert rms(model_decode(d, q, scale, *keep) - ref) / rms(ref) > bound


# ------------------------------------------------------------------ the kernels
@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,KV,D,n,before", PROMPTS + [
    (2, 1, 192, 129, 11), (1, 1, 96, 65, 959), (130, 1, 64, 290, 0), (130, 1, 128, 290, 0), (130, 2, 256, 290, 0)])
def test_prompt_precision(enc, t, H, KV, D, n, before):
    """f32 within the bound above; f16 / bf16: every weight and the output rounded by up to half a
    step, eps / 2, so eps / sqrt(12) each, twice that allowed."""
    q, k, v = (dev(x, {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[t]) for x in prompt_inputs(H, KV, D, n, before))
    scale = D ** -0.5
    got = run_prompt(enc, q, k, v, [0, n], [0, n + before], t, 0, scale, H, KV, D)
    q, k, v = host(q), host(k), host(v)
    ref = ao.prompt(q, k, v, [0, n], [0, n + before], 0, scale)
    bound = prompt_bound(scores_rms(q, k, scale, before), D, n + before)
    if t != "f32":
        bound += 2 * torch.finfo(torch.float16 if t == "f16" else torch.bfloat16).eps * np.sqrt(2 / 12)
    err = rms(got - ref) / rms(ref)
    print("prompt", t, D, err, bound, flush=True)
    assert err <= bound


@gpu
@pytest.mark.parametrize("H,KV,D,T,lens,seed", DECODES)
def test_decode_precision(enc, H, KV, D, T, lens, seed):
    """Outputs, and the weights that the tokens got, whose own roundings the outputs' bound covers."""
    d, q, scale = decode_inputs(H, KV, D, T, lens)
    o, wo = torch.empty(q.shape, device="cuda"), torch.zeros((len(lens), KV, d.stride * 64), device="cuda")
    enc.attn_decode(d.cache, d.seqs, dev(q), o, T, H, scale, w_out=wo, w_stride=d.stride * 64)
    enc.sync()
    ref, add = decode_ref(d, q, 0, scale)
    bound = decode_bound(decode_scores_rms(d, q, scale), max(lens))
    print("decode", D, rms(host(o) - ref) / rms(ref), rms(host(wo) - add) / rms(add), bound, flush=True)
    assert rms(host(o) - ref) / rms(ref) <= bound
    assert rms(host(wo) - add) / rms(add) <= bound


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_same_bits_again(enc, t):
    """The same call on the same inputs gives the same bits: no sum depends on the order in which workgroups end."""
    H, KV, D, n = 16, 4, 128, 700
    q, k, v = (dev(x, {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[t]) for x in prompt_inputs(H, KV, D, n, 300))
    first = run_prompt(enc, q, k, v, [0, n], [0, n + 300], t, 0, 0.1, H, KV, D)
    d, x, scale = decode_inputs(8, 2, 128, 2, [3000, 65, 900])
    outs = []
    for i in range(4):
        o, wo = torch.empty(x.shape, device="cuda"), torch.zeros((3, 2, d.stride * 64), device="cuda")
        enc.attn_decode(d.cache, d.seqs, dev(x), o, 2, 8, scale, w_out=wo, w_stride=d.stride * 64)
        enc.sync()
        outs.append((host(o), host(wo)))
        assert np.array_equal(run_prompt(enc, q, k, v, [0, n], [0, n + 300], t, 0, 0.1, H, KV, D), first)
    for o, wo in outs[1:]:
        assert np.array_equal(o, outs[0][0]) and np.array_equal(wo, outs[0][1])
