"""The short causal convolution over packed sequences with states (okf_conv_rows) against 64 bits.

Tolerance (u = 2^-24): a sum of W products and a bias is off by (W + 2) u of its absolute values, SiLU
has slope 1.1 at most and adds 6 u of its value; 16-bit types: half a step.  States are copies."""
import numpy as np
import pytest

import layer_oracle as lo

torch = pytest.importorskip("torch")
import chatokf_amd as ok  # noqa: E402
from test_attn import FAKE, TYPES, U, dev, fails, gpu, host, ints, starts  # noqa: E402

FAR, NAN = FAKE << 8, float("nan")


@pytest.fixture()
def detached():
    e = ok.Enc(-1)
    yield e
    e.close()


@pytest.mark.parametrize("over,status", [
    ({}, ok.OKF_E_NODEV), ({"type": ok.F16, "bias": FAKE, "silu": True}, ok.OKF_E_NODEV), ({"x": 0}, ok.OKF_E_ARG), ({"w": 0}, ok.OKF_E_ARG),
    ({"y": 0}, ok.OKF_E_ARG), ({"start": 0}, ok.OKF_E_ARG), ({"type": ok.Q4_K}, ok.OKF_E_TYPE), ({"channels": 0}, ok.OKF_E_SHAPE),
    ({"width": 1}, ok.OKF_E_SHAPE), ({"width": 9}, ok.OKF_E_SHAPE), ({"n": 0}, ok.OKF_E_SHAPE), ({"seqs": 0}, ok.OKF_E_SHAPE),
    ({"n": 2 ** 31 - 1}, ok.OKF_E_SHAPE), ({"slots": 1}, ok.OKF_E_SHAPE), ({"slots": 1, "slot": FAKE}, ok.OKF_E_NODEV),
    ({"slots": 2 ** 31}, ok.OKF_E_SHAPE), ({"x": FAKE + 2}, ok.OKF_E_SHAPE), ({"x": FAKE + 4}, ok.OKF_E_NODEV), ({"x": FAKE + 2, "type": ok.BF16}, ok.OKF_E_NODEV),
    ({"w": FAKE + 2}, ok.OKF_E_SHAPE), ({"start": FAKE + 2}, ok.OKF_E_SHAPE), ({"slot": FAKE + 2, "slots": 9}, ok.OKF_E_SHAPE),
    ({"strides": (9, 0)}, ok.OKF_E_SHAPE), ({"strides": (0, 2 ** 41)}, ok.OKF_E_SHAPE), ({"channels": 2 ** 32 - 1, "n": 10 ** 6}, ok.OKF_E_SHAPE),
    ({"y": FAKE}, ok.OKF_E_ARG), ({"y": FAKE + 40}, ok.OKF_E_ARG), ({"y": FAKE + 40, "strides": (20, 20)}, ok.OKF_E_NODEV),
    ({"state_in": FAR, "state_out": FAR}, ok.OKF_E_NODEV), ({"state_in": FAR, "state_out": FAR + 120}, ok.OKF_E_ARG),
    ({"state_in": FAR, "state_out": FAR + 240}, ok.OKF_E_NODEV), ({"state_out": FAKE}, ok.OKF_E_ARG), ({"state_out": FAKE << 4}, ok.OKF_E_ARG),
    ({"state_in": FAKE << 4}, ok.OKF_E_ARG), ({"state_in": FAKE}, ok.OKF_E_NODEV)])
def test_refusals(detached, over, status):
    a = dict(x=FAKE, w=FAKE, y=FAKE << 4, start=FAKE, seqs=2, n=7, channels=10, width=4)
    fails(lambda: detached.conv(**{**a, **over}), status)


def bound(y, size, W, t):
    b = 1.1 * (W + 2) * U * size + 6 * U * np.abs(y)
    return b + (0 if t == "f32" else torch.finfo(TYPES[t]).eps / 2 * (np.abs(y) + b) + 2.0 ** -25)


def check(enc, t, C, W, lens, silu=True, bias=True, state=True, keep=True, slot=None, slots=0, inplace=False, pad=(0, 0), seed=0):
    rng = np.random.default_rng(seed + C + W)
    n, s = sum(lens), starts(lens)
    count = slots or len(lens)
    xs = torch.full((n + 2, C + pad[0]), NAN, dtype=TYPES[t], device="cuda")
    ys = torch.full((n + 2, C + pad[1]), 5.0, dtype=TYPES[t], device="cuda")
    xs[:n, :C] = dev(rng.standard_normal((n, C)).astype(np.float32), TYPES[t])
    w, b = rng.standard_normal((C, W)).astype(np.float32), rng.standard_normal(C).astype(np.float32) if bias else None
    st = dev(rng.standard_normal((count, W - 1, C)).astype(np.float32), TYPES[t])
    was = host(st)
    out = st if inplace else torch.full_like(st, 9.0)
    left = host(out)
    enc.conv(xs, dev(w), ys, ints(s), len(lens), n + 1, C, W, type=ok.BY_NAME[t], bias=dev(b) if bias else None, silu=silu,
             state_in=st if state else None, state_out=out if keep else None, slot=None if slot is None else ints(slot), slots=slots,
             strides=(C + pad[0], C + pad[1]))
    enc.sync()
    x, y = host(xs), host(ys)
    for i in range(len(lens)):
        at = i if slot is None else slot[i]
        begin = was[at] if state and 0 <= at < count else np.zeros((W - 1, C))
        ref, size, after = lo.conv(x[s[i]:s[i + 1], :C], w, b, begin, silu)
        assert (np.abs(y[s[i]:s[i + 1], :C] - ref) <= bound(ref, size, W, t)).all()
        if keep and 0 <= at < count:
            left[at] = after
    assert np.array_equal(host(out), left)
    assert (y[n:] == 5).all() and (y[:, C:] == 5).all()  # rows behind the last sequence, and what lies between rows


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("C,W,lens", [
    (1, 2, [1]), (8, 4, [1, 1, 1]), (24, 4, [33, 0, 2, 64, 1]), (2050, 4, [5, 31]), (1024, 4, [100]), (7, 8, [3, 9, 40]), (16, 5, [32, 33]),
    (40, 3, [i * 5 % 13 for i in range(70)]), (520, 6, [2, 1]), (96, 7, [65])])
def test_conv(enc, t, C, W, lens):
    check(enc, t, C, W, lens)
    check(enc, t, C, W, lens, silu=False, bias=False, state=False)
    check(enc, t, C, W, lens, inplace=True, seed=1)
    check(enc, t, C, W, lens, keep=False, pad=(3, 8))
    check(enc, t, C, W, lens, pad=(8, 16), seed=2)


@gpu
@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("lens", [[4000], [5001, 0, 17], [3000, 1, 6003], [7, 12999, 33], [20000]])
def test_long(enc, t, lens):
    """Sums of rows from which a thread goes through 8, 16, 24 and 32 of them."""
    check(enc, t, 40, 4, lens)
    check(enc, t, 17, 3, lens, inplace=True)


@gpu
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_slots(enc, t):
    """States anywhere in a pool; slots outside it begin from zeros and are not kept."""
    check(enc, t, 64, 4, [3, 1, 0, 40], slot=[6, 0, 3, 2], slots=8)
    check(enc, t, 64, 4, [3, 1, 0, 40], slot=[6, 0, 3, 2], slots=8, inplace=True)
    check(enc, t, 64, 4, [3, 1, 2, 40], slot=[6, -1, 8, 2 ** 31 - 1], slots=8, inplace=True)


@gpu
def test_in_parts(enc):
    """A sequence in one call and in several: the same bits."""
    rng = np.random.default_rng(6)
    n, C, W = 150, 48, 4
    x, w = dev(rng.standard_normal((n, C)).astype(np.float32)), dev(rng.standard_normal((C, W)).astype(np.float32))
    one, parts, st = torch.empty(n, C, device="cuda"), torch.empty(n, C, device="cuda"), torch.zeros(1, W - 1, C, device="cuda")
    enc.conv(x, w, one, ints([0, n]), 1, n, C, W, silu=True)
    at = 0
    for m in (1, 2, 1, 70, 3, 73):
        enc.conv(x[at:], w, parts[at:], ints([0, m]), 1, m, C, W, silu=True, state_in=st, state_out=st)
        at += m
    enc.sync()
    assert torch.equal(one, parts) and torch.equal(st[0], x[-3:])


@gpu
def test_starts_that_do_not_fit(enc):
    """Starts that leave the rows or decrease are clamped: nothing outside is read or written."""
    x = torch.ones(10, 16, device="cuda")
    for s in ([-5, 4, 100], [3, 3, 12], [2, 1, 6]):
        y = torch.full((12, 16), 5.0, device="cuda")
        enc.conv(x, torch.ones(16, 4, device="cuda"), y, ints(s), 2, 10, 16, 4)
        enc.sync()
        got, want = host(y), np.full((12, 16), 5.0)
        for a, b in zip(s, s[1:]):
            a = min(max(a, 0), 10)
            b = min(max(b, a), 10)
            want[a:b] = np.minimum(np.arange(1, b - a + 1), 4)[:, None]
        assert np.array_equal(got, want)


@gpu
def test_not_finite(enc):
    """A NaN reaches the rows that see it, of its channel; large sums do not overflow SiLU."""
    x = torch.ones(40, 8, device="cuda")
    x[20, 3] = NAN
    x[5, 0], x[6, 1] = 1e38, -1e38
    y = torch.empty(40, 8, device="cuda")
    enc.conv(x, torch.ones(8, 4, device="cuda"), y, ints([0, 40]), 1, 40, 8, 4, silu=True)
    enc.sync()
    bad = np.zeros((40, 8), bool)
    bad[20:24, 3] = True
    assert np.array_equal(np.isnan(host(y)), bad) and (host(y)[5:9, 0] == np.float32(1e38)).all() and (host(y)[6:10, 1] == 0).all()
