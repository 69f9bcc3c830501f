"""The gated delta rule, token by token and in chunks (okf_delta_step, okf_delta_prompt), against 64 bits.

Tolerance (u = 2^-24), with unit keys and queries and beta <= 1, for which a token changes
a column of the state by no more than it decays it: each token adds to a column's
error, relative to the largest length M that the column or v had, the dot product's
K u, the decay's, correction's and update's 8 u; chunks of c tokens solve for theirs with sums of c
terms, twice.  Over m tokens: m (K + 2 c + 8) u M, and o the last dot product's K u M on top; c = 64 covers
any chunk here.  M bounds a single value.  16-bit outputs: half a step."""
import ctypes

import numpy as np
import pytest

import layer_oracle as lo

torch = pytest.importorskip("torch")
import chatokf_amd as ok  # noqa: E402
from test_attn import FAKE, TYPES, U, dev, fails, gpu, host, ints, starts  # noqa: E402

FAR, NAN = FAKE << 12, float("nan")
FORMS = ["step", "prompt"]


def calls(e, form):
    return {"step": e.delta_step, "prompt": e.delta_prompt}[form]


@pytest.fixture()
def detached():
    e = ok.Enc(-1)
    yield e
    e.close()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("over,status", [
    ({}, ok.OKF_E_NODEV), ({"type": ok.BF16}, ok.OKF_E_NODEV), ({"q": 0}, ok.OKF_E_ARG), ({"k": 0}, ok.OKF_E_ARG), ({"v": 0}, ok.OKF_E_ARG),
    ({"g": 0}, ok.OKF_E_ARG), ({"beta": 0}, ok.OKF_E_ARG), ({"out": 0}, ok.OKF_E_ARG), ({"start": 0}, ok.OKF_E_ARG), ({"type": ok.Q8_0}, ok.OKF_E_TYPE),
    ({"k_heads": 0}, ok.OKF_E_SHAPE), ({"v_heads": 3}, ok.OKF_E_SHAPE), ({"v_heads": 0}, ok.OKF_E_SHAPE), ({"v_heads": 65536}, ok.OKF_E_SHAPE),
    ({"k_dim": 24}, ok.OKF_E_SHAPE), ({"k_dim": 272}, ok.OKF_E_SHAPE), ({"v_dim": 8}, ok.OKF_E_SHAPE), ({"v_dim": 0}, ok.OKF_E_SHAPE),
    ({"n": 0}, ok.OKF_E_SHAPE), ({"seqs": 0}, ok.OKF_E_SHAPE), ({"n": 2 ** 31 - 1}, ok.OKF_E_SHAPE), ({"seqs": 2 ** 26, "slots": 2 ** 26}, ok.OKF_E_SHAPE),
    ({"slots": 1}, ok.OKF_E_SHAPE), ({"slots": 1, "slot": FAKE}, ok.OKF_E_NODEV), ({"q": FAKE + 8}, ok.OKF_E_SHAPE), ({"g": FAKE + 2}, ok.OKF_E_SHAPE),
    ({"beta": FAKE + 4}, ok.OKF_E_NODEV), ({"slot": FAKE + 2, "slots": 9}, ok.OKF_E_SHAPE), ({"state_in": FAR + 4}, ok.OKF_E_SHAPE),
    ({"state_out": FAR + 8}, ok.OKF_E_SHAPE), ({"strides": (127, 0, 0, 0)}, ok.OKF_E_SHAPE), ({"strides": (0, 130, 0, 0)}, ok.OKF_E_SHAPE),
    ({"strides": (0, 132, 0, 0)}, ok.OKF_E_NODEV), ({"strides": (0, 132, 0, 0), "type": ok.F16}, ok.OKF_E_SHAPE), ({"gate_strides": (3, 0)}, ok.OKF_E_SHAPE),
    ({"gate_strides": (5, 2 ** 41)}, ok.OKF_E_SHAPE), ({"gate_strides": (5, 9)}, ok.OKF_E_NODEV),
    # overlaps: a step's over v is fine, with another stride or a place in it not; over q, k or the gates never; columns of the same rows are
    ({"out": FAKE * 4}, {"step": ok.OKF_E_NODEV, "prompt": ok.OKF_E_ARG}), ({"out": FAKE * 4, "strides": (0, 0, 0, 516)}, ok.OKF_E_ARG), ({"out": FAKE * 4 + 16}, ok.OKF_E_ARG),
    ({"out": FAKE}, ok.OKF_E_ARG), ({"out": FAKE * 2}, ok.OKF_E_ARG), ({"out": FAKE * 8 - 16}, ok.OKF_E_ARG), ({"out": FAKE * 16 - 4080}, ok.OKF_E_ARG),
    ({"v": FAKE + 1024, "k": FAKE + 512, "out": FAKE + 3072, "strides": (1280,) * 4}, ok.OKF_E_NODEV),
    ({"v": FAKE + 1024, "k": FAKE + 512, "out": FAKE + 3056, "strides": (1280,) * 4}, ok.OKF_E_ARG),
    ({"state_in": FAR, "state_out": FAR}, ok.OKF_E_NODEV), ({"state_in": FAR, "state_out": FAR + 131072}, ok.OKF_E_ARG),
    ({"state_in": FAR, "state_out": FAR + 262144}, ok.OKF_E_NODEV), ({"state_out": FAKE * 32}, ok.OKF_E_ARG), ({"state_in": FAKE * 32}, ok.OKF_E_ARG),
    ({"state_out": FAKE}, ok.OKF_E_ARG), ({"state_out": FAKE * 2}, ok.OKF_E_ARG), ({"state_out": FAKE * 4}, ok.OKF_E_ARG),
    ({"state_out": FAKE * 8}, ok.OKF_E_ARG), ({"state_out": FAKE * 16}, ok.OKF_E_ARG), ({"state_in": FAKE * 4}, ok.OKF_E_NODEV)])
def test_refusals(detached, form, over, status):
    a = dict(q=FAKE, k=FAKE * 2, v=FAKE * 4, g=FAKE * 8, beta=FAKE * 16, out=FAKE * 32, start=FAKE, seqs=2, n=7, k_heads=2, v_heads=4, k_dim=64,
             v_dim=128)
    fails(lambda: calls(detached, form)(**{**a, **over}), status[form] if isinstance(status, dict) else status)


def test_reserve_refusals(detached):
    good = dict(n=100, seqs=2, k_heads=2, v_heads=4, k_dim=64, v_dim=128)
    fails(lambda: detached.delta_reserve(**good), ok.OKF_E_NODEV)
    fails(lambda: detached.delta_reserve(**good, type=ok.Q8_0), ok.OKF_E_TYPE)
    for bad in (dict(n=0), dict(n=2 ** 31 - 1), dict(seqs=0), dict(k_heads=0), dict(k_heads=3), dict(v_heads=0), dict(v_heads=65536, k_heads=1),
                dict(k_dim=40), dict(v_dim=0), dict(v_dim=512)):
        fails(lambda: detached.delta_reserve(**{**good, **bad}), ok.OKF_E_SHAPE)


# ------------------------------------------------------------------- results
class Case:
    """Inputs of packed sequences, on the GPU in their type, and as 64-bit values."""

    def __init__(self, t, KH, VH, DK, DV, lens, seed=0, slots=0, forget=None):
        rng = self.rng = np.random.default_rng(seed + 1000 * len(lens) + DK + DV)
        self.t, self.dims, self.lens, self.start = t, (KH, VH, DK, DV), lens, starts(lens)
        n = max(self.start[-1], 1)

        def unit(*shape):
            x = rng.standard_normal(shape) + 0.5 * rng.standard_normal(shape[1:])
            return (x / np.sqrt((x ** 2).sum(-1, keepdims=True)) * 0.999).astype(np.float32)
        self.q, self.k = (dev(unit(n, KH, DK), TYPES[t]) for _ in range(2))
        self.v = dev(rng.standard_normal((n, VH, DV)).astype(np.float32), TYPES[t])
        rate = np.exp(rng.uniform(np.log(1e-4), np.log(8), VH)) if forget is None else np.full(VH, forget)
        self.g = dev((-rate * rng.exponential(1, (n, VH))).astype(np.float32))
        self.beta = dev((1 / (1 + np.exp(-1.5 * rng.standard_normal((n, VH))))).astype(np.float32))
        self.slots = slots or len(lens)
        self.state = dev((0.3 * rng.standard_normal((self.slots, VH, DK, DV))).astype(np.float32))

    def want(self, i, state, scale):
        r = slice(self.start[i], self.start[i + 1])
        return lo.delta(*(host(x[r]) for x in (self.q, self.k, self.v, self.g, self.beta)), state, scale)

    def bounds(self, i, state, o, scale):
        """Of the state, and of o."""
        m, K = self.lens[i], self.dims[2]
        M = np.sqrt((state ** 2).sum(1)).max(initial=0) + np.abs(host(self.v[self.start[i]:self.start[i + 1]])).max(initial=0) * 2
        s = m * (K + 2 * 64 + 8) * U * M
        b = scale * (s + K * U * M)
        return s, b + (0 if self.t == "f32" else torch.finfo(TYPES[self.t]).eps / 2 * (np.abs(o) + b) + 2.0 ** -25)


def check(enc, form, c, state=True, keep=True, slot=None, inplace=False, over_v=False, scale=0.25):
    KH, VH, DK, DV = c.dims
    n = c.start[-1]
    o = c.v if over_v else torch.full((n + 2, VH, DV), 5.0, dtype=TYPES[c.t], device="cuda")
    was = host(c.state)
    out = c.state if inplace else torch.full_like(c.state, 9.0)
    left, refs = host(out), []
    for i in range(len(c.lens)):
        at = i if slot is None else slot[i]
        begin = was[at] if state and 0 <= at < c.slots else np.zeros((VH, DK, DV))
        refs.append((at, begin, *c.want(i, begin, scale)))
    calls(enc, form)(c.q, c.k, c.v, c.g, c.beta, o, ints(c.start), len(c.lens), max(n, 1), KH, VH, DK, DV, type=ok.BY_NAME[c.t], scale=scale,
                     state_in=c.state if state else None, state_out=out if keep else None, slot=None if slot is None else ints(slot), slots=c.slots)
    enc.sync()
    got, after = host(o), host(out)
    for i, (at, begin, ref, S) in enumerate(refs):
        s, b = c.bounds(i, begin, ref, scale)
        if c.lens[i]:
            assert (np.abs(got[c.start[i]:c.start[i + 1]] - ref) <= b).all(), (form, i, np.abs(got[c.start[i]:c.start[i + 1]] - ref).max(), np.max(b))
        if keep and 0 <= at < c.slots:
            assert np.abs(after[at] - S).max() <= s + (0 if c.lens[i] else 0), (form, i, np.abs(after[at] - S).max(), s)
            left[at] = after[at]
    assert np.array_equal(after, left)  # slots of no sequence
    assert over_v or (got[n:] == 5).all()
    return got, after


@gpu
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("KH,VH,DK,DV,lens", [
    (1, 1, 16, 16, [1]), (1, 2, 128, 128, [1, 1, 1]), (2, 4, 64, 128, [4, 2, 0, 5]), (1, 3, 96, 208, [31, 32, 33]), (2, 2, 80, 80, [64, 1, 65]),
    (1, 1, 256, 256, [40]), (1, 2, 240, 32, [7, 100]), (3, 3, 128, 64, [0, 0, 17]), (1, 1, 32, 48, [i * 7 % 11 for i in range(70)]),
    (1, 4, 128, 128, [200]), (1, 1, 112, 16, [129]), (1, 1, 160, 96, [33, 63]), (1, 1, 192, 144, [70]), (1, 1, 208, 112, [35])])
def test_delta(enc, form, t, KH, VH, DK, DV, lens):
    check(enc, form, Case(t, KH, VH, DK, DV, lens))
    check(enc, form, Case(t, KH, VH, DK, DV, lens, seed=1), state=False)
    check(enc, form, Case(t, KH, VH, DK, DV, lens, seed=2), inplace=True)


@gpu
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_places(enc, form, t):
    """States anywhere in a pool, slots outside it, nothing kept, o over v."""
    lens = [40, 3, 0, 1, 70]
    check(enc, form, Case(t, 1, 2, 64, 64, lens, slots=9), slot=[8, 0, 3, 5, 2])
    check(enc, form, Case(t, 1, 2, 64, 64, lens, slots=9), slot=[8, 0, 3, 5, 2], inplace=True)
    check(enc, form, Case(t, 1, 2, 64, 64, lens, slots=6), slot=[5, -1, 3, 6, 2 ** 31 - 1], inplace=True)
    check(enc, form, Case(t, 1, 2, 64, 64, lens, slots=6), slot=[5, 5, 5, 5, 0], keep=False)
    if form == "step":
        check(enc, form, Case(t, 1, 2, 64, 64, lens), over_v=True)


@gpu
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_strides(enc, form, t):
    """Queries, keys, values and the output as columns of the same rows, gates as columns of others."""
    KH, VH, DK, DV, lens = 2, 4, 64, 80, [50, 37]
    c = Case(t, KH, VH, DK, DV, lens)
    plain, state = check(enc, form, c)
    n, w = c.start[-1], (KH * DK, KH * DK, VH * DV, VH * DV)
    x = torch.full((n, sum(w) + 16), 3.0, dtype=TYPES[t], device="cuda")
    at = np.cumsum([0, *w])
    for i, y in enumerate((c.q, c.k, c.v)):
        x[:, at[i]:at[i + 1]] = y.reshape(n, -1)
    gates = torch.full((n, 2 * VH + 3), NAN, device="cuda")
    gates[:, 1:1 + VH], gates[:, 2 + VH:2 + 2 * VH] = c.g, c.beta
    out = torch.empty_like(c.state)
    calls(enc, form)(x, x[:, at[1]:], x[:, at[2]:], gates[:, 1:], gates[:, 2 + VH:], x[:, at[3]:], ints(c.start), 2, n, KH, VH, DK, DV,
                     type=ok.BY_NAME[t], scale=0.25, state_in=c.state, state_out=out, strides=(x.shape[1],) * 4, gate_strides=(gates.shape[1],) * 2)
    enc.sync()
    assert np.array_equal(host(x[:, at[3]:at[4]]).reshape(n, VH, DV), plain[:n]) and np.array_equal(host(out), state)
    assert np.array_equal(host(x[:, :at[1]]), host(c.q).reshape(n, -1)) and (host(x[:, at[4]:]) == 3).all()


@gpu
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("g", [float("-inf"), -1e4, -200.0, -88.0, 0.0])
def test_decays(enc, form, t, g):
    """A state cleared before a token (also of what came in its own chunk), nearly, and kept whole."""
    c = Case(t, 1, 2, 64, 64, [100, 33], forget=0.01)
    c.g[[0, 7, 8, 31, 32, 63, 90, 99, 100, 120]] = g
    check(enc, form, c)
    c.g[:] = g
    check(enc, form, c)


@gpu
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_keys_alike(enc, form, t):
    """All keys of a sequence the same, written whole: each token replaces what the one before left."""
    c = Case(t, 1, 1, 64, 32, [90], forget=0.0)
    c.k[:] = c.k[0].clone()
    c.beta[:] = 1
    check(enc, form, c)


@gpu
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bad", [NAN, float("inf")])
def test_what_comes_later_has_no_influence(enc, form, t, bad):
    """Values that are not finite, in any input: the tokens before, the other sequences and the other columns or heads are as ever."""
    for what in ("q", "k", "v", "g", "beta"):
        c = Case(t, 1, 2, 64, 64, [80, 40], seed=3)
        clean, state = check(enc, form, c)
        _, b = c.bounds(0, host(c.state)[0], clean[:80], 0.25)
        at, x = 45, getattr(c, what)
        if what == "v":
            x[at, 1, 5] = bad
        elif what in "qk":
            x[at, 0, 9] = bad
        else:
            x[at, 1] = bad
        o, out = torch.full((120, 2, 64), 5.0, dtype=TYPES[t], device="cuda"), torch.empty_like(c.state)
        calls(enc, form)(c.q, c.k, c.v, c.g, c.beta, o, ints(c.start), 2, 120, 1, 2, 64, 64, type=ok.BY_NAME[t], scale=0.25, state_in=c.state,
                         state_out=out)
        enc.sync()
        got, after = host(o), host(out)
        ref, S = c.want(0, host(c.state)[0], 0.25)
        fine = np.isfinite(ref)
        assert fine[:at].all() and not fine[at:].all()
        assert np.array_equal(np.isfinite(got[:80]), fine), what
        with np.errstate(invalid="ignore"):
            assert (np.abs(got[:80] - ref) <= b)[fine].all()
        assert np.array_equal(got[80:], clean[80:120]) and np.array_equal(after[1], state[1])
        assert np.array_equal(np.isfinite(after[0]), np.isfinite(S))
        c = None


@gpu
@pytest.mark.parametrize("form", FORMS)
def test_state_not_finite(enc, form):
    """A NaN in a state's column stays in it."""
    c = Case("f32", 1, 1, 64, 64, [50])
    _, state = check(enc, form, c)
    c.state[0, 0, 3, 7] = NAN
    out = torch.empty_like(c.state)
    calls(enc, form)(c.q, c.k, c.v, c.g, c.beta, torch.empty_like(c.v), ints(c.start), 1, 50, 1, 1, 64, 64, state_in=c.state, state_out=out, scale=0.25)
    enc.sync()
    bad = np.zeros(64, bool)
    bad[7] = True
    assert np.array_equal(np.isnan(host(out)).any((0, 1, 2)), bad)


@gpu
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("size", [1e-25, 1e25])
def test_sizes(enc, form, size):
    """Values and states far from one: the results scale with them."""
    c = Case("f32", 1, 2, 64, 64, [70])
    ref, S = c.want(0, host(c.state)[0], 0.25)
    s, b = c.bounds(0, host(c.state)[0], ref, 0.25)
    v, st = dev((host(c.v) * size).astype(np.float32)), dev((host(c.state) * size).astype(np.float32))
    o, out = torch.empty_like(v), torch.empty_like(st)
    calls(enc, form)(c.q, c.k, v, c.g, c.beta, o, ints(c.start), 1, 70, 1, 2, 64, 64, scale=0.25, state_in=st, state_out=out)
    enc.sync()
    assert (np.abs(host(o) / size - ref) <= b + 4 * U * np.abs(ref).max()).all() and np.abs(host(out)[0] / size - S).max() <= s + 4 * U * np.abs(S).max()


@gpu
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_in_parts(enc, t):
    """A sequence in one call, in chunks behind each other and in steps: the same within the bounds."""
    c = Case(t, 1, 2, 64, 80, [150])
    begin = host(c.state)
    ref, S = c.want(0, begin[0], 0.25)
    s, b = c.bounds(0, begin[0], ref, 0.25)
    o, at = torch.empty_like(c.v), 0
    for form, m in (("prompt", 40), ("step", 3), ("prompt", 1), ("prompt", 70), ("step", 1), ("prompt", 35)):
        r = slice(at, at + m)
        calls(enc, form)(c.q[r], c.k[r], c.v[r], c.g[r], c.beta[r], o[r], ints([0, m]), 1, m, 1, 2, 64, 80, type=ok.BY_NAME[t], scale=0.25,
                         state_in=c.state, state_out=c.state)
        at += m
    enc.sync()
    assert at == 150 and (np.abs(host(o) - ref) <= b).all() and np.abs(host(c.state)[0] - S).max() <= s


@gpu
@pytest.mark.parametrize("form", FORMS)
def test_starts_that_do_not_fit(enc, form):
    """Starts that leave the rows or decrease are clamped: nothing outside is read or written."""
    for start in ([-5, 20, 1000], [30, 30, 55], [20, 10, 40], [100, 200, 300]):
        c = Case("f32", 1, 1, 64, 64, [50])
        c.state = dev(np.zeros((2, 1, 64, 64), np.float32))
        o, out = torch.full((60, 1, 64), 5.0, device="cuda"), torch.full((2, 1, 64, 64), 9.0, device="cuda")
        calls(enc, form)(c.q, c.k, c.v, c.g, c.beta, o, ints(start), 2, 50, 1, 1, 64, 64, scale=0.25, state_out=out)
        enc.sync()
        got, written = host(o), np.zeros(60, bool)
        for i, (x, y) in enumerate(zip(start, start[1:])):
            x = min(max(x, 0), 50)
            y = min(max(y, x), 50)
            c.start, c.lens = [x, y], [y - x]
            ref, S = c.want(0, np.zeros((1, 64, 64)), 0.25)
            s, b = c.bounds(0, np.zeros((1, 64, 64)), ref, 0.25)
            assert (np.abs(got[x:y] - ref) <= b).all() and np.abs(host(out)[i] - S).max() <= s
            written[x:y] = True
        assert (got[~written] == 5).all()


@gpu
@pytest.mark.parametrize("form", FORMS)
def test_offsets_past_32_bits(enc, form):
    """A state past 4 GB of its pool, rows whose values' offsets pass 2^32."""
    VH, DK, DV, slots = 16, 128, 128, 4500   # (4.7 GB)
    pool = torch.empty(slots, VH, DK, DV, device="cuda")
    c = Case("f32", 1, VH, DK, DV, [2, 3])
    pool[[slots - 1, 7]] = c.state
    ref = [c.want(i, host(c.state)[i], 0.25) for i in range(2)]
    st = 1 << 30
    v = torch.empty(4 * st + 2 * VH * DV, dtype=torch.float32, device="cuda")
    rows = torch.as_strided(v, (5, 2, VH, DV), (st, VH * DV, DV, 1))
    rows[:, 0].copy_(c.v)
    calls(enc, form)(c.q, c.k, v, c.g, c.beta, v[VH * DV:], ints(c.start), 2, 5, 1, VH, DK, DV, scale=0.25, state_in=pool, state_out=pool,
                     slot=ints([slots - 1, 7]), slots=slots, strides=(0, 0, st, st))
    rows = rows[:, 1]
    enc.sync()
    for i, at in enumerate((slots - 1, 7)):
        s, b = c.bounds(i, host(c.state)[i], ref[i][0], 0.25)
        assert (np.abs(host(rows[c.start[i]:c.start[i + 1]].contiguous()) - ref[i][0]) <= b).all() and np.abs(host(pool[at]) - ref[i][1]).max() <= s


@gpu
@pytest.mark.parametrize("form", FORMS)
def test_captured(enc, form):
    """A captured call, replayed with other inputs between eager work: each replay as an eager call."""
    mine = ok.Enc(0)
    hip, vp = ctypes.CDLL("libamdhip64.so"), ctypes.c_void_p
    graph, exe, stream = vp(), vp(), vp(mine.stream)
    try:
        c = Case("f32", 1, 2, 64, 64, [70, 1, 40], seed=4)
        o, out, start = torch.empty_like(c.v), torch.empty_like(c.state), ints(c.start)
        mine.delta_reserve(111, 3, 1, 2, 64, 64)

        def step():
            calls(mine, form)(c.q, c.k, c.v, c.g, c.beta, o, start, 3, 111, 1, 2, 64, 64, scale=0.25, state_in=c.state, state_out=out)
        torch.cuda.synchronize()
        assert hip.hipStreamBeginCapture(stream, 0) == 0
        step()
        assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
        assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0) == 0
        for turn in range(4):
            c.v.mul_(1.5)
            start.copy_(ints([[0, 70, 71, 111], [0, 1, 80, 81], [0, 0, 111, 111], [5, 60, 100, 100]][turn]))
            o.fill_(5.0)
            out.fill_(9.0)
            torch.cuda.synchronize()
            assert hip.hipGraphLaunch(exe, stream) == 0
            mine.sync()
            got = o.clone(), out.clone()
            o.fill_(5.0)
            out.fill_(9.0)
            torch.cuda.synchronize()
            step()
            mine.sync()
            assert torch.equal(got[0], o) and torch.equal(got[1], out) and torch.isfinite(o).all()
        hip.hipGraphExecDestroy(exe)
        hip.hipGraphDestroy(graph)
    finally:
        mine.close()
