"""What the gated delta rule's calls launch, and the scratch that they take, on a HIP runtime that only records
(fake_hip.cpp); and on the GPU: prompts through scratch of few chunks, both widths of a step, the same bits again."""
import ctypes

import numpy as np
import pytest

import fakehip
import fakehip_delta

torch = pytest.importorskip("torch")
import chatokf_amd as ok  # noqa: E402
from test_attn import TYPES, gpu, host, ints  # noqa: E402
from test_delta import Case, calls, check  # noqa: E402

FIX = ["reserve", 1, 1, 1]


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    return fakehip.build(tmp_path_factory.mktemp("fake_hip"))


# (type, rows, sequences, key heads, value heads, widths)
PROMPTS = [("f32", 202, 2, 16, 16, 128, 128), ("bf16", 8192, 1, 16, 48, 128, 128), ("f16", 5000, 8, 16, 32, 128, 128), ("f32", 512, 1, 16, 48, 64, 128),
           ("f32", 17, 1, 1, 1, 16, 16), ("bf16", 40, 4000, 2, 6, 80, 96), ("f32", 100000, 3, 16, 48, 256, 128), ("f16", 70000, 70000, 1, 1, 32, 16)]


@pytest.mark.parametrize("call", PROMPTS)
@pytest.mark.parametrize("order", ["first", "last", "alone", "captured"])
def test_reserved_as_grown(fake, call, order):
    """The plan of a context that grows, with nothing allocated, also for fewer rows and sequences."""
    t, n, seqs, *dims = call
    calls_ = [call, (t, n, 1, *dims), (t, max(1, n // 3), seqs, *dims), (t, 1, 1, *dims)]
    reserve = ["delta_reserve", *call]
    before = {"first": [reserve, FIX], "last": [FIX, reserve], "alone": [reserve], "captured": [reserve, ["capture", 1]]}[order]
    got = fakehip_delta.run(fake, before + [["delta", "prompt", *c] for c in calls_])[len(before):]
    assert [s["status"] for s in got] == [0] * len(got)
    assert all(s["allocs"] == got[0]["allocs"] for s in got) and not got[0]["allocs"][-1][1]
    for c, g in zip(calls_, got):
        (free,) = fakehip_delta.run(fake, [["delta", "prompt", *c]])
        assert free["status"] == 0 and g["launches"] == free["launches"]


@pytest.mark.parametrize("t,n,seqs,KH,VH,DK,DV", PROMPTS)
def test_prompt_plan(fake, t, n, seqs, KH, VH, DK, DV):
    """Pairs of launches that go over all chunks, a wavefront for each two value heads of a key head and chunk,
    a workgroup for each 32 columns of a sequence's head; no more than 512 MB of scratch beside two sets of states."""
    (r,) = fakehip_delta.run(fake, [["delta", "prompt", t, n, seqs, KH, VH, DK, DV]])
    names = [x["name"] for x in r["launches"]]
    assert r["status"] == 0 and names == ["delta_prepare_kernel", "delta_scan_kernel"] * (len(names) // 2)
    waves = sum(x["grid"][0] * 4 for x in r["launches"][::2])
    need = min(n, n // 32 + seqs) * KH * ((VH // KH + 1) // 2)
    assert need <= waves < need + 4 * len(names) // 2
    assert all(x["grid"][0] == seqs * VH * ((DV // 16 + 1) // 2) for x in r["launches"][1::2])
    assert all(x["args"] == [(DK + 31) // 32] for x in r["launches"])
    assert r["allocs"][-1][0] <= (512 << 20) + 8 * VH * DK * DV and (len(names) > 2) == (n >= 70000)


def test_scratch_that_may_not_grow(fake):
    """Fewer chunks at a time; token by token where not even few fit; another call's reservation will do."""
    call = ["delta", "prompt", "f32", 3200, 1, 2, 4, 64, 64]
    r = fakehip_delta.run(fake, [["delta_reserve", "f32", 1000, 1, 2, 4, 64, 64], FIX, call])
    assert [x["name"] for x in r[2]["launches"]] == ["delta_prepare_kernel", "delta_scan_kernel"] * 4 and r[2]["allocs"] == r[0]["allocs"] + r[2]["allocs"][len(r[0]["allocs"]):]
    r = fakehip_delta.run(fake, [FIX, ["delta_reserve", "f32", 300, 1, 2, 4, 64, 64], call, ["delta", "prompt", "f32", 290, 1, 2, 4, 64, 64]])
    assert [[x["name"] for x in s["launches"]] for s in r[2:]] == [["delta_step_kernel"], ["delta_prepare_kernel", "delta_scan_kernel"]]
    r = fakehip_delta.run(fake, [["capture", 1], call])
    assert r[1]["status"] == 0 and [x["name"] for x in r[1]["launches"]] == ["delta_step_kernel"]
    r = fakehip_delta.run(fake, [["attn_reserve", 32, 128, 40, 8, 128, 1, 1], FIX, call])
    assert r[2]["status"] == 0 and r[2]["launches"][0]["name"] == "delta_prepare_kernel" and r[2]["allocs"] == r[1]["allocs"]


def test_scratch_that_cannot_be_had(fake):
    """A device without room for the chunks: fewer of them, or token by token, and no error."""
    call = ["delta", "prompt", "f32", 3200, 1, 2, 4, 64, 64]
    r = fakehip_delta.run(fake, [["fail_above", 4000], call, call])  # (101 chunks are 12 MB, a quarter of them 3)
    assert [s["status"] for s in r] == [0] * 3 and len(r[1]["launches"]) == 10 and r[2]["launches"] == r[1]["launches"]
    r = fakehip_delta.run(fake, [["fail_above", 1], call, ["delta", "step", "f32", 3200, 1, 2, 4, 64, 64]])
    assert [s["status"] for s in r] == [0] * 3 and r[1]["launches"] == r[2]["launches"]


@pytest.mark.parametrize("seqs", [1, 5, 30])
def test_few_rows_go_token_by_token(fake, seqs):
    r = fakehip_delta.run(fake, [["delta", "prompt", "bf16", n, seqs, 2, 4, 64, 64] for n in (1, 16, 17)] + [["delta", "step", "bf16", 16, seqs, 2, 4, 64, 64]])
    assert r[0]["launches"] == r[1]["launches"] == r[3]["launches"] and [x["name"] for x in r[2]["launches"]] == ["delta_prepare_kernel", "delta_scan_kernel"]


def test_reserved_while_captured(fake):
    r = fakehip_delta.run(fake, [["capture", 1], ["delta_reserve", "f32", 3200, 1, 2, 4, 64, 64]])
    assert r[1]["status"] == ok.OKF_E_SHAPE and r[1]["allocs"] == r[0]["allocs"]


@pytest.mark.parametrize("seqs,VH,DK,DV,args,grid", [(1, 48, 128, 128, [4, 8], 96), (32, 48, 128, 128, [8, 16], 1536), (5, 24, 96, 208, [4, 6], 390),
                                                     (1, 1, 16, 16, [4, 1], 1), (600, 4, 256, 16, [8, 32], 600), (64, 16, 64, 80, [8, 8], 768)])
def test_step_plan(fake, seqs, VH, DK, DV, args, grid):
    """16 columns a wavefront, 32 where that leaves eight a CU (of 256)."""
    (r,) = fakehip_delta.run(fake, [["delta", "step", "f32", seqs, seqs, 1, VH, DK, DV]])
    (x,) = r["launches"]
    assert (x["name"], x["args"], x["grid"][0]) == ("delta_step_kernel", args, grid)


@pytest.mark.parametrize("t,n,seqs,C,rows,wide", [("f32", 1, 1, 10240, 8, 4), ("bf16", 512, 1, 10240, 8, 8), ("bf16", 1000, 3, 10240, 16, 8),
                                                  ("bf16", 2000, 1, 10240, 24, 8), ("bf16", 7036, 4, 10240, 32, 8), ("f32", 409, 2, 10240, 8, 4),
                                                  ("f16", 500, 1, 2047, 8, 1), ("f32", 2 ** 31 - 256, 1, 16, 256, 4)])
def test_conv_plan(fake, t, n, seqs, C, rows, wide):
    """Rows a thread by the workgroups that they leave; 16 bytes of channels where rows begin and end with whole ones."""
    (r,) = fakehip_delta.run(fake, [["conv", t, n, seqs, C, 4]])
    (x,) = r["launches"]
    assert (x["name"], x["args"], x["grid"][1]) == ("conv_kernel", [4, wide], -(-C // (256 * wide)))
    assert x["grid"][0] == min(n, n // rows + seqs) + seqs


# ------------------------------------------------------------------ on the GPU
@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("KH,VH,DK,DV,lens", [(1, 2, 64, 64, [1300]), (2, 4, 80, 48, [0, 700, 1, 0, 33, 600, 0]), (1, 1, 128, 128, [20] * 60),
                                              (1, 3, 96, 32, [511, 0, 0, 513, 31, 32])])
def test_in_few_chunks(t, KH, VH, DK, DV, lens):
    """Sequences that begin, go on and end in different pairs of launches: the bits of one pair, also in place."""
    n, seqs = sum(lens), len(lens)
    big, small = ok.Enc(0), ok.Enc(0)
    try:
        small.delta_reserve(17 * 32, 1, KH, VH, DK, DV, ok.BY_NAME[t])  # (18 chunks at a time)
        small.reserve(1, 1, 1)
        out = []
        for e, inplace in ((big, False), (small, False), (small, True)):
            out.append(check(e, "prompt", Case(t, KH, VH, DK, DV, lens, seed=8), inplace=inplace))
        assert all(np.array_equal(x, y) for o in out[1:] for x, y in zip(out[0], o))
        check(small, "prompt", Case(t, KH, VH, DK, DV, lens, seed=9), state=False)
        check(small, "prompt", Case(t, KH, VH, DK, DV, lens, seed=9), keep=False)
        check(small, "prompt", Case(t, KH, VH, DK, DV, lens, seed=9, slots=seqs + 2), slot=[(seqs - i) % (seqs + 3) - 1 for i in range(seqs)])
    finally:
        big.close()
        small.close()


@gpu
def test_token_by_token_where_nothing_fits():
    mine = ok.Enc(0)
    try:
        mine.reserve(1, 1, 1)
        c = Case("f32", 1, 2, 64, 64, [600, 90])
        got = check(mine, "prompt", c)
        assert all(np.array_equal(x, y) for x, y in zip(got, check(mine, "step", c)))
    finally:
        mine.close()


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("KH,VH,DK,DV", [(16, 32, 16, 16), (8, 16, 80, 48), (4, 8, 240, 80), (8, 16, 128, 112), (16, 32, 64, 128)])
def test_wide_steps(enc, t, KH, VH, DK, DV):
    """Enough wavefronts for 32 columns each: widths that are and are not multiples of them; sequences in a pool, without rows, of several."""
    tiles = (DV + 31) // 32
    seqs = -(-8 * torch.cuda.get_device_properties(0).multi_processor_count // (VH * tiles)) + 1
    lens = [(1, 3, 0, 1)[i % 4] for i in range(seqs)]
    slot = [(i * 5 + 3) % (seqs + 4) for i in range(seqs)]
    if (seqs + 4) % 5 == 0:
        slot = list(range(2, seqs + 2))
    check(enc, "step", Case(t, KH, VH, DK, DV, lens))
    check(enc, "step", Case(t, KH, VH, DK, DV, lens, slots=seqs + 4), slot=slot, inplace=True, over_v=True)


@gpu
@pytest.mark.parametrize("KH,VH,DK,DV", [(2, 10, 64, 64), (1, 7, 48, 16), (4, 4, 128, 32)])
def test_many_value_heads_and_sequences(enc, KH, VH, DK, DV):
    """More value heads a key head than a wavefront prepares, odd ones; workgroups that are and are not a multiple of eight."""
    check(enc, "prompt", Case("bf16", KH, VH, DK, DV, [65, 3, 40]))
    check(enc, "prompt", Case("f32", KH, VH, DK, DV, [i % 5 * 9 for i in range(33)]))


@gpu
@pytest.mark.parametrize("form", ["step", "prompt"])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_same_bits(enc, form, t):
    c = Case(t, 2, 4, 128, 128, [300, 77, 1])
    first = check(enc, form, c)
    for _ in range(5):
        assert all(np.array_equal(x, y) for x, y in zip(first, check(enc, form, c)))


@gpu
def test_two_contexts(enc):
    """Calls of two contexts at once, each with its own scratch."""
    mine = ok.Enc(0)
    try:
        c = [Case("f32", 2, 4, 64, 64, [900, 50], seed=s) for s in (1, 2)]
        want = [check(enc, "prompt", x) for x in c]
        o, st = [[torch.empty_like(x.v) for x in c] for _ in range(2)], [[torch.empty_like(x.state) for x in c] for _ in range(2)]
        start = ints(c[0].start)
        torch.cuda.synchronize()
        for turn in range(2):
            for e, x, y, z in zip((enc, mine), c, o[turn], st[turn]):
                e.delta_prompt(x.q, x.k, x.v, x.g, x.beta, y, start, 2, 950, 2, 4, 64, 64, scale=0.25, state_in=x.state, state_out=z)
        enc.sync()
        mine.sync()
        for turn in range(2):
            for w, y, z in zip(want, o[turn], st[turn]):
                assert np.array_equal(w[0][:950], host(y)) and np.array_equal(w[1], host(z))
    finally:
        mine.close()


@gpu
def test_reserved_in_a_graph():
    """A prompt of several pairs of launches captured on fixed scratch, an eager call that uses the same scratch between the replays."""
    mine = ok.Enc(0)
    hip, vp = ctypes.CDLL("libamdhip64.so"), ctypes.c_void_p
    graph, exe, stream = vp(), vp(), vp(mine.stream)
    try:
        mine.delta_reserve(17 * 32, 1, 1, 2, 64, 64)
        mine.reserve(1, 1, 1)
        c, other = Case("f32", 1, 2, 64, 64, [1300, 20]), Case("f32", 1, 2, 64, 64, [700], seed=5)
        want = check(mine, "prompt", c)
        o, out, start = torch.empty_like(c.v), torch.empty_like(c.state), ints(c.start)
        torch.cuda.synchronize()
        assert hip.hipStreamBeginCapture(stream, 0) == 0
        calls(mine, "prompt")(c.q, c.k, c.v, c.g, c.beta, o, start, 2, 1320, 1, 2, 64, 64, scale=0.25, state_in=c.state, state_out=out)
        assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
        assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0) == 0
        for _ in range(3):
            o.fill_(5.0)
            out.fill_(9.0)
            torch.cuda.synchronize()
            assert hip.hipGraphLaunch(exe, stream) == 0
            check(mine, "prompt", other)
            assert np.array_equal(host(o), want[0][:1320]) and np.array_equal(host(out), want[1])
        hip.hipGraphExecDestroy(exe)
        hip.hipGraphDestroy(graph)
    finally:
        mine.close()
