"""What the attention calls launch, and the scratch that they take, on a HIP runtime that only
records (fake_hip.cpp); and on the GPU a context with reserved scratch against one whose scratch grows."""
import ctypes

import numpy as np
import pytest

import fakehip
import fakehip_attn
from test_attn import Dev, dev, fails, gpu, host

torch = pytest.importorskip("torch")
import chatokf_amd as ok  # noqa: E402


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    return fakehip.build(tmp_path_factory.mktemp("fake_hip"))


# ------------------------------------------------------------------ reserved scratch
# (sequences, stride, heads, kv heads, width, tokens, weights)
CALLS = [(1, 40, 4, 1, 64, 1, 1), (1, 1600, 20, 4, 256, 4, 0), (1, 1600, 20, 4, 256, 4, 1), (32, 128, 40, 8, 128, 1, 0),
         (32, 128, 40, 8, 128, 1, 1), (8, 250, 16, 8, 64, 1, 1), (3, 7, 5, 1, 80, 2, 1), (1, 32, 16, 8, 128, 1, 0),
         (5, 999, 24, 8, 96, 1, 1), (64, 300, 64, 8, 128, 1, 1), (1, 100000, 8, 8, 128, 2, 1), (600, 1, 40, 1, 64, 1, 1), (1200, 2, 40, 1, 64, 1, 1)]


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("order", ["first", "last", "alone", "captured"])
def test_reserved_as_grown(fake, call, order):
    """The plan of a context that grows, with nothing allocated, also for fewer sequences, tokens and pages."""
    seqs, stride, heads, kv, dim, tokens, w = call
    calls = [call, call[:6] + (0,), (1,) + call[1:], (seqs, max(1, stride // 3)) + call[2:], (max(1, seqs // 2),) + call[1:5] + (1, w),
             call + (100,), call + (0, True), (seqs, 1) + call[2:] + (0, True)]
    reserve, fix = ["attn_reserve", *call], ["reserve", 1, 1, 1]
    before = {"first": [reserve, fix], "last": [fix, reserve], "alone": [reserve], "captured": [reserve, ["capture", 1]]}[order]
    steps = [["decode", *c] for c in calls if w or not c[6]]
    got = fakehip_attn.run(fake, before + steps)[len(before):]
    assert [s["status"] for s in got] == [0] * len(got)
    assert all(s["allocs"] == got[0]["allocs"] for s in got) and not any(freed for _, freed in got[0]["allocs"][-1:])
    for step, g in zip(steps, got):
        (free,) = fakehip_attn.run(fake, [step])
        assert free["status"] == 0 and g["launches"] == free["launches"]


def test_reserve_refusals_and_size(fake):
    e = ok.Enc(-1)
    for args, status in (((1, 4, 8, 2, 64, 1), ok.OKF_E_NODEV), ((0, 4, 8, 2, 64, 1), ok.OKF_E_SHAPE), ((1, 0, 8, 2, 64, 1), ok.OKF_E_SHAPE),
                         ((1, 4, 7, 2, 64, 1), ok.OKF_E_SHAPE), ((1, 4, 8, 0, 64, 1), ok.OKF_E_SHAPE), ((1, 4, 8, 2, 72, 1), ok.OKF_E_SHAPE),
                         ((1, 4, 8, 2, 64, 0), ok.OKF_E_SHAPE), ((1, 4, 65536, 1, 64, 1), ok.OKF_E_SHAPE),
                         ((2 ** 31, 4, 8, 1, 64, 1), ok.OKF_E_SHAPE)):
        fails(lambda: e.attn_reserve(*args), status)
    e.close()
    # at most 256 MiB of scores, however long the table; none without weights; not while a graph is captured
    r = fakehip_attn.run(fake, [["attn_reserve", 1, 2 ** 32 - 1, 8, 8, 128, 1, 1], ["close"]])
    assert r[0]["status"] == 0 and (256 << 20) <= r[0]["allocs"][-1][0] < (300 << 20)
    r = fakehip_attn.run(fake, [["attn_reserve", 1, 2 ** 32 - 1, 8, 8, 128, 1, 0]])
    assert r[0]["status"] == 0 and r[0]["allocs"][-1][0] < (20 << 20)
    r = fakehip_attn.run(fake, [["capture", 1], ["attn_reserve", 1, 40, 8, 8, 128, 1, 1]])
    assert r[1]["status"] == ok.OKF_E_SHAPE and r[1]["allocs"] == r[0]["allocs"]


@gpu
@pytest.mark.parametrize("H,KV,D,T,lens", [(4, 1, 64, 1, [2500]), (24, 2, 128, 2, [900, 64, 3001]), (8, 4, 256, 1, [1500, 20])])
def test_reserved_gives_the_same_bits(H, KV, D, T, lens):
    d = Dev(lens, KV, D, H + T)
    q = dev(d.rng.standard_normal((len(lens), T, H, D)).astype(np.float32))
    out = []
    for how in ("grown", "reserved", "captured"):
        mine = ok.Enc(0)
        try:
            if how != "grown":
                mine.reserve(1, 1, 1)
                mine.attn_reserve(len(lens), d.stride, H, KV, D, T, True)
            o, w = torch.full(q.shape, float("nan"), device="cuda"), torch.zeros(len(lens), KV, d.stride * 64, device="cuda")

            def step():
                mine.attn_decode(d.cache, d.seqs, q, o, T, H, 0.1, w_in=w, w_out=w, w_stride=w.shape[2])
            if how != "captured":
                step()
                mine.sync()
                out.append((host(o), host(w)))
                continue
            hip, vp = ctypes.CDLL("libamdhip64.so"), ctypes.c_void_p
            graph, exe, stream = vp(), vp(), vp(mine.stream)
            torch.cuda.synchronize()
            assert hip.hipStreamBeginCapture(stream, 0) == 0
            step()
            assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
            assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0) == 0
            try:
                for _ in range(3):
                    w.zero_()
                    o.fill_(float("nan"))
                    torch.cuda.synchronize()
                    assert hip.hipGraphLaunch(exe, stream) == 0
                    mine.sync()
                    out.append((host(o), host(w)))
            finally:
                hip.hipGraphExecDestroy(exe)
                hip.hipGraphDestroy(graph)
        finally:
            mine.close()
    for o, w in out[1:]:
        assert np.array_equal(o, out[0][0]) and np.array_equal(w, out[0][1])


# --------------------------------------------------------------------------- plans
# Rows and key groups of a prompt's workgroups: 2 x 4 for few tiles of many keys, 2 x 2 up to two tiles a CU.
@pytest.mark.parametrize("t,seqs,n_q,n_k,heads,dim,window,shape", [
    ("bf16", 1, 64, 2064, 32, 128, 0, (2, 4)), ("bf16", 1, 64, 700, 32, 128, 0, (2, 2)), ("bf16", 1, 64, 2064, 32, 128, 500, (2, 2)),
    ("f16", 1, 1000, 1000, 32, 128, 0, (2, 2)), ("f16", 1, 1300, 1300, 32, 128, 0, (4, 1)), ("f16", 1, 8192, 8192, 40, 128, 0, (4, 1)),
    ("f32", 2, 202, 202, 16, 128, 0, (2, 2)), ("f32", 1, 50, 2000, 8, 64, 0, (2, 4)), ("f32", 1, 50, 2000, 8, 128, 0, (2, 2)),
    ("f32", 1, 50, 2000, 8, 256, 0, (4, 1)), ("bf16", 1, 512, 4012, 20, 256, 1024, (2, 2)), ("bf16", 1, 64, 2064, 32, 112, 0, (2, 2))])
def test_prompt_workgroups_plan(fake, t, seqs, n_q, n_k, heads, dim, window, shape):
    (r,) = fakehip_attn.run(fake, [["prompt", t, seqs, n_q, n_k, heads, heads // 4, dim, window]])
    (k,) = r["launches"]
    assert r["status"] == 0 and k["name"] == "attn_prompt_kernel"
    rg, kg = shape
    assert tuple(k["args"][-2:]) == shape and k["block"] == 64 * rg * kg and k["lds"] <= 160 * 1024
    tiles = min(n_q // (32 * rg) + seqs, n_q)
    assert tiles * heads <= k["grid"][0] < tiles * heads + 8 * 4


# Splits of a decode step: a workgroup for every four or eight pages until the CUs are full.
@pytest.mark.parametrize("call,splits,then", [
    ((1, 32, 16, 8, 128, 1, 0), 8, "attn_dec_join_kernel"), ((1, 4, 16, 8, 128, 1, 0), 1, None), ((1, 4, 16, 8, 128, 1, 1), 1, "attn_dec_sum_kernel"),
    ((32, 128, 40, 8, 128, 1, 0), 4, "attn_dec_join_kernel"), ((1, 1563, 20, 4, 256, 4, 0), 64, "attn_dec_join_kernel"),
    ((1, 1563, 20, 4, 256, 4, 1), 64, "attn_dec_weights_kernel"), ((8, 250, 16, 8, 64, 1, 1), 16, "attn_dec_sum_kernel"),
    ((1, 200000, 8, 8, 128, 4, 1), 64, "attn_dec_weights_kernel")])   # (scores of more than 256 MB are not kept)
def test_decode_plan(fake, call, splits, then):
    seqs, stride, heads, kv, dim, tokens, w = call
    (r,) = fakehip_attn.run(fake, [["decode", *call]])
    assert r["status"] == 0
    k, *rest = r["launches"]
    rows = tokens * (heads // kv)
    assert k["name"] == "attn_dec_kernel" and k["args"] == [(dim + 63) // 64, 2 if rows > 16 else 1]
    assert k["grid"][0] == -(-seqs * kv * splits // 8) * 8 * -(-rows // (32 if rows > 16 else 16))
    assert [v["name"] for v in rest] == ([then] if then else [])


# o over q: written by the join behind the launch that reads q again for the weights.
@pytest.mark.parametrize("call,names", [
    ((600, 1, 40, 1, 64, 1, 1), ["attn_dec_kernel", "attn_dec_weights_kernel", "attn_dec_join_kernel"]),
    ((1, 1563, 20, 4, 256, 4, 1), ["attn_dec_kernel", "attn_dec_weights_kernel", "attn_dec_join_kernel"]),
    ((8, 250, 16, 8, 64, 1, 1), ["attn_dec_kernel", "attn_dec_sum_kernel"]), ((1, 4, 16, 8, 128, 1, 0), ["attn_dec_kernel"])])
def test_decode_over_its_queries(fake, call, names):
    (r,) = fakehip_attn.run(fake, [["decode", *call, 0, True]])
    assert r["status"] == 0 and [v["name"] for v in r["launches"]] == names
    rows, base = call[5] * call[2] // call[3], call[0] * call[3]
    if "attn_dec_join_kernel" in names:
        assert r["launches"][0]["grid"][0] >= 2 * base * -(-rows // (32 if rows > 16 else 16))
        assert r["launches"][1]["grid"][0] == base * max(1, min(1024 // base, -(-call[1] // 4))) and r["launches"][2]["grid"][0] == base * rows
