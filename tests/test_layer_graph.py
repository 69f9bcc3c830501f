"""A decode step of the gated delta rule's layer and one of an attention layer's rotation as captured graphs: each
replay, with other inputs, positions, sequences' lengths and eager calls between, is the eager step bit for bit."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import chatokf_amd as ok  # noqa: E402
from test_attn import TYPES, dev, gpu, ints  # noqa: E402


@gpu
@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("seqs,KH,VH,DK,DV,W", [(1, 2, 4, 64, 64, 4), (5, 1, 3, 80, 48, 2), (40, 16, 32, 64, 64, 8)])
def test_step(t, seqs, KH, VH, DK, DV, W):
    mine = ok.Enc(0)
    hip, vp = ctypes.CDLL("libamdhip64.so"), ctypes.c_void_p
    graph, exe, stream = vp(), vp(), vp(mine.stream)
    rng, T = np.random.default_rng(seqs + DK), TYPES[t]
    keys, C, n, slots = KH * DK, 2 * KH * DK + VH * DV, 2 * seqs, seqs + 2

    def normal(*shape, to=torch.float32):
        return dev(rng.standard_normal(shape).astype(np.float32), to)
    try:
        x, w = normal(n, C, to=T), normal(C, W)
        hold, state = normal(slots, W - 1, C, to=T), 0.3 * normal(slots, VH, DK, DV)
        start, slot, pos = ints([0] * (seqs + 1)), ints([0] * seqs), ints([0] * n)
        y, o, q = torch.empty_like(x), torch.empty((n, VH, DV), dtype=T, device="cuda"), torch.empty((n, KH, DK), dtype=T, device="cuda")
        g, beta, unit = -torch.rand(n, VH, device="cuda"), torch.rand(n, VH, device="cuda"), torch.full((DK,), DK ** -0.5, device="cuda")

        def step():
            kind = ok.BY_NAME[t]
            mine.conv(x, w, y, start, seqs, n, C, W, type=kind, silu=True, state_in=hold, state_out=hold, slot=slot, slots=slots)
            mine.norm_rope(ok.Rope(0), None, n, y, y, KH, y[:, keys:], y[:, keys:], KH, DK, type=kind, q_norm=unit, k_norm=unit, eps=1e-6 / DK,
                           strides=(C,) * 4)
            mine.norm_rope(ok.Rope(DK // 2), pos, n, y, q, KH, dim=DK, type=kind, strides=(C, 0, 0, 0))
            mine.delta_step(y, y[:, keys:], y[:, 2 * keys:], g, beta, o, start, seqs, n, KH, VH, DK, DV, type=kind, scale=DK ** -0.5,
                            state_in=state, state_out=state, slot=slot, slots=slots, strides=(C, C, C, 0))

        def everything():
            return [v.clone() for v in (y[:rows], q, o[:rows], hold, state)]
        torch.cuda.synchronize()
        assert hip.hipStreamBeginCapture(stream, 0) == 0
        step()
        assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
        assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0) == 0
        for turn in range(4):
            lens = rng.integers(0, 3, seqs)
            rows = int(lens.sum())
            start.copy_(ints([0, *np.cumsum(lens)]))
            slot.copy_(ints(rng.permutation(slots)[:seqs]))
            pos.copy_(ints(rng.integers(0, 10 ** 6, n)))
            x.copy_(normal(n, C, to=T))
            for v in (y, o, q):
                v.zero_()
            before = hold.clone(), state.clone()
            torch.cuda.synchronize()
            assert hip.hipGraphLaunch(exe, stream) == 0
            mine.sync()
            got = everything()
            hold.copy_(before[0])
            state.copy_(before[1])
            for v in (y, o, q):
                v.zero_()
            torch.cuda.synchronize()
            step()
            mine.sync()
            for a, b in zip(got, everything()):
                assert torch.equal(a, b) and torch.isfinite(a).all()
        hip.hipGraphExecDestroy(exe)
        hip.hipGraphDestroy(graph)
    finally:
        mine.close()
