"""okf_kv_evict with one array of lengths, or of weights, for both sides: in place, against the
oracle; arrays that overlap in any other way are refused."""
import numpy as np
import pytest

import attn_oracle as ao

torch = pytest.importorskip("torch")
import chatokf_amd as ok  # noqa: E402
from test_attn import FAKE, Dev, dev, fails, fake_cache, fake_seqs, gpu, host, ints  # noqa: E402

NODEV, ARG = ok.OKF_E_NODEV, ok.OKF_E_ARG


@pytest.mark.parametrize("over,status", [
    ({}, NODEV), ({"to": {"lens": FAKE + 4}}, ARG), ({"to": {"lens": FAKE + 8}}, ARG), ({"to": {"lens": FAKE + 12}}, NODEV),
    ({"to": {"lens": FAKE - 8}}, ARG), ({"to": {"lens": FAKE - 12}}, NODEV),
    ({"wo": FAKE + 4}, ARG), ({"wo": FAKE - 4}, ARG), ({"wos": 100}, ARG), ({"wos": 129}, ARG),
    ({"wo": FAKE + 6 * 128 * 4}, NODEV), ({"wo": FAKE + (6 * 128 - 1) * 4}, ARG),        # 3 sequences x 2 heads
    ({"wo": FAKE - (5 * 128 + 100) * 4}, NODEV), ({"wo": FAKE - (5 * 128 + 99) * 4}, ARG),
    ({"ws": 256, "wo": FAKE + 128 * 4, "wos": 256}, NODEV),                              # row by row side by side
    ({"ws": 256, "wo": FAKE + 127 * 4, "wos": 256}, ARG), ({"ws": 256, "wo": FAKE + 157 * 4, "wos": 256}, ARG),
    ({"ws": 256, "wo": FAKE + 156 * 4, "wos": 256}, NODEV), ({"ws": 256, "wo": FAKE - 128 * 4, "wos": 256}, NODEV),
    ({"ws": 256, "wo": FAKE + 128 * 4, "wos": 257}, NODEV), ({"ws": 256, "wo": FAKE + 128 * 4, "wos": 250}, ARG)])
def test_overlap_refusals(over, status):
    """w: rows of 128 values read, of 100 written, six of each."""
    e = ok.Enc(-1)
    a = {**dict(to={}, ws=128, wo=FAKE, wos=128), **over}
    fails(lambda: e.kv_evict(fake_cache(), fake_seqs(), fake_cache(), fake_seqs(**a["to"]), 100, 4, 10, FAKE, a["ws"], a["wo"],
                             a["wos"], FAKE), status)
    e.close()


@gpu
@pytest.mark.parametrize("lens,heads,keep,sink,recent", [
    ([300, 100, 0, 4097], 8, 96, 4, 20), ([33000, 16385, 900], 4, 900, 3, 64), ([5000] * 16, 8, 64, 0, 0), ([20000], 2, 19000, 8, 8)])
@pytest.mark.parametrize("same_len,same_w", [(True, True), (True, False), (False, True)])
def test_evict_in_place(enc, lens, heads, keep, sink, recent, same_len, same_w):
    D, nb = 16, (keep + 63) // 64
    d = Dev(lens, heads, D, keep, spare=nb * len(lens))
    n = d.stride * 64
    w = (d.rng.integers(0, 300, (len(lens), heads, n)) / 8).astype(np.float32)
    to = np.array([[d.free.pop() for _ in range(nb)] for _ in lens], np.int32)
    dto, dw = dev(to), dev(w)
    new_len = d.dlen if same_len else ints([-9] * len(lens))
    wo, wos = (dw, n) if same_w else (torch.full((len(lens), heads, keep), 7.0, device="cuda"), keep)
    kept = torch.full((len(lens), heads, keep), -9, dtype=torch.int32, device="cuda")
    enc.kv_evict(d.cache, d.seqs, d.cache, ok.KVSeqs(dto, new_len, len(lens), nb), keep, sink, recent, dw, n, wo, wos, kept)
    enc.sync()
    gk, gv, gw, gkept = host(d.k), ao.Cache.tokens_of(host(d.v)), host(wo), host(kept)
    assert host(new_len).tolist() == [min(m, keep) for m in lens]
    for s, m in enumerate(lens):
        for h, (tok, ck, _, cv, _) in enumerate(d.c.evict(d.table[s], m, w[s], keep, sink, recent)):
            assert gkept[s, h].tolist() == tok + [-1] * (keep - len(tok))
            assert np.array_equal(gw[s, h, :len(tok)], w[s, h, tok].astype(np.float64))
            for b in range((len(tok) + 63) // 64):
                e = min(64, len(tok) - 64 * b)
                assert np.array_equal(gk[to[s, b], h, :e], ck[64 * b:64 * b + e])
                assert np.array_equal(gv[to[s, b], h, :e], cv[64 * b:64 * b + e])
            if same_w:  # (the rest of a row stays as it was)
                assert np.array_equal(gw[s, h, min(m, keep):], w[s, h, min(m, keep):].astype(np.float64))
