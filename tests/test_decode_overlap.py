"""okf_attn_decode with arrays that overlap: in place where that is right, else refused."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
import chatokf_amd as ok  # noqa: E402
from test_attn import FAKE, Dev, dev, fails, fake_cache, fake_seqs, gpu, host  # noqa: E402

NODEV, ARG = ok.OKF_E_NODEV, ok.OKF_E_ARG
FAR = FAKE * 16


@pytest.mark.parametrize("over,status", [
    ({"o": FAR}, NODEV), ({"o": FAKE}, NODEV), ({"o": FAKE, "wo": FAR}, NODEV), ({"o": FAKE + 16}, ARG), ({"o": FAKE - 16}, ARG),
    ({"o": FAKE + 3 * 8 * 64 * 4}, NODEV), ({"o": FAKE + 3 * 8 * 64 * 4 - 16}, ARG), ({"o": FAKE - 3 * 8 * 64 * 4}, NODEV),
    ({"o": FAR, "wi": FAR * 2, "wo": FAR * 2}, NODEV), ({"o": FAR, "wi": FAR * 2, "wo": FAR * 2 + 4}, ARG),
    ({"o": FAR, "wi": FAR * 2, "wo": FAR * 2 + 128 * 4}, ARG), ({"o": FAR, "wi": FAR * 2, "wo": FAR * 2 + 6 * 128 * 4}, NODEV),
    ({"o": FAR, "wi": FAR * 2, "wo": FAR * 2 + 128 * 4, "ws": 256}, NODEV),
    ({"o": FAR, "wi": FAR * 2, "wo": FAR * 2 + 127 * 4, "ws": 256}, ARG)])
def test_overlap_refusals(over, status):
    """Queries of 3 sequences x 8 heads of 64; weights in six rows of 128 values."""
    e = ok.Enc(-1)
    a = {**dict(wi=None, wo=None, ws=128), **over}
    fails(lambda: e.attn_decode(fake_cache(), fake_seqs(), FAKE, a["o"], 1, 8, 1.0, w_in=a["wi"], w_out=a["wo"], w_stride=a["ws"]), status)
    e.close()


@gpu
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("H,KV,D,T,lens", [(8, 2, 128, 1, [3000]), (40, 2, 64, 2, [300, 64, 1]), (4, 4, 256, 1, [50, 0]),
                                           (40, 1, 64, 1, [60] * 600)])
def test_output_over_the_queries(enc, H, KV, D, T, lens, weights):
    """With the weights from scores that are kept, and made again from the queries; split and (600 sequences) not."""
    d = Dev(lens, KV, D, H)
    q = dev(d.rng.standard_normal((len(lens), T, H, D)).astype(np.float32))
    o, w = torch.empty_like(q), [torch.zeros(len(lens), KV, d.stride * 64, device="cuda") if weights else None for _ in range(2)]
    for out, x in ((o, w[0]), (q, w[1])):
        enc.attn_decode(d.cache, d.seqs, q, out, T, H, 0.1, w_out=x, w_stride=d.stride * 64)
    enc.sync()
    err = np.abs(host(q) - host(o)).max()
    assert err == 0 or (weights and err <= 1e-6 * np.abs(host(o)).max())   # (in two splits there: sums in another order)
    assert not weights or np.abs(host(w[0]) - host(w[1])).max() <= 1e-6 * host(w[0]).max()
