"""okf_norm_rope_rows: outputs whose heads meet each other are refused, whatever lies between rows and between heads (CPU)."""
import itertools

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import chatokf_amd as ok  # noqa: E402
from test_attn import FAKE, fails  # noqa: E402

FAR = FAKE << 8


@pytest.fixture()
def detached():
    e = ok.Enc(-1)
    yield e
    e.close()


def call(e, **over):
    a = dict(pos=FAKE, n=4, q=FAKE, q_out=FAR, heads=8, k=FAKE * 2, k_out=FAR << 4, kv_heads=2, dim=64)
    e.norm_rope(ok.Rope(64), **{**a, **over})


@pytest.mark.parametrize("over,status", [
    # a head's width as the row stride: row r's head h + 1 is row r + 1's head h
    ({"strides": (0, 0, 64, 0)}, ok.OKF_E_ARG), ({"strides": (0, 0, 0, 64)}, ok.OKF_E_ARG), ({"strides": (0, 0, 64, 0), "type": ok.BF16}, ok.OKF_E_ARG),
    ({"strides": (64, 0, 64, 0), "q": FAR}, ok.OKF_E_ARG), ({"strides": (0, 64, 0, 64), "k": FAR << 4}, ok.OKF_E_ARG),
    # a head stride without the row stride that goes with it
    ({"head_strides": (0, 0, 128, 0)}, ok.OKF_E_ARG), ({"head_strides": (0, 0, 128, 0), "strides": (0, 0, 960, 0)}, ok.OKF_E_NODEV),
    ({"strides": (0, 0, 512, 0)}, ok.OKF_E_NODEV), ({"strides": (0, 0, 508, 0)}, ok.OKF_E_ARG),
    # planes of rows
    ({"strides": (0, 0, 64, 0), "head_strides": (0, 0, 256, 0)}, ok.OKF_E_NODEV), ({"strides": (0, 0, 64, 0), "head_strides": (0, 0, 252, 0)}, ok.OKF_E_ARG),
    ({"strides": (64, 0, 64, 0), "head_strides": (256, 0, 256, 0), "q": FAR}, ok.OKF_E_NODEV),
    # one row, one head: nothing to meet
    ({"strides": (0, 0, 64, 64), "n": 1}, ok.OKF_E_NODEV), ({"strides": (0, 0, 64, 0), "heads": 1}, ok.OKF_E_NODEV),
    # heads of rows between those of others
    ({"strides": (0, 0, 192, 0), "head_strides": (0, 0, 128, 0), "n": 2, "heads": 2}, ok.OKF_E_NODEV),
    ({"strides": (0, 0, 160, 0), "head_strides": (0, 0, 128, 0), "n": 2, "heads": 2}, ok.OKF_E_ARG),
    # inputs may repeat themselves
    ({"strides": (64, 64, 0, 0)}, ok.OKF_E_NODEV),
    # the largest strides and counts, and a last row 2^64 values past the first
    ({"strides": (0, 0, 1 << 40, 0), "head_strides": (0, 0, (1 << 40) - 4, 0), "n": 2 ** 24 + 1, "k": 0, "k_out": 0, "kv_heads": 0, "q_out": 1 << 60,
      "heads": 16}, ok.OKF_E_ARG),
    ({"strides": (0, 0, 64, 0), "head_strides": (0, 0, 1 << 40, 0), "n": 2 ** 31 - 256, "k": 0, "k_out": 0, "kv_heads": 0, "heads": 65535,
      "q_out": 1 << 60}, ok.OKF_E_NODEV),
    ({"strides": (0, 0, 1 << 40, 0), "head_strides": (0, 0, 1 << 40, 0), "n": 2 ** 31 - 256, "k": 0, "k_out": 0, "kv_heads": 0, "heads": 65535,
      "q_out": 1 << 60}, ok.OKF_E_ARG)])
def test_outputs_that_meet_themselves(detached, over, status):
    fails(lambda: call(detached, **over), status)


def test_all_strides(detached):
    """Every small layout: refused where two heads share a value, and only there."""
    dim, rng = 16, np.random.default_rng(0)
    cases = [(n, h, s, d) for n, h, s, d in itertools.product((1, 2, 3, 5), (1, 2, 3, 4), range(16, 100, 4), range(16, 100, 4))]
    seen = [0, 0]
    for i in rng.permutation(len(cases))[:2000]:
        n, heads, s, d = cases[i]
        at = (np.arange(n)[:, None, None] * s + np.arange(heads)[:, None] * d + np.arange(dim)).ravel()
        meet = len(np.unique(at)) < len(at)
        seen[meet] += 1
        fails(lambda: detached.norm_rope(ok.Rope(0), None, n, FAKE, FAR, heads, dim=dim, strides=(0, 0, s, 0), head_strides=(0, 0, d, 0)),
              ok.OKF_E_ARG if meet else ok.OKF_E_NODEV)
    assert min(seen) > 200
