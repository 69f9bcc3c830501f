"""A chat through prompt, chunk, steps and eviction (chatokf_amd/session.py): each output against
attention in 64 bits over the values that the cache reads back."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
import attn_oracle as ao  # noqa: E402
import chatokf_amd as ok  # noqa: E402

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (6, 3, 80)])
def test_chat(enc, heads, kv, dim):
    from chatokf_amd.session import Chat, Layer
    K = 256
    layer = Layer(enc, K, heads, kv, dim)
    chat = Chat(layer, limit=200, keep=96, sink=2, recent=16)
    rng = np.random.default_rng(3)
    seen = {}
    plain = layer.output
    layer.output = lambda a: plain(seen.setdefault("a", a))  # (the attention's rows, before their projection)

    def check(call, n):
        x = torch.from_numpy(rng.standard_normal((n, K)).astype(np.float32)).cuda()
        seen.clear()
        y = call(x)
        enc.sync()
        assert y.shape == (n, K) and torch.isfinite(y).all()
        first = chat.n == n  # (a first prompt attends to its own values, not to the cache's)
        q, k, v = layer.project(x)
        if not first:
            k, v = chat.values()
        enc.sync()
        q, k, v, a = (t.double().cpu().numpy() for t in (q, k, v, seen["a"]))
        at = np.arange(chat.n - n, chat.n)
        big = np.sqrt((q ** 2).sum(-1)).max() * np.sqrt((k ** 2).sum(-1)).max() * dim ** -0.5
        bound = (2 * (dim + 4) * big + 2 * chat.n + 16) * 2.0 ** -24 * np.abs(v).max()  # (as in test_attn.py)
        w = np.zeros((kv, chat.n))
        for h in range(heads):
            ref, p = ao.attend(q[:, h], k[:, h // (heads // kv)], v[:, h // (heads // kv)], at, 0, dim ** -0.5)
            assert np.abs(a[:, h] - ref).max() <= bound
            w[h // (heads // kv)] += p.sum(0)
        return w, bound / np.abs(v).max()

    check(chat.prompt, 90)
    check(chat.prompt, 70)
    assert chat.n == 160
    total, rel = np.zeros((kv, 200)), 0.0
    for n in (1, 3, 1, 1):
        w, r = check(chat.step, n)
        total[:, :w.shape[1]] += w
        rel += r * n * (heads // kv)
    assert np.abs(chat.w[chat.at].double().cpu().numpy()[:, :200] - total).max() <= 2 * rel
    check(chat.prompt, 40)   # does not fit: cut to 96 first
    assert chat.n == 136 and chat.at == 1
    kept = chat.kept.cpu().numpy()
    for h in range(kv):
        assert kept[h, :2].tolist() == [0, 1] and kept[h, -16:].tolist() == list(range(150, 166))
        assert (np.diff(kept[h]) > 0).all()
        inner = total[h, 2:150]
        assert total[h, kept[h, 2:-16]].min() >= np.sort(inner)[::-1][77] - 4 * rel  # the 78 largest
    assert (chat.w[1].cpu().numpy()[:, 96:136] == 0).all()
    check(chat.step, 1)


@gpu
def test_chat_that_does_not_fit(enc):
    from chatokf_amd.session import Chat, Layer
    layer = Layer(enc, 64, 2, 1, 64)
    chat = Chat(layer, limit=64, keep=32, sink=1, recent=8)
    with pytest.raises(ValueError):
        chat.prompt(torch.zeros(65, 64, device="cuda"))


@gpu
def test_decode_on_reserved_scratch():
    """With scratch that may not grow: fewer splits, the same result; sums of weights that do not fit are refused."""
    mine = ok.Enc(0)
    try:
        mine.reserve(1, 1, 1)
        c = ok.KVCache.new(40, 1, 64)
        rng = np.random.default_rng(5)
        n = 2500
        x = [torch.from_numpy(rng.standard_normal((n, 1, 64)).astype(np.float32)).cuda() for _ in range(2)]
        table, lens = torch.arange(40, dtype=torch.int32, device="cuda"), torch.tensor([n], dtype=torch.int32, device="cuda")
        seqs = ok.KVSeqs(table, lens, 1, 40)
        mine.kv_append(c, seqs, *x, torch.tensor([0, n], dtype=torch.int32, device="cuda"), n)
        q = torch.from_numpy(rng.standard_normal((1, 1, 4, 64)).astype(np.float32)).cuda()
        o, w = torch.empty_like(q), torch.zeros(1, 1, 2560, device="cuda")
        mine.attn_decode(c, seqs, q, o, 1, 4, 0.125)
        with pytest.raises(ok.OkfError) as e:
            mine.attn_decode(c, seqs, q, o, 1, 4, 0.125, w_out=w, w_stride=2560)
        assert e.value.status == ok.OKF_E_SHAPE
        k, v = torch.empty(n, 1, 64, device="cuda"), torch.empty(n, 1, 64, device="cuda")
        mine.kv_read(c, seqs, k, v, torch.tensor([0, n], dtype=torch.int32, device="cuda"), n)
        mine.sync()
        q, k, v, o = (t.double().cpu().numpy() for t in (q, k, v, o))
        ref = np.stack([ao.attend(q[0, :, h], k[:, 0], v[:, 0], [n - 1], 0, 0.125)[0] for h in range(4)], 1)[0]
        big = np.sqrt((q ** 2).sum(-1)).max() * np.sqrt((k ** 2).sum(-1)).max() * 0.125
        assert np.abs(o[0, 0] - ref).max() <= (2 * 68 * big + 2 * n + 16) * 2.0 ** -24 * np.abs(v).max()
    finally:
        mine.close()
