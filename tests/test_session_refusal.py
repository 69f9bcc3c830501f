"""A chat that refuses new tokens keeps what it holds."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
import chatokf_amd as ok  # noqa: E402

gpu = pytest.mark.gpu


class Stub:
    """The library's calls that Chat makes for new tokens, recorded."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a, **k: self.calls.append(name)


@pytest.mark.parametrize("held,new,fits", [(150, 105, False), (96, 105, False), (50, 151, False), (0, 201, False),
                                           (150, 104, True), (150, 50, True), (50, 150, True), (96, 104, True)])
def test_eviction_only_for_what_fits(held, new, fits):
    """limit 200, keep 96: refused before anything is done, evicted only where the tokens fit afterwards."""
    from chatokf_amd.session import Chat
    chat = Chat.__new__(Chat)
    chat.limit, chat.keep, chat.sink, chat.recent, chat.at, chat.n = 200, 96, 2, 16, 0, held
    enc = Stub()
    chat.layer = type("Layer", (), {"enc": enc, "kv_heads": 1, "dim": 16})()
    chat.lens = torch.full((2, 1), held, dtype=torch.int32)
    chat.w, chat.kept = torch.ones(2, 1, 256), torch.zeros(1, 96, dtype=torch.int32)
    chat.cache, chat.seqs = None, [None, None]
    chat._starts = lambda n: torch.tensor([0, n], dtype=torch.int32)
    k = torch.zeros(new, 1, 16)
    if fits:
        chat._append(k, k)
        assert enc.calls == ["kv_evict"] * (held + new > 200) + ["kv_append"]
        assert chat.n == (held if held + new <= 200 else min(held, 96)) + new
    else:
        with pytest.raises(ValueError):
            chat._append(k, k)
        assert enc.calls == [] and (chat.n, chat.at) == (held, 0)
        assert (chat.lens == held).all() and (chat.w == 1).all()


@gpu
def test_refused_prompt_leaves_the_chat(enc):
    from chatokf_amd.session import Chat, Layer
    layer = Layer(enc, 64, 2, 1, 64)
    chat = Chat(layer, limit=200, keep=96, sink=2, recent=16)
    rng = np.random.default_rng(4)

    def rows(n):
        return torch.from_numpy(rng.standard_normal((n, 64)).astype(np.float32)).cuda()
    chat.prompt(rows(150))
    chat.step(rows(1))
    before = [x.clone() for x in (*chat.values(), chat.w)]
    for call in (chat.prompt, chat.step):
        with pytest.raises(ValueError):
            call(rows(105))
        assert (chat.n, chat.at) == (151, 0)
        after = (*chat.values(), chat.w)
        enc.sync()
        assert all(torch.equal(a, b) for a, b in zip(after, before))
    chat.prompt(rows(104))
    enc.sync()
    assert (chat.n, chat.at) == (200, 1)
