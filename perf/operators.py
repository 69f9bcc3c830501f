"""The attention path of a program on top of this library, as timed cases.

Five operators around a paged KV cache that holds 8-bit codes with one fp32
scale for each block of 64 tokens and head:

* ``prompt``: causal attention over packed sequences of different lengths,
  grouped heads, an optional window; the queries are the last rows of their
  sequence (a first prompt, or a later chunk behind a cached prefix).
* ``append``: new tokens' keys and values quantized into the cache, then the
  end of every sequence read back as values (what a later chunk's attention
  over the prompt takes).
* ``decode``: the last few tokens of every sequence (one, or a verify pass of
  several) attend to the cache, with the attention weight that each cached
  token got added up where a program evicts by it.
* ``evict``: per sequence and head the first and the most recent tokens and
  those of the largest accumulated weight are moved to a smaller cache, which
  is read back as values.

Inputs are N(0, 1) with queries widened so that the softmax is neither flat
nor a single token; cached codes are N(0, 36) as int8 with scales around
1 / 36, so that cached keys and values are about N(0, 1) too.
"""
import random

import torch

own = False

BLOCK = 64                       # tokens of a cache block
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
MAX_FLOPS = 4.0 * 40 * 128 * 8192 * 8192 / 2   # what a drawn prompt may cost
MAX_CACHE = 32 * 8192 * 8 * 256                # bytes of codes that a drawn cache may hold


def listed():
    return [
        # a chat turn of two short messages in this library's own fp32 activations: the smallest prompt
        {"name": "prompt_f32_101", "kind": "prompt", "type": "f32", "heads": 16, "kv_heads": 8, "dim": 128, "seqs": 2,
         "longest": 101, "prefix": 0, "window": 0, "fused": False},
        # a batch of ragged prompts, read in place from a fused projection's rows
        {"name": "prompt_bf16_packed8", "kind": "prompt", "type": "bf16", "heads": 16, "kv_heads": 4, "dim": 128,
         "seqs": 8, "longest": 1111, "prefix": 0, "window": 0, "fused": True},
        # a document as one prompt (the most flops)
        {"name": "prompt_f16_8192", "kind": "prompt", "type": "f16", "heads": 40, "kv_heads": 8, "dim": 128, "seqs": 1,
         "longest": 8192, "prefix": 0, "window": 0, "fused": False},
        # a prompt chunk behind a cached prefix, wide heads and a sliding window
        {"name": "prompt_bf16_chunk512_window", "kind": "prompt", "type": "bf16", "heads": 20, "kv_heads": 4,
         "dim": 256, "seqs": 1, "longest": 512, "prefix": 3500, "window": 1024, "fused": False},
        # one decode step of a batch: a token for each sequence, and the block that it went to
        {"name": "append1_batch32", "kind": "append", "type": "f32", "heads": 8, "dim": 128, "seqs": 32, "longest": 1,
         "prefix": 4000, "read": 64, "out": "f32"},
        # a batch of ragged prompts into the cache and the whole of it read back for the next chunk
        {"name": "append_bf16_prompts4", "kind": "append", "type": "bf16", "heads": 8, "dim": 128, "seqs": 4,
         "longest": 2500, "prefix": 0, "read": 2500, "out": "bf16"},
        # one token of one chat: the smallest call
        {"name": "decode1_1999", "kind": "decode", "heads": 16, "kv_heads": 8, "dim": 128, "seqs": 1, "tokens": 1,
         "longest": 1999, "window": 0, "weights": False},
        # one token each for a batch of ragged chats
        {"name": "decode1_batch32", "kind": "decode", "heads": 40, "kv_heads": 8, "dim": 128, "seqs": 32, "tokens": 1,
         "longest": 8192, "window": 0, "weights": False},
        # four drafted tokens verified behind a long document, wide heads (the longest cache)
        {"name": "verify4_100003", "kind": "decode", "heads": 20, "kv_heads": 4, "dim": 256, "seqs": 1, "tokens": 4,
         "longest": 100003, "window": 0, "weights": False},
        # decode steps of a program that evicts: attention weights added up
        {"name": "decode1_weights_batch8", "kind": "decode", "heads": 16, "kv_heads": 8, "dim": 64, "seqs": 8,
         "tokens": 1, "longest": 16000, "window": 0, "weights": True},
        # one chat cut to its budget
        {"name": "evict_4096_to_1024", "kind": "evict", "heads": 8, "dim": 128, "seqs": 1, "longest": 4096,
         "keep": 1024, "sink": 4, "recent": 128},
        # a ragged batch cut to its budget, some of it shorter than that
        {"name": "evict_batch16_to_2000", "kind": "evict", "heads": 8, "dim": 128, "seqs": 16, "longest": 16000,
         "keep": 2000, "sink": 16, "recent": 500},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(("prompt", "prompt", "append", "decode", "decode", "decode", "evict"))
    kv, dim, seqs = rng.choice((1, 2, 4, 8)), rng.choice((64, 80, 96, 128, 128, 256)), _log(rng, 1, 32)
    heads = kv * rng.choice((1, 2, 4, 5, 8))
    if kind == "prompt":
        seqs, longest, prefix = _log(rng, 1, 16), _log(rng, 1, 4000), rng.choice((0, 0, _log(rng, 1, 4000)))
        while 4.0 * heads * dim * seqs * longest * (prefix + longest / 2) > MAX_FLOPS:
            longest, prefix = longest // 2 + 1, prefix // 2
        return {"kind": kind, "type": rng.choice(("f32", "f16", "bf16", "bf16")), "heads": heads, "kv_heads": kv,
                "dim": dim, "seqs": seqs, "longest": longest, "prefix": prefix,
                "window": rng.choice((0, 0, _log(rng, 16, 2000))), "fused": prefix == 0 and rng.random() < 0.5}
    if kind == "append":
        longest = rng.choice((1, _log(rng, 2, 8), _log(rng, 9, 2500)))
        longest, prefix = max(1, min(longest, 80000 // (seqs * kv))), _log(rng, 1, 4000)
        return {"kind": kind, "type": rng.choice(("f32", "f16", "bf16")), "heads": kv, "dim": dim, "seqs": seqs,
                "longest": longest, "prefix": prefix, "read": rng.choice((64, longest, longest + 100)),
                "out": rng.choice(("f32", "f16", "bf16"))}
    longest = max(1, min(_log(rng, 1, 100000), MAX_CACHE // (seqs * kv * 2 * dim)))
    if kind == "decode":
        return {"kind": kind, "heads": heads, "kv_heads": kv, "dim": dim, "seqs": seqs, "tokens": rng.choice((1, 1, 1, 2, 4, 5)),
                "longest": longest, "window": rng.choice((0, 0, 0, _log(rng, 16, 4000))), "weights": rng.random() < 0.4}
    longest = min(longest, 16000)
    keep = _log(rng, 1, max(1, longest // 2))
    sink = rng.randint(0, min(16, keep))
    return {"kind": kind, "heads": kv, "dim": dim, "seqs": min(seqs, 16), "longest": longest, "keep": keep, "sink": sink,
            "recent": rng.randint(0, keep - sink)}


def _lens(case):
    """The sequences' lengths: the longest first, the others spread down to a tenth of it."""
    rng, top = random.Random(case["seqs"] * 1000003 + case["longest"]), case["longest"]
    return [top] + [max(1, int(top * rng.uniform(0.1, 1.0))) for _ in range(case["seqs"] - 1)]


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _starts(lens):
    v = [0]
    for n in lens:
        v.append(v[-1] + n)
    return _ints(v)


def _cache(s, gen, heads, dim, lens, spare=0):
    """A cache whose sequences hold `lens` tokens, pages in random order; `spare`: pages left free for each sequence.

    k [page][head][token][dim], v [page][head][dim][slot of the token] (``_slot``)."""
    blocks = [(n + BLOCK - 1) // BLOCK for n in lens]
    stride = max(max(blocks), 1)
    pages = sum(blocks) + spare * len(lens)
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    table = torch.full((len(lens), stride), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(blocks):
        table[i, :n] = order[at:at + n]
        at += n
    shape = (pages, heads, BLOCK, dim)
    codes = lambda: torch.empty(pages * heads * BLOCK * dim, device="cuda").normal_(0, 36, generator=gen).round_().clamp_(-127, 127).to(torch.int8)  # noqa: E731
    s["k"], s["v"] = codes().view(shape), codes().view(pages, heads, dim, BLOCK)
    s["ks"] = (0.5 + torch.rand(pages, heads, device="cuda", generator=gen)) / 36
    s["vs"] = (0.5 + torch.rand(pages, heads, device="cuda", generator=gen)) / 36
    s["table"], s["stride"], s["pages"], s["free"] = table, stride, pages, order[at:]
    s["lens"], s["len"] = lens, _ints(lens)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, device="cuda", generator=gen)  # noqa: E731
    s, lens, D = {"case": case}, _lens(case), case["dim"]
    if case["kind"] == "prompt":
        H, KV, t = case["heads"], case["kv_heads"], TYPES[case["type"]]
        klens = [n + case["prefix"] for n in lens]
        nq, nk = sum(lens), sum(klens)
        s["q_start"], s["k_start"], s["mq"], s["mk"] = _starts(lens), _starts(klens), max(lens), max(klens)
        if case["fused"]:  # rows of one projection: queries, keys, values
            x = randn(nq, H + 2 * KV, D)
            x[:, :H] *= 2
            x = x.to(t)
            s["q"], s["kk"], s["vv"] = x[:, :H], x[:, H:H + KV], x[:, H + KV:]
        else:
            s["q"], s["kk"], s["vv"] = (2 * randn(nq, H, D)).to(t), randn(nk, KV, D).to(t), randn(nk, KV, D).to(t)
        s["o"] = torch.empty((nq, H, D), dtype=t, device="cuda")
    elif case["kind"] == "append":
        H, t = case["heads"], TYPES[case["type"]]
        full = [n + case["prefix"] - (i if case["prefix"] > 64 else 0) for i, n in enumerate(lens)]
        _cache(s, gen, H, D, full)
        s["new"], s["kn"], s["vn"] = lens, randn(sum(lens), H, D).to(t), (3 * randn(sum(lens), H, D)).to(t)
        s["start"] = _starts(lens)
        s["tail"] = [min(n, case["read"]) for n in full]
        s["tail_start"] = _starts(s["tail"])
        s["ko"], s["vo"] = (torch.empty((sum(s["tail"]), H, D), dtype=TYPES[case["out"]], device="cuda") for _ in range(2))
    elif case["kind"] == "decode":
        H, KV, T = case["heads"], case["kv_heads"], case["tokens"]
        _cache(s, gen, KV, D, lens)
        s["q"], s["o"] = 2 * randn(case["seqs"], T, H, D), torch.empty((case["seqs"], T, H, D), device="cuda")
        if case["weights"]:
            w = torch.rand((case["seqs"], KV, s["stride"] * BLOCK), device="cuda", generator=gen)
            s["w"], s["wo"] = w, torch.zeros_like(w)
    else:
        H = case["heads"]
        spare = (case["keep"] + BLOCK - 1) // BLOCK
        _cache(s, gen, H, D, lens, spare)
        s["to"] = s["free"].view(case["seqs"], spare).contiguous()
        w = torch.rand((case["seqs"], H, s["stride"] * BLOCK), device="cuda", generator=gen)
        s["w"] = (w * 4000).floor() / 256  # weights in steps: many are equal
        s["wo"] = torch.zeros((case["seqs"], H, spare * BLOCK), device="cuda")
        s["kept"] = torch.empty((case["seqs"], H, case["keep"]), dtype=torch.int32, device="cuda")
        s["len_to"] = torch.empty(case["seqs"], dtype=torch.int32, device="cuda")
        s["left"] = [min(n, case["keep"]) for n in lens]
        s["left_start"] = _starts(s["left"])
        s["ko"], s["vo"] = (torch.empty((sum(s["left"]), H, D), device="cuda") for _ in range(2))
    return s


# ------------------------------------------------------------- plain forms
def _slot(tok):
    """Where the value of a block's token stands in its row of 64."""
    return tok % 16 // 4 * 16 + tok // 16 * 4 + tok % 4


def _row_seq(start, n):
    """For each of n packed rows its sequence and its place there."""
    row = torch.arange(n, device="cuda")
    seq = torch.searchsorted(start[1:], row, right=True)
    return seq, row - start[seq]


def _softmax(sc, seen):
    """Weights of masked scores; a row that sees nothing weighs nothing."""
    sc = torch.where(seen, sc, -torch.inf)
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(torch.isinf(m), 0.0, m))
    return p / torch.clamp(p.sum(-1, keepdim=True), min=1e-37)


def _plain_prompt(s):
    c = s["case"]
    H, KV, D, S, mq, mk = c["heads"], c["kv_heads"], c["dim"], c["seqs"], s["mq"], s["mk"]
    G = H // KV
    nq, nk = s["q_start"].diff(), s["k_start"].diff()
    iq, ik = torch.arange(mq, device="cuda"), torch.arange(mk, device="cuda")
    q = s["q"][(s["q_start"][:-1, None] + iq).clamp(max=s["q"].shape[0] - 1)].float()
    k = s["kk"][(s["k_start"][:-1, None] + ik).clamp(max=s["kk"].shape[0] - 1)].float()
    v = s["vv"][(s["k_start"][:-1, None] + ik).clamp(max=s["vv"].shape[0] - 1)].float()
    q = q.view(S, mq, KV, G, D).permute(0, 2, 3, 1, 4).reshape(S * KV, G * mq, D)
    k = k.permute(0, 2, 3, 1).reshape(S * KV, D, mk)
    v = v.permute(0, 2, 1, 3).reshape(S * KV, mk, D)
    sc = torch.bmm(q, k).view(S, KV, G, mq, mk) * D ** -0.5
    at = (nk - nq)[:, None, None] + iq[:, None]
    seen = ik <= at
    if c["window"]:
        seen = seen & (ik > at - c["window"])
    p = _softmax(sc, seen[:, None, None])
    o = torch.bmm(p.view(S * KV, G * mq, mk), v).view(S, KV, G, mq, D)
    seq, i = _row_seq(s["q_start"], s["q"].shape[0])
    return o.permute(0, 3, 1, 2, 4)[seq, i].reshape(-1, H, D).to(s["o"].dtype)


def _values(s, table, seq, tok):
    """Keys and values of tokens `tok` of sequences `seq`, as fp32 [n][head][dim]."""
    page = table[seq, tok // BLOCK].long()
    at = tok % BLOCK
    return (s["k"][page, :, at].float() * s["ks"][page][:, :, None],
            s["v"][page, :, :, _slot(at)].float() * s["vs"][page][:, :, None])


def _plain_append(s):
    c = s["case"]
    n, out = s["kn"].shape[0], TYPES[c["out"]]
    seq, i = _row_seq(s["start"], n)
    old = s["len"] - s["start"].diff()             # tokens before
    tok = old[seq] + i
    page = s["table"][seq, tok // BLOCK].long()
    first = s["table"].gather(1, (old // BLOCK).clamp(max=s["stride"] - 1).long()[:, None])[:, 0].long()
    had = old % BLOCK                              # tokens that the first block held
    inside = (torch.arange(BLOCK, device="cuda") < had[:, None])[:, None]   # [seq][1][64]
    for name, x in (("k", s["kn"]), ("v", s["vn"])):
        codes, scale, x = s[name], s[name + "s"], x.double()
        top = torch.zeros(scale.shape, dtype=torch.float64, device="cuda")
        top.scatter_reduce_(0, page[:, None].expand(-1, x.shape[1]), x.abs().amax(2), "amax")
        top = (top / 127).float()
        before = torch.where((had > 0)[:, None], scale[first], 0.0)
        scale[page] = top[page]
        after = torch.maximum(before, top[first])
        scale[first] = torch.where((had > 0)[:, None], after, scale[first])
        ratio = (before.double() / after.clamp(min=1e-300).double())[:, :, None, None]
        block = codes[first]
        again = torch.round(block.double() * ratio).to(torch.int8)
        if name == "k":
            codes[first] = torch.where(inside[..., None], again, block)
        else:
            slot = _slot(torch.arange(BLOCK, device="cuda"))
            in_slots = torch.zeros_like(inside)
            in_slots[:, :, slot] = inside
            codes[first] = torch.where(in_slots[:, :, None], again, block)
        new = torch.round(x / scale[page].double().clamp(min=1e-300)[:, :, None]).to(torch.int8)
        if name == "k":
            codes[page, :, tok % BLOCK] = new
        else:
            codes[page, :, :, _slot(tok % BLOCK)] = new
    seq, i = _row_seq(s["tail_start"], s["ko"].shape[0])
    tok = (s["len"] - s["tail_start"].diff())[seq] + i
    k, v = _values(s, s["table"], seq, tok)
    return {"k": k.to(out), "v": v.to(out)}


def _plain_decode(s):
    c = s["case"]
    H, KV, D, B, T = c["heads"], c["kv_heads"], c["dim"], c["seqs"], c["tokens"]
    G, L = H // KV, s["stride"] * BLOCK
    page = s["table"].clamp(min=0).long()
    slot = _slot(torch.arange(BLOCK, device="cuda"))
    k = (s["k"][page].float() * s["ks"][page][..., None, None]).permute(0, 2, 4, 1, 3).reshape(B * KV, D, L)
    v = (s["v"][page][..., slot].float() * s["vs"][page][..., None, None]).permute(0, 2, 1, 4, 3).reshape(B * KV, L, D)
    q = s["q"].view(B, T, KV, G, D).permute(0, 2, 1, 3, 4).reshape(B * KV, T * G, D)
    sc = torch.bmm(q, k).view(B, KV, T, G, L) * D ** -0.5
    j = torch.arange(L, device="cuda")
    at = s["len"][:, None] - T + torch.arange(T, device="cuda")
    seen = j <= at[..., None]
    if c["window"]:
        seen = seen & (j > at[..., None] - c["window"])
    p = _softmax(sc, seen[:, None, :, None])
    o = torch.bmm(p.view(B * KV, T * G, L), v).view(B, KV, T, G, D).permute(0, 2, 1, 3, 4).reshape(B, T, H, D)
    if not c["weights"]:
        return o
    here = (j < s["len"][:, None])[:, None]
    return {"o": o, "w": torch.where(here, s["w"] + p.sum((2, 3)), s["wo"])}


def _plain_evict(s):
    c = s["case"]
    H, keep, B, L = c["heads"], c["keep"], c["seqs"], s["stride"] * BLOCK
    j, n = torch.arange(L, device="cuda"), s["len"][:, None]
    always = (j < torch.clamp(n, max=c["sink"])) | ((j >= n - c["recent"]) & (j < n)) | ((n <= keep) & (j < n))
    w = torch.where((always | (j >= n))[:, None], -torch.inf, s["w"])
    order = torch.sort(w, dim=2, descending=True, stable=True)[1]   # the largest first, the lowest index among equals
    rank = torch.empty_like(order).scatter_(2, order, j.expand_as(order).contiguous())
    keeps = always[:, None] | ((rank < keep - c["sink"] - c["recent"]) & (n > keep)[:, None] & (j < n)[:, None])
    N = (keep + BLOCK - 1) // BLOCK * BLOCK
    at = torch.where(keeps, j, L).sort(2).values
    at = torch.cat([at, torch.full((B, H, max(0, N - L)), L, device="cuda")], 2)[:, :, :N]
    here = at < L
    tok = torch.where(here, at, 0)
    page = s["table"].long().gather(1, (tok // BLOCK).view(B, -1)).view(B, H, N).clamp(min=0)
    h = torch.arange(H, device="cuda")[None, :, None]
    k, v = s["k"][page, h, tok % BLOCK], s["v"][page, h, :, _slot(tok % BLOCK)]
    new = []
    for codes, scale in ((k, s["ks"]), (v, s["vs"])):
        sc = torch.where(here, scale[page, h], 0.0)
        top = sc.view(B, H, -1, BLOCK).amax(3).repeat_interleave(BLOCK, 2)
        again = torch.round(codes.double() * (sc.double() / top.double().clamp(min=1e-300))[..., None])
        new.append((again.float() * top[..., None]).permute(0, 2, 1, 3))
    seq, i = _row_seq(s["left_start"], s["ko"].shape[0])
    return {"kept": torch.where(here, at, -1)[:, :, :keep].to(torch.int32), "len": torch.clamp(s["len"], max=keep),
            "w": torch.where(here, s["w"].gather(2, tok), 0.0), "k": new[0][seq, i], "v": new[1][seq, i]}


# ------------------------------------------------------- the library's calls
_ENC = None


def _own(s):
    """The calls of a program: one context for the process, plain handles on the tensors."""
    global _ENC
    import chatokf_amd as ok
    if _ENC is None:
        _ENC = ok.Enc(0)
    enc, c = _ENC, s["case"]
    kind, D = c["kind"], c["dim"]
    if kind == "prompt":
        H, KV = c["heads"], c["kv_heads"]
        enc.attn_prompt(s["q"], s["kk"], s["vv"], s["o"], s["q_start"], s["k_start"], c["seqs"], s["q"].shape[0],
                        s["kk"].shape[0], H, KV, D, type=ok.BY_NAME[c["type"]], scale=D ** -0.5, window=c["window"],
                        strides=[x.stride(0) for x in (s["q"], s["kk"], s["vv"], s["o"])])
        return s["o"]
    cache = ok.KVCache(s["k"], s["v"], s["ks"], s["vs"], s["pages"], s["k"].shape[1], D)
    seqs = ok.KVSeqs(s["table"], s["len"], c["seqs"], s["stride"])
    if kind == "append":
        enc.kv_append(cache, seqs, s["kn"], s["vn"], s["start"], s["kn"].shape[0], type=ok.BY_NAME[c["type"]])
        enc.kv_read(cache, seqs, s["ko"], s["vo"], s["tail_start"], s["ko"].shape[0], type=ok.BY_NAME[c["out"]])
        return {"k": s["ko"], "v": s["vo"]}
    if kind == "decode":
        if not c["weights"]:
            enc.attn_decode(cache, seqs, s["q"], s["o"], c["tokens"], c["heads"], D ** -0.5, window=c["window"])
            return s["o"]
        enc.attn_decode(cache, seqs, s["q"], s["o"], c["tokens"], c["heads"], D ** -0.5, window=c["window"],
                        w_in=s["w"], w_out=s["wo"], w_stride=s["stride"] * BLOCK)
        return {"o": s["o"], "w": s["wo"]}
    to = ok.KVSeqs(s["to"], s["len_to"], c["seqs"], s["to"].shape[1])
    enc.kv_evict(cache, seqs, cache, to, c["keep"], c["sink"], c["recent"], s["w"], s["stride"] * BLOCK, s["wo"],
                 s["wo"].shape[2], s["kept"])
    enc.kv_read(cache, to, s["ko"], s["vo"], s["left_start"], s["ko"].shape[0])
    return {"kept": s["kept"], "len": s["len_to"], "w": s["wo"], "k": s["ko"], "v": s["vo"]}


def run(state):
    if own:
        return _own(state)
    return {"prompt": _plain_prompt, "append": _plain_append, "decode": _plain_decode,
            "evict": _plain_evict}[state["case"]["kind"]](state)


# ------------------------------------------------------------------- work
def _pairs(first, n, window):
    """Query-key pairs of n queries whose first sees `first` + 1 keys."""
    if not window:
        return n * first + n * (n + 1) // 2
    full = max(0, min(n, window - first))          # queries whose keys the window does not cut
    return full * first + full * (full + 1) // 2 + (n - full) * window


def work(case):
    """Each input read once and each output written once; two products a query, key, head and dimension."""
    D, lens, k = case["dim"], _lens(case), case["kind"]
    if k == "prompt":
        H, KV, size = case["heads"], case["kv_heads"], 4 if case["type"] == "f32" else 2
        nq, nk = sum(lens), sum(n + (min(case["prefix"], case["window"]) if case["window"] else case["prefix"]) for n in lens)
        pairs = sum(_pairs(case["prefix"], n, case["window"]) for n in lens)
        return {"bytes": size * D * (2 * nq * H + 2 * nk * KV), "flops": 4.0 * D * H * pairs}
    if k == "append":
        H, size, out = case["heads"], 4 if case["type"] == "f32" else 2, 4 if case["out"] == "f32" else 2
        full = [n + case["prefix"] - (i if case["prefix"] > 64 else 0) for i, n in enumerate(lens)]
        n, r = sum(lens), sum(min(f, case["read"]) for f in full)
        return {"bytes": 2 * H * D * (n * (size + 1) + r * (1 + out)), "flops": 2.0 * H * D * (3 * n + r)}
    if k == "decode":
        H, KV, T = case["heads"], case["kv_heads"], case["tokens"]
        span = [min(n, case["window"] + T - 1) if case["window"] else n for n in lens]
        b = sum(span) * KV * 2 * D + sum((n + 63) // 64 for n in span) * KV * 8 + 8 * len(lens) * T * H * D
        return {"bytes": b + (8 * KV * sum(lens) if case["weights"] else 0), "flops": 4.0 * D * H * T * sum(span)}
    H = case["heads"]
    left = sum(min(n, case["keep"]) for n in lens)
    return {"bytes": H * (4 * sum(lens) + left * (4 + 4 + 4 * D + 8 * D)), "flops": H * (4.0 * sum(lens) + 6.0 * left * D)}


# ---------------------------------------------------------------- 64 bits
def _sure_blocks(s, b):
    """A sequence's dequantized cache in 64 bits, token by token: keys and values [head][token][dim]."""
    n = s["lens"][b]
    pages = [int(p) for p in s["table"][b, :(n + BLOCK - 1) // BLOCK].tolist()]
    k = s["k"][pages].double() * s["ks"][pages].double()[..., None, None]
    v = s["v"][pages].double() * s["vs"][pages].double()[..., None, None]
    H, D = k.shape[1], k.shape[3]
    v = v.view(-1, H, D, 4, 4, 4).permute(0, 1, 4, 3, 5, 2).reshape(-1, H, BLOCK, D)  # slot (g, t, i) -> token (t, g, i)
    return (x.transpose(0, 1).reshape(H, -1, D)[:, :n].contiguous() for x in (k, v))


def _sure_rows(q, k, v, at, window, scale, weights=None):
    """One head: queries [n][D] at positions `at` over k, v [m][D] in 64 bits; adds their weights to `weights`."""
    out, j = torch.zeros_like(q), torch.arange(k.shape[0], device="cuda")
    for r in range(0, q.shape[0], 1024):
        sc = torch.mm(q[r:r + 1024], k.t().contiguous()) * scale
        hide = j[None] > at[r:r + 1024, None]
        if window:
            hide |= j[None] <= at[r:r + 1024, None] - window
        sc.masked_fill_(hide, -torch.inf)
        e = torch.exp(sc - sc.logsumexp(1, keepdim=True)).masked_fill(hide, 0.0)
        if weights is not None:
            weights += e.sum(0)
        out[r:r + 1024] = torch.mm(e, v)
    return out


def _sure_codes(x, scale):
    return torch.round(x / scale) if scale > 0 else torch.zeros_like(x)


def exact(case, seed):
    s, D = prepare(case, seed), case["dim"]
    if case["kind"] == "prompt":
        H, G = case["heads"], case["heads"] // case["kv_heads"]
        o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        qs, ks = s["q_start"].tolist(), s["k_start"].tolist()
        for b in range(case["seqs"]):
            at = torch.arange(qs[b + 1] - qs[b], device="cuda") + (ks[b + 1] - ks[b]) - (qs[b + 1] - qs[b])
            for h in range(H):
                rows = slice(ks[b], ks[b + 1])
                o[qs[b]:qs[b + 1], h] = _sure_rows(s["q"][qs[b]:qs[b + 1], h].double(), s["kk"][rows, h // G].double(),
                                                   s["vv"][rows, h // G].double(), at, case["window"], D ** -0.5)
        return o
    if case["kind"] == "decode":
        G, T = case["heads"] // case["kv_heads"], case["tokens"]
        o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        w = s["wo"].double() if case["weights"] else None
        for b, n in enumerate(s["lens"]):
            k, v = _sure_blocks(s, b)
            at = torch.arange(n - T, n, device="cuda")
            for h in range(case["heads"]):
                got = torch.zeros(n, dtype=torch.float64, device="cuda")
                o[b, :, h] = _sure_rows(s["q"][b, :, h].double(), k[h // G], v[h // G], at, case["window"], D ** -0.5, got)
                if T > n:
                    o[b, :T - n, h] = 0
                    if case["weights"]:
                        got = got.nan_to_num(0.0)
                if w is not None:
                    w[b, h // G, :n] += got + (s["w"][b, h // G, :n].double() if h % G == 0 else 0.0)
        return {"o": o, "w": w} if case["weights"] else o
    if case["kind"] == "append":
        ks, vs = [], []
        for b, n in enumerate(s["lens"]):
            old = n - s["new"][b]
            first, lo = int(s["start"][b]), old // BLOCK * BLOCK
            k, v = _sure_blocks(s, b)
            for whole, x, scales in ((k, s["kn"], s["ks"]), (v, s["vn"], s["vs"])):
                whole[:, old:] = x[first:first + n - old].double().transpose(0, 1)
                for at in range(lo, n, BLOCK):
                    part, page = whole[:, at:min(n, at + BLOCK)], int(s["table"][b, at // BLOCK])
                    new = part[:, max(0, old - at):]
                    scale = (new.abs().amax((1, 2)) / 127).float().double()
                    if at < old:
                        was = scales[page].double()
                        scale = torch.maximum(scale, was)
                        held = torch.round(part[:, :old - at] / was[:, None, None])
                        part[:, :old - at] = torch.round(held * (was / scale)[:, None, None])
                        part[:, :old - at] *= scale[:, None, None]
                    new.copy_(torch.round(new / scale[:, None, None]) * scale[:, None, None])
            ks.append(k[:, n - s["tail"][b]:].transpose(0, 1))
            vs.append(v[:, n - s["tail"][b]:].transpose(0, 1))
        return {"k": torch.cat(ks), "v": torch.cat(vs)}
    ks, vs, w = [], [], s["wo"].double()
    for b, n in enumerate(s["lens"]):
        k, v = _sure_blocks(s, b)
        left = min(n, case["keep"])
        bk, bv = (torch.empty((left, case["heads"], D), dtype=torch.float64, device="cuda") for _ in range(2))
        pages = s["table"][b].long()
        got = s["w"][b, :, :n].cpu().tolist()
        for h in range(case["heads"]):
            keep = list(range(n))
            if n > left:
                inner = sorted(range(case["sink"], n - case["recent"]), key=lambda i: (-got[h][i], i))
                inner = inner[:case["keep"] - case["sink"] - case["recent"]]
                keep = sorted(list(range(case["sink"])) + inner + list(range(n - case["recent"], n)))
            tok = torch.tensor(keep, device="cuda")
            w[b, h, :left] = s["w"][b, h, tok].double()
            for whole, scales, out in ((k, s["ks"], bk), (v, s["vs"], bv)):
                sc = scales[pages[tok // BLOCK], h].double()
                codes = torch.round(whole[h, tok] / sc[:, None])
                for at in range(0, left, BLOCK):
                    top = sc[at:at + BLOCK].max()
                    out[at:at + BLOCK, h] = torch.round(codes[at:at + BLOCK] * (sc[at:at + BLOCK] / top)[:, None]) * top
        ks.append(bk)
        vs.append(bv)
    return {"kept": None, "len": None, "w": w, "k": torch.cat(ks), "v": torch.cat(vs)}
