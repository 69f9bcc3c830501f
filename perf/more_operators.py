"""What a hybrid model's layers compute around their projections, as timed cases.

Four operators.  One stands in front of attention and of the delta rule, two
are the delta rule's layer:

* ``rope``: the norms of queries and keys for each head and the rotation by
  their positions (a head's halves or its neighbours as pairs, the whole head or
  its first part, frequencies as they are, divided, or scaled for long contexts).
* ``conv``: the short causal convolution of each channel over packed sequences,
  with SiLU; a sequence's last inputs are its state.
* ``delta``: the gated delta rule over packed sequences of many tokens (a
  prompt, or a chunk behind one): per value head a matrix state S that each
  token decays, corrects and reads.
* ``step``: the same for the few tokens of a decode step or a verify pass, with
  the sequences' states anywhere in a pool.

Queries and keys of the delta rule are unit vectors with a common part (as they
come out of a norm behind a SiLU), decays are spread from heads that forget
within a token to ones that keep thousands.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CHUNK = 64                                   # tokens of the plain form's chunks
MAX_ROPE = 8192 * 48 * 128                   # values that a drawn rotation may have
MAX_CONV = 8192 * 10240                      # values that a drawn convolution may have
MAX_DELTA = 8192 * 48 * 128 * 128            # tokens x state values of a drawn delta rule
MAX_STATES = 32 * 48 * 128 * 128             # state values of a drawn step


def listed():
    return [
        # one token of one chat: queries and keys between their projections and the cache (the smallest call)
        {"name": "rope_f32_1", "kind": "rope", "type": "f32", "heads": 16, "kv_heads": 8, "dim": 128, "rot": 128, "pairs": False,
         "norm": True, "seqs": 1, "longest": 1, "first": 1999, "scaling": "none", "fused": False},
        # a batch of ragged prompts in place in a fused projection's rows: neighbours as pairs, a quarter of wide heads, divided frequencies
        {"name": "rope_f16_packed8_part", "kind": "rope", "type": "f16", "heads": 16, "kv_heads": 4, "dim": 256, "rot": 64,
         "pairs": True, "norm": True, "seqs": 8, "longest": 1111, "first": 0, "scaling": "divided", "fused": True},
        # a chunk of a long document, positions scaled past the context that the model was trained on (the most bytes)
        {"name": "rope_bf16_8192_far", "kind": "rope", "type": "bf16", "heads": 40, "kv_heads": 8, "dim": 128, "rot": 128, "pairs": False,
         "norm": True, "seqs": 1, "longest": 8192, "first": 100003, "scaling": "yarn", "fused": False},
        # a decode step of a batch: a token each, every sequence's last inputs from its state
        {"name": "conv_f32_batch32", "kind": "conv", "type": "f32", "channels": 10240, "width": 4, "seqs": 32, "longest": 1, "bias": False},
        # ragged prompts through the convolution
        {"name": "conv_bf16_prompts4", "kind": "conv", "type": "bf16", "channels": 10240, "width": 4, "seqs": 4, "longest": 2500, "bias": True},
        # a chat turn of two short messages in this library's own fp32 activations
        {"name": "delta_f32_101", "kind": "delta", "type": "f32", "k_heads": 16, "v_heads": 16, "k_dim": 128, "v_dim": 128, "seqs": 2,
         "longest": 101, "state": False},
        # a batch of ragged prompts
        {"name": "delta_bf16_packed8", "kind": "delta", "type": "bf16", "k_heads": 16, "v_heads": 32, "k_dim": 128, "v_dim": 128, "seqs": 8,
         "longest": 1111, "state": False},
        # a prompt chunk behind what a chat holds already, fp32, narrow keys
        {"name": "delta_f32_chunk512", "kind": "delta", "type": "f32", "k_heads": 16, "v_heads": 48, "k_dim": 64, "v_dim": 128, "seqs": 1,
         "longest": 512, "state": True},
        # a document as one prompt (the most flops)
        {"name": "delta_bf16_8192", "kind": "delta", "type": "bf16", "k_heads": 16, "v_heads": 48, "k_dim": 128, "v_dim": 128, "seqs": 1,
         "longest": 8192, "state": True},
        # one token of one chat
        {"name": "step1", "kind": "step", "type": "f32", "k_heads": 16, "v_heads": 48, "k_dim": 128, "v_dim": 128, "seqs": 1, "tokens": 1,
         "spare": 0},
        # one token each for a batch whose states lie anywhere in a pool
        {"name": "step1_batch32", "kind": "step", "type": "f32", "k_heads": 16, "v_heads": 48, "k_dim": 128, "v_dim": 128, "seqs": 32,
         "tokens": 1, "spare": 8},
        # four drafted tokens of a few chats verified, odd widths
        {"name": "verify4_batch5", "kind": "step", "type": "bf16", "k_heads": 8, "v_heads": 24, "k_dim": 96, "v_dim": 208, "seqs": 5, "tokens": 4,
         "spare": 3},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(("rope", "rope", "conv", "delta", "delta", "delta", "step", "step"))
    t = rng.choice(("f32", "f16", "bf16", "bf16"))
    if kind == "rope":
        kv, dim = rng.choice((1, 2, 4, 8)), rng.choice((16, 64, 80, 96, 128, 128, 256))
        heads, seqs = kv * rng.choice((1, 2, 4, 5, 8)), _log(rng, 1, 32)
        longest = max(1, min(_log(rng, 1, 8192), MAX_ROPE // (seqs * (heads + kv) * dim)))
        rot = rng.choice((dim, dim, dim // 2, dim // 4, 2 * rng.randint(1, dim // 2)))
        return {"kind": kind, "type": t, "heads": heads, "kv_heads": kv, "dim": dim, "rot": rot, "pairs": rng.random() < 0.4,
                "norm": rng.random() < 0.7, "seqs": seqs, "longest": longest, "first": rng.choice((0, _log(rng, 1, 1000000))),
                "scaling": rng.choice(("none", "linear", "divided", "yarn")), "fused": rng.random() < 0.4}
    if kind == "conv":
        channels, seqs = rng.choice((1, 3, 5)) * _log(rng, 8, 2500) + rng.choice((0, 0, 1)), _log(rng, 1, 64)
        return {"kind": kind, "type": t, "channels": channels, "width": rng.choice((2, 3, 4, 4, 4, 8)), "seqs": seqs,
                "longest": max(1, min(rng.choice((1, _log(rng, 1, 8192))), MAX_CONV // (seqs * channels))), "bias": rng.random() < 0.4}
    kh, kd, vd = rng.choice((1, 2, 4, 8, 16)), rng.choice((64, 96, 128, 128, 128, 256)), rng.choice((64, 80, 128, 128, 128, 256))
    vh = min(48, kh * rng.choice((1, 2, 3, 4)))
    vh -= vh % kh
    if kind == "delta":
        seqs = _log(rng, 1, 16)
        longest = max(1, min(_log(rng, 2, 8192), MAX_DELTA // (seqs * vh * kd * vd)))
        return {"kind": kind, "type": t, "k_heads": kh, "v_heads": vh, "k_dim": kd, "v_dim": vd, "seqs": seqs, "longest": longest,
                "state": rng.random() < 0.5}
    kd, vd = rng.choice((kd, 16 * rng.randint(1, 16))), rng.choice((vd, 16 * rng.randint(1, 16)))
    seqs = max(1, min(_log(rng, 1, 64), MAX_STATES // (vh * kd * vd)))
    return {"kind": kind, "type": t, "k_heads": kh, "v_heads": vh, "k_dim": kd, "v_dim": vd, "seqs": seqs,
            "tokens": rng.choice((1, 1, 1, 2, 4, 5)), "spare": rng.randint(0, 8)}


def _lens(case):
    """The sequences' lengths: the longest first, the others spread down to a tenth of it."""
    top = case["tokens"] if case["kind"] == "step" else case["longest"]
    if case["kind"] == "step":
        return [top] * case["seqs"]
    rng = random.Random(case["seqs"] * 1000003 + top)
    return [top] + [max(1, int(top * rng.uniform(0.1, 1.0))) for _ in range(case["seqs"] - 1)]


def _starts(lens):
    v = [0]
    for n in lens:
        v.append(v[-1] + n)
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, device="cuda", generator=gen)  # noqa: E731
    rand = lambda *shape: torch.rand(shape, device="cuda", generator=gen)  # noqa: E731
    lens, t = _lens(case), TYPES[case["type"]]
    n = sum(lens)
    s = {"case": case, "lens": lens, "start": _starts(lens), "n": n}
    if case["kind"] == "rope":
        H, KV, D = case["heads"], case["kv_heads"], case["dim"]
        spread = lambda h: torch.exp(0.5 * randn(1, h, 1))  # heads of different sizes  # noqa: E731
        if case["fused"]:  # rows of one projection: queries, keys, values
            x = (randn(n, H + 2 * KV, D) * spread(H + 2 * KV)).to(t)
            s["q"], s["k"] = x[:, :H], x[:, H:H + KV]
        else:
            s["q"], s["k"] = (randn(n, H, D) * spread(H)).to(t), (randn(n, KV, D) * spread(KV)).to(t)
        s["qo"], s["ko"] = torch.empty((n, H, D), dtype=t, device="cuda"), torch.empty((n, KV, D), dtype=t, device="cuda")
        s["qn"], s["kn"] = (1 + 0.2 * randn(D), 1 + 0.2 * randn(D)) if case["norm"] else (None, None)
        at = [case["first"] + (17 * i if case["first"] else 0) for i in range(len(lens))]
        s["pos"] = torch.cat([torch.arange(a, a + m, dtype=torch.int32, device="cuda") for a, m in zip(at, lens)])
        s["div"] = 1 + 7 * torch.sort(rand(case["rot"] // 2)).values if case["scaling"] == "divided" else None
        s["rope"] = {"base": 1e6 if case["first"] > 10000 else 1e4, "factor": {"linear": 4.0, "yarn": 4.0}.get(case["scaling"], 1.0),
                     "original": 32768 if case["scaling"] == "yarn" else 0}
    elif case["kind"] == "conv":
        C, W, S = case["channels"], case["width"], case["seqs"]
        s["x"], s["w"], s["b"] = randn(n, C).to(t), randn(C, W) * W ** -0.5, randn(C) if case["bias"] else None
        s["h"] = randn(S, W - 1, C).to(t)
        s["y"], s["ho"] = torch.empty((n, C), dtype=t, device="cuda"), torch.empty((S, W - 1, C), dtype=t, device="cuda")
    else:
        KH, VH, DK, DV, S = case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"], case["seqs"]
        unit = lambda x: (x / x.square().sum(-1, keepdim=True).sqrt()).to(t)  # noqa: E731
        s["q"], s["k"] = (unit(randn(n, KH, DK) + 0.5 * randn(1, KH, DK)) for _ in range(2))
        s["v"], s["beta"] = randn(n, VH, DV).to(t), torch.sigmoid(1.5 * randn(n, VH))
        forget = torch.exp(math.log(1e-4) + rand(VH) * (math.log(8.0) - math.log(1e-4)))
        s["g"] = -forget * torch.log1p(torch.exp(randn(n, VH)))
        s["o"] = torch.empty((n, VH, DV), dtype=t, device="cuda")
        slots = S + case.get("spare", 0)
        s["slots"], s["slot"] = slots, None
        if case["kind"] == "step":
            s["slot"] = torch.randperm(slots, device="cuda", generator=gen)[:S].to(torch.int32)
        s["s"] = 0.3 * randn(slots, VH, DK, DV) if case["kind"] == "step" or case["state"] else None
        s["so"] = torch.zeros((slots, VH, DK, DV), device="cuda")
    return s


# ------------------------------------------------------------- plain forms
def _freqs(c, s):
    """Radians a position of each pair, in 64 bits, and what the rotated values are multiplied by."""
    rot, r = c["rot"], s["rope"]
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    f = torch.pow(torch.tensor(r["base"], dtype=torch.float64, device="cuda"), -2 * i / rot)
    if s["div"] is not None:
        f = f / s["div"].double()
    if not r["original"]:
        return f / r["factor"], 1.0
    # the pairs that turn more than 32 times in the original context stay, those of less than one turn are scaled, a ramp between
    at = lambda turns: rot * math.log(r["original"] / (turns * 2 * math.pi)) / (2 * math.log(r["base"]))  # noqa: E731
    low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
    ramp = torch.clamp((i - low) / max(high - low, 0.001), 0, 1)
    return f * (ramp / r["factor"] + 1 - ramp), 0.1 * math.log(r["factor"]) + 1


def _plain_rope(s):
    c = s["case"]
    rot = c["rot"]
    f, mag = _freqs(c, s)
    a = s["pos"].double()[:, None] * f
    cos, sin = (torch.cos(a).float() * mag)[:, None], (torch.sin(a).float() * mag)[:, None]
    out = {}
    for name, x, w in (("q", s["q"], s["qn"]), ("k", s["k"], s["kn"])):
        x = x.float()
        if w is not None:
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
        if c["pairs"]:
            x0, x1 = x[..., 0:rot:2], x[..., 1:rot:2]
            y = torch.stack((x0 * cos - x1 * sin, x0 * sin + x1 * cos), -1).flatten(-2)
        else:
            x0, x1 = x[..., :rot // 2], x[..., rot // 2:rot]
            y = torch.cat((x0 * cos - x1 * sin, x0 * sin + x1 * cos), -1)
        out[name] = torch.cat((y, x[..., rot:]), -1).to(TYPES[c["type"]])
    return out


def _places(s, n):
    """Rows of padded sequences of n tokens: [seq][n] rows of the packed ones (past the end: the first), and whether they are there."""
    i = torch.arange(n, device="cuda")
    here = i < s["start"].diff()[:, None]
    return torch.where(here, s["start"][:-1, None] + i, 0).long(), here


def _packed(s, x):
    """The packed rows of padded ones x [seq][n]..."""
    _, here = _places(s, x.shape[1])
    return x[here]


def _plain_conv(s):
    c = s["case"]
    W, n = c["width"], max(s["lens"])
    at, here = _places(s, n)
    x = torch.cat((s["h"], torch.where(here[..., None], s["x"][at], 0)), 1)
    last = s["start"].diff()[:, None] + torch.arange(W - 1, device="cuda")
    state = x.gather(1, last.long()[..., None].expand(-1, -1, x.shape[2]))
    x = x.float()
    y = (x.unfold(1, W, 1) * s["w"]).sum(-1)
    if s["b"] is not None:
        y = y + s["b"]
    return {"y": _packed(s, y / (1 + torch.exp(-y))).to(TYPES[c["type"]]), "state": state}


def _plain_delta(s):
    c = s["case"]
    VH, DK, DV, S = c["v_heads"], c["k_dim"], c["v_dim"], c["seqs"]
    G, longest = VH // c["k_heads"], max(s["lens"])
    C = min(CHUNK, longest)
    nc = (longest + C - 1) // C
    at, here = _places(s, nc * C)

    def rows(x, heads):  # [seq * head][chunk][token]... in 32 bits, 0 past the end
        x = torch.where(here.view(here.shape + (1,) * (x.dim() - 1)), x[at].float(), 0)
        return x.transpose(1, 2).repeat_interleave(VH // heads, 1).reshape(S * VH, nc, C, *x.shape[3:]).contiguous()
    q, k, v = rows(s["q"], c["k_heads"]), rows(s["k"], c["k_heads"]), rows(s["v"], VH)
    beta, g = rows(s["beta"], VH), rows(s["g"], VH).double().cumsum(-1)
    i = torch.arange(C, device="cuda")
    upto = i[:, None] >= i
    decay = torch.exp((g[..., :, None] - g[..., None, :]).masked_fill(~upto, 0)).float() * upto
    kt = k.transpose(-1, -2).contiguous()
    a = torch.matmul(k, kt) * decay * beta[..., None] * (i[:, None] > i)
    p = torch.matmul(q, kt) * decay
    # (I + a)^-1: its rows one behind the other
    inv = torch.eye(C, device="cuda").expand(S * VH, nc, C, C).contiguous()
    for r in range(1, C):
        inv[:, :, r, :r] = -(a[:, :, r, :r, None] * inv[:, :, :r, :r]).sum(2)
    u = torch.matmul(inv, v * beta[..., None])
    eg = torch.exp(g).float()[..., None]
    w = torch.matmul(inv, k * beta[..., None] * eg)
    left = torch.exp(g[..., -1:] - g).float()[..., None]
    pick = torch.arange(S, device="cuda") if s["slot"] is None else s["slot"].long()
    state = torch.zeros((S * VH, DK, DV), device="cuda") if s["s"] is None else s["s"][pick].view(S * VH, DK, DV)
    out = torch.empty_like(v)
    for j in range(nc):  # a chunk needs the state that the one before left
        new = u[:, j] - torch.bmm(w[:, j], state)
        out[:, j] = torch.bmm(q[:, j] * eg[:, j], state) + torch.bmm(p[:, j], new)
        state = state * eg[:, j, -1:] + torch.bmm(kt[:, j], new * left[:, j])
    o = _packed(s, out.view(S, VH, nc * C, DV).transpose(1, 2)) * DK ** -0.5
    s["so"][pick] = state.view(S, VH, DK, DV)
    return {"o": o.to(TYPES[c["type"]]), "state": s["so"]}


# ------------------------------------------------------- the library's calls
_ENC = None


def _own(s):
    """The calls of a program: one context for the process, plain handles on the tensors."""
    global _ENC
    import chatokf_amd as ok
    if _ENC is None:
        _ENC = ok.Enc(0)
    enc, c, t = _ENC, s["case"], ok.BY_NAME[s["case"]["type"]]
    if c["kind"] == "rope":
        r = ok.Rope(c["rot"], pairs=c["pairs"], div=s["div"], **s["rope"])
        enc.norm_rope(r, s["pos"], s["n"], s["q"], s["qo"], c["heads"], s["k"], s["ko"], c["kv_heads"], c["dim"], type=t,
                      q_norm=s["qn"], k_norm=s["kn"], eps=1e-6, strides=[x.stride(0) for x in (s["q"], s["k"], s["qo"], s["ko"])])
        return {"q": s["qo"], "k": s["ko"]}
    if c["kind"] == "conv":
        enc.conv(s["x"], s["w"], s["y"], s["start"], c["seqs"], s["n"], c["channels"], c["width"], type=t, bias=s["b"], silu=True,
                 state_in=s["h"], state_out=s["ho"])
        return {"y": s["y"], "state": s["ho"]}
    call = enc.delta_step if c["kind"] == "step" else enc.delta_prompt
    call(s["q"], s["k"], s["v"], s["g"], s["beta"], s["o"], s["start"], c["seqs"], s["n"], c["k_heads"], c["v_heads"], c["k_dim"], c["v_dim"],
         type=t, scale=c["k_dim"] ** -0.5, state_in=s["s"], state_out=s["so"], slot=s["slot"], slots=s["slots"])
    return {"o": s["o"], "state": s["so"]}


def run(state):
    if own:
        return _own(state)
    return {"rope": _plain_rope, "conv": _plain_conv, "delta": _plain_delta, "step": _plain_delta}[state["case"]["kind"]](state)


# ------------------------------------------------------------------- work
def work(case):
    """Each input read once and each output written once."""
    n, size = sum(_lens(case)), 4 if case["type"] == "f32" else 2
    if case["kind"] == "rope":
        values = n * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 2 * size * values + 4 * n + 8 * case["dim"], "flops": 7.0 * values}
    if case["kind"] == "conv":
        C, W, held = case["channels"], case["width"], case["seqs"] * (case["width"] - 1) * case["channels"]
        return {"bytes": 2 * size * (n * C + held) + 4 * C * (W + 1), "flops": (2.0 * W + 4) * n * C}
    KH, VH, DK, DV = case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"]
    states = (2 if case["kind"] == "step" or case["state"] else 1) * case["seqs"] * VH * DK * DV
    # a token and head: the state decayed (1), S^T k (2), the correction added (2), S^T q (2)
    return {"bytes": size * n * 2 * (KH * DK + VH * DV) + 8 * n * VH + 4 * states, "flops": 7.0 * n * VH * DK * DV}


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rope":
        rot, r, D = case["rot"], s["rope"], case["dim"]
        f = [r["base"] ** (-2.0 * i / rot) for i in range(rot // 2)]
        mag = 1.0
        if s["div"] is not None:
            f = [x / d for x, d in zip(f, s["div"].double().tolist())]
        elif r["original"]:
            dim_of = lambda turns: rot * math.log(r["original"] / (turns * 2 * math.pi)) / (2 * math.log(r["base"]))  # noqa: E731
            lo, hi = max(math.floor(dim_of(32.0)), 0), min(math.ceil(dim_of(1.0)), rot - 1)
            part = [min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0) for i in range(rot // 2)]
            f = [x * (1 - p) + x / r["factor"] * p for x, p in zip(f, part)]
            mag = 1 + math.log(r["factor"]) / 10
        else:
            f = [x / r["factor"] for x in f]
        turn = torch.polar(torch.tensor(mag, dtype=torch.float64, device="cuda"),
                           s["pos"].double()[:, None, None] * torch.tensor(f, dtype=torch.float64, device="cuda"))
        out = {}
        for name, x, w in (("q", s["q"], s["qn"]), ("k", s["k"], s["kn"])):
            x = x.double().clone()
            if w is not None:
                x *= w.double() * ((x ** 2).sum(-1, keepdim=True) / D + 1e-6) ** -0.5
            first, second = (slice(0, rot, 2), slice(1, rot, 2)) if case["pairs"] else (slice(0, rot // 2), slice(rot // 2, rot))
            z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
            x[..., first], x[..., second] = z.real, z.imag
            out[name] = x
        return out
    if case["kind"] == "conv":
        W, ys, hs = case["width"], [], []
        for b, m in enumerate(s["lens"]):
            a = int(s["start"][b])
            x = torch.cat((s["h"][b].double(), s["x"][a:a + m].double()))
            y = torch.zeros((m, case["channels"]), dtype=torch.float64, device="cuda")
            if s["b"] is not None:
                y += s["b"].double()
            for j in range(W):
                y += x[j:j + m] * s["w"][:, j].double()
            ys.append(y * torch.sigmoid(y))
            hs.append(x[m:])
        return {"y": torch.cat(ys), "state": torch.stack(hs)}
    G, S = case["v_heads"] // case["k_heads"], case["seqs"]
    slot = list(range(S)) if s["slot"] is None else s["slot"].tolist()
    state = s["so"].double()
    st = torch.zeros((S,) + s["so"].shape[1:], dtype=torch.float64, device="cuda") if s["s"] is None else s["s"][slot].double()
    o = torch.zeros(s["o"].shape, dtype=torch.float64, device="cuda")
    order = sorted(range(S), key=lambda b: -s["lens"][b])   # the longest first: those that are left at a token are the first ones
    st, first = st[order], torch.tensor([int(s["start"][b]) for b in order], device="cuda")
    q, k = (s[x].double().repeat_interleave(G, 1) for x in ("q", "k"))
    v, decay, beta = s["v"].double(), torch.exp(s["g"].double()), s["beta"].double()
    for i in range(max(s["lens"])):
        m = sum(s["lens"][b] > i for b in order)
        r, cur = first[:m] + i, st[:m]
        cur *= decay[r][..., None, None]
        read = torch.matmul(k[r][..., None, :], cur)[..., 0, :]
        cur += k[r][..., None] * (beta[r][..., None] * (v[r] - read))[..., None, :]
        o[r] = torch.matmul(q[r][..., None, :], cur)[..., 0, :] * case["k_dim"] ** -0.5
    state[torch.tensor(slot, device="cuda")[torch.tensor(order, device="cuda")]] = st
    return {"o": o, "state": state}
