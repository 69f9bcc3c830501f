"""A chat's layers on this library.

The attention layer: projections on quantized weights, head norms and rotation by
positions where the layer has them, a prompt, an 8-bit paged KV cache, decode
steps that add up attention weights, and eviction by them when the chat reaches
its limit.  Cached keys have their positions in them: what is kept keeps its own, and the next
token's goes on counting.

The gated delta rule's layer: projections, the short convolution, unit queries and
keys, the rule itself and a gated norm of what it reads.  A chat's state has one
size however long the chat is; several chats' tokens go through it as packed rows.

Weights come from decode steps and verify passes alone: a prompt adds none.  A
chat cut before its first step has equal weights for all tokens, so that its
first tokens stay; one cut soon after, what the last steps looked at.

Torch's own work (tensors made, filled, freed) belongs on the default stream,
which the context's stream keeps in order with; on another one the caller waits
where they meet.

``python -m chatokf_amd.session`` runs a layer of each with random weights through two
prompt chunks and some steps, and prints what they took.
"""
import time

import numpy as np
import torch

import chatokf_amd as ok
from chatokf_amd import synth


def _weight(ggml_type, M, K, seed):
    return ok.QuantTensor(torch.from_numpy(synth.weights(ggml_type, M, K, seed)).cuda(), K, M, ggml_type)


class Layer:
    """Query, key, value and output projections of one attention layer (rows of K activations), with a
    rotation by positions and norms of each query's and key's head (their weights) where given."""

    def __init__(self, enc: ok.Enc, K: int, heads: int, kv_heads: int, dim: int, seed: int = 1, ggml_type: int = ok.Q8_0,
                 rope: ok.Rope = None, q_norm=None, k_norm=None, eps: float = 1e-6):
        self.enc, self.K, self.heads, self.kv_heads, self.dim = enc, K, heads, kv_heads, dim
        self.rope, self.q_norm, self.k_norm, self.eps = rope or ok.Rope(0), q_norm, k_norm, eps
        self.q, self.k, self.v = (_weight(ggml_type, h * dim, K, seed + s) for s, h in enumerate((heads, kv_heads, kv_heads)))
        self.o = _weight(ggml_type, K, heads * dim, seed + 3)

    def project(self, x, at: int = 0):
        """Queries [n][heads][dim], keys and values [n][kv_heads][dim] of the rows x (fp32) at positions at, at + 1, ..."""
        n = x.shape[0]
        out = [torch.empty((n, w.M // self.dim, self.dim), device=x.device) for w in (self.q, self.k, self.v)]
        for w, y in zip((self.q, self.k, self.v), out):
            self.enc.gemm(w, x, y, n)
        q, k, _ = out
        turns = self.rope.c().rot > 0
        if turns or self.q_norm is not None or self.k_norm is not None:
            pos = torch.arange(at, at + n, dtype=torch.int32, device=x.device) if turns else None
            self.enc.norm_rope(self.rope, pos, n, q, q, self.heads, k, k, self.kv_heads, self.dim, q_norm=self.q_norm,
                               k_norm=self.k_norm, eps=self.eps)
        return out

    def output(self, a):
        y = torch.empty((a.shape[0], self.K), device=a.device)
        self.enc.gemm(self.o, a, y, a.shape[0])
        return y


class Chat:
    """One sequence of at most ``limit`` tokens, cut to ``keep`` of them a head where the next would
    not fit: its first ``sink``, its last ``recent``, and those of the most attention.  Its pages are
    two halves of a cache; eviction moves it from one to the other."""

    def __init__(self, layer: Layer, limit: int, keep: int, sink: int = 4, recent: int = 64):
        self.layer, self.limit, self.keep, self.sink, self.recent = layer, limit, keep, sink, recent
        blocks = (limit + ok.KV_BLOCK - 1) // ok.KV_BLOCK
        self.cache = ok.KVCache.new(2 * blocks, layer.kv_heads, layer.dim)
        self.tables = torch.arange(2 * blocks, dtype=torch.int32, device="cuda").view(2, blocks)
        self.lens = torch.zeros((2, 1), dtype=torch.int32, device="cuda")
        self.seqs = [ok.KVSeqs(self.tables[i], self.lens[i], 1, blocks) for i in range(2)]
        self.w = torch.zeros((2, layer.kv_heads, blocks * ok.KV_BLOCK), device="cuda")
        self.kept = torch.empty((layer.kv_heads, keep), dtype=torch.int32, device="cuda")
        self.at, self.n, self.scale = 0, 0, layer.dim ** -0.5
        self.pos = 0  # of the next token: those evicted count

    def _starts(self, n):
        return torch.tensor([0, n], dtype=torch.int32, device="cuda")

    def _append(self, k, v):
        n, cut = k.shape[0], min(self.n, self.keep)
        if cut + n > self.limit:  # (refused before anything is evicted for it)
            raise ValueError(f"{n} new tokens do not fit beside {cut} of {self.limit}")
        if self.n + n > self.limit:
            self.evict()
        self.n += n
        self.lens[self.at].fill_(self.n)
        self.layer.enc.kv_append(self.cache, self.seqs[self.at], k, v, self._starts(n), n)

    def values(self):
        """The cache's keys and values as fp32 [tokens][kv_heads][dim]."""
        k, v = (torch.empty((self.n, self.layer.kv_heads, self.layer.dim), device="cuda") for _ in range(2))
        self.layer.enc.kv_read(self.cache, self.seqs[self.at], k, v, self._starts(self.n), self.n)
        return k, v

    def prompt(self, x):
        """A prompt's rows, or the next chunk's behind what the chat holds: their attention's output rows."""
        a, layer = x.shape[0], self.layer
        q, k, v = layer.project(x, self.pos)
        self._append(k, v)
        self.pos += a
        if self.n > a:
            k, v = self.values()
        o = torch.empty_like(q)
        layer.enc.attn_prompt(q, k, v, o, self._starts(a), self._starts(self.n), 1, a, self.n, layer.heads, layer.kv_heads,
                              layer.dim, scale=self.scale)
        return layer.output(o)

    def step(self, x):
        """The next token's row; several rows are a verify pass."""
        layer = self.layer
        q, k, v = layer.project(x, self.pos)
        self._append(k, v)
        self.pos += x.shape[0]
        o = torch.empty_like(q)
        w = self.w[self.at]
        layer.enc.attn_decode(self.cache, self.seqs[self.at], q, o, x.shape[0], layer.heads, self.scale, w_in=w, w_out=w,
                              w_stride=w.shape[1])
        return layer.output(o)

    def evict(self):
        a, b = self.at, 1 - self.at
        self.w[b].zero_()
        self.layer.enc.kv_evict(self.cache, self.seqs[a], self.cache, self.seqs[b], self.keep, self.sink, self.recent,
                                self.w[a], self.w.shape[2], self.w[b], self.w.shape[2], self.kept)
        self.at, self.n = b, min(self.n, self.keep)


class DeltaLayer:
    """One layer of the gated delta rule (rows of K activations): a projection to queries, keys and values,
    which go through the short convolution, one to the output's gates, one to the two gates of
    each value head (what the state forgets, how much it takes in), and the output's."""

    def __init__(self, enc: ok.Enc, K: int, k_heads: int, v_heads: int, k_dim: int, v_dim: int, width: int = 4, seed: int = 1,
                 ggml_type: int = ok.Q8_0, eps: float = 1e-6):
        self.enc, self.K, self.k_heads, self.v_heads, self.k_dim, self.v_dim, self.width = enc, K, k_heads, v_heads, k_dim, v_dim, width
        self.keys, self.values, self.eps = k_heads * k_dim, v_heads * v_dim, eps
        self.channels = 2 * self.keys + self.values
        self.qkv, self.z, self.gates, self.o = (_weight(ggml_type, M, k, seed + s) for s, (M, k) in enumerate(
            ((self.channels, K), (self.values, K), (2 * v_heads, K), (K, self.values))))
        rng = np.random.default_rng(seed)
        self.conv = torch.from_numpy((rng.standard_normal((self.channels, width)) * width ** -0.5).astype(np.float32)).cuda()
        self.decay = torch.from_numpy(np.geomspace(1e-3, 8, v_heads).astype(np.float32)).cuda()  # (a token's, at a gate of 1)
        self.norm = torch.ones(v_dim, device="cuda")
        self.unit = torch.full((k_dim,), k_dim ** -0.5, device="cuda")  # (a head's norm with these weights: its length)

    def __call__(self, x, start, seqs, conv, state, keep: bool, few: bool):
        """The output rows of the packed sequences' rows x; their states conv and state move on where they are kept."""
        enc, n, C = self.enc, x.shape[0], self.channels
        u, z, ab = (torch.empty((n, m), device=x.device) for m in (C, self.values, 2 * self.v_heads))
        for w, y in ((self.qkv, u), (self.z, z), (self.gates, ab)):
            enc.gemm(w, x, y, n)
        y, o = torch.empty_like(u), torch.empty_like(z)
        enc.conv(u, self.conv, y, start, seqs, n, C, self.width, silu=True, state_in=conv, state_out=conv if keep else None)
        q, k, v = y[:, :self.keys], y[:, self.keys:2 * self.keys], y[:, 2 * self.keys:]
        enc.norm_rope(ok.Rope(0), None, n, q, q, self.k_heads, k, k, self.k_heads, self.k_dim, q_norm=self.unit, k_norm=self.unit,
                      eps=self.eps / self.k_dim, strides=(C, C, C, C))
        g = -self.decay * torch.nn.functional.softplus(ab[:, :self.v_heads])
        beta = torch.sigmoid(ab[:, self.v_heads:])
        run = enc.delta_step if few else enc.delta_prompt
        run(q, k, v, g, beta, o, start, seqs, n, self.k_heads, self.v_heads, self.k_dim, self.v_dim, scale=self.k_dim ** -0.5,
            state_in=state, state_out=state if keep else None, strides=(C, C, C, 0))
        enc.norm_rope(ok.Rope(0), None, n, o, o, self.v_heads, dim=self.v_dim, q_norm=self.norm, eps=self.eps)
        enc.silu_mul(z, o, n * self.values)
        out = torch.empty((n, self.K), device=x.device)
        enc.gemm(self.o, z, out, n)
        return out


class DeltaChats:
    """The states of some chats in one DeltaLayer.  Each call takes the chats' rows packed, `lens` of each
    (all of them the first chat's where not given; 0: its state stays)."""

    def __init__(self, layer: DeltaLayer, chats: int = 1):
        self.layer, self.chats = layer, chats
        self.conv = torch.zeros((chats, layer.width - 1, layer.channels), device="cuda")
        self.state = torch.zeros((chats, layer.v_heads, layer.k_dim, layer.v_dim), device="cuda")

    def _run(self, x, lens, keep, few):
        lens = [x.shape[0]] + [0] * (self.chats - 1) if lens is None else list(lens)
        if not x.shape[0] or len(lens) != self.chats or min(lens) < 0 or sum(lens) != x.shape[0]:
            raise ValueError(f"{lens} are not the rows of {self.chats} chats in {x.shape[0]}")
        start = torch.tensor([0, *np.cumsum(lens)], dtype=torch.int32, device=x.device)
        return self.layer(x, start, self.chats, self.conv, self.state, keep, few)

    def prompt(self, x, lens=None):
        """Prompts' rows, or the next chunks' behind what the chats hold."""
        return self._run(x, lens, True, False)

    def step(self, x, lens=None):
        """The next token's row of each chat, or a few."""
        return self._run(x, lens, True, True)

    def verify(self, x, lens=None):
        """A step that moves no state: the accepted rows go through step."""
        return self._run(x, lens, False, True)


def main():
    enc = ok.Enc(0)
    layer = Layer(enc, 2048, 16, 8, 128, rope=ok.Rope(128), q_norm=torch.ones(128, device="cuda"), k_norm=torch.ones(128, device="cuda"))
    chat = Chat(layer, limit=4096, keep=1024)
    delta = DeltaChats(DeltaLayer(enc, 2048, 16, 32, 128, 128))
    rng = np.random.default_rng(0)

    def rows(n):
        return torch.from_numpy(rng.standard_normal((n, 2048)).astype(np.float32) / 10).cuda()

    def run(what, call, parts, holds):
        torch.cuda.synchronize()
        t = time.perf_counter()
        for x in parts:
            y = call(x)
        enc.sync()
        t = time.perf_counter() - t
        assert torch.isfinite(y).all()
        print(f"{len(parts)} {what} of {parts[0].shape[0]}: {t * 1e3:.2f} ms, {holds()}")

    tokens = (("prompt", [rows(3000)]), ("chunk", [rows(500)]), ("steps", [rows(1) for _ in range(700)]),
              ("verify passes", [rows(4) for _ in range(8)]))
    for what, parts in tokens:
        run("attention " + what, chat.prompt if len(parts) == 1 else chat.step, parts, lambda: f"the chat holds {chat.n} tokens")
    size = (delta.conv.nbytes + delta.state.nbytes) / 2 ** 20
    for (what, parts), call in zip(tokens, (delta.prompt, delta.prompt, delta.step, delta.verify)):
        run("delta rule " + what, call, parts, lambda: f"the chat holds {size:.2f} MiB")
    enc.close()


if __name__ == "__main__":
    main()
