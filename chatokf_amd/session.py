"""A chat's attention layer on this library: projections on quantized weights, a
prompt, an 8-bit paged KV cache, decode steps that add up attention weights, and
eviction by them when the chat reaches its limit.

Weights come from decode steps and verify passes alone: a prompt adds none.  A
chat cut before its first step has equal weights for all tokens, so that its
first tokens stay; one cut soon after, what the last steps looked at.

Torch's own work (tensors made, filled, freed) belongs on the default stream,
which the context's stream keeps in order with; on another one the caller waits
where they meet.

``python -m chatokf_amd.session`` runs a layer with random weights through two
prompt chunks and some steps, and prints what they took.
"""
import time

import numpy as np
import torch

import chatokf_amd as ok
from chatokf_amd import synth


class Layer:
    """Query, key, value and output projections of one attention layer (rows of K activations)."""

    def __init__(self, enc: ok.Enc, K: int, heads: int, kv_heads: int, dim: int, seed: int = 1, ggml_type: int = ok.Q8_0):
        self.enc, self.K, self.heads, self.kv_heads, self.dim = enc, K, heads, kv_heads, dim

        def weight(M, K, s):
            return ok.QuantTensor(torch.from_numpy(synth.weights(ggml_type, M, K, seed + s)).cuda(), K, M, ggml_type)
        self.q, self.k, self.v = (weight(h * dim, K, s) for s, h in enumerate((heads, kv_heads, kv_heads)))
        self.o = weight(K, heads * dim, 3)

    def project(self, x):
        """Queries [n][heads][dim], keys and values [n][kv_heads][dim] of the rows x (fp32)."""
        out = [torch.empty((x.shape[0], w.M // self.dim, self.dim), device=x.device) for w in (self.q, self.k, self.v)]
        for w, y in zip((self.q, self.k, self.v), out):
            self.enc.gemm(w, x, y, x.shape[0])
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
        q, k, v = layer.project(x)
        self._append(k, v)
        if self.n > a:
            k, v = self.values()
        o = torch.empty_like(q)
        layer.enc.attn_prompt(q, k, v, o, self._starts(a), self._starts(self.n), 1, a, self.n, layer.heads, layer.kv_heads,
                              layer.dim, scale=self.scale)
        return layer.output(o)

    def step(self, x):
        """The next token's row; several rows are a verify pass."""
        layer = self.layer
        q, k, v = layer.project(x)
        self._append(k, v)
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


def main():
    enc = ok.Enc(0)
    layer = Layer(enc, 2048, 16, 8, 128)
    chat = Chat(layer, limit=4096, keep=1024)
    rng = np.random.default_rng(0)

    def rows(n):
        return torch.from_numpy(rng.standard_normal((n, layer.K)).astype(np.float32) / 10).cuda()
    for what, call, parts in (("prompt", chat.prompt, [rows(3000)]), ("chunk", chat.prompt, [rows(500)]),
                              ("steps", chat.step, [rows(1) for _ in range(700)]), ("verify passes", chat.step, [rows(4) for _ in range(8)])):
        torch.cuda.synchronize()
        t = time.perf_counter()
        for x in parts:
            y = call(x)
        enc.sync()
        t = time.perf_counter() - t
        assert torch.isfinite(y).all()
        print(f"{len(parts)} {what} of {parts[0].shape[0]}: {t * 1e3:.2f} ms, the chat holds {chat.n} tokens")
    enc.close()


if __name__ == "__main__":
    main()
