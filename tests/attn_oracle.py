"""Attention and the paged 8-bit KV cache in 64 bits, row by row (numpy)."""
import numpy as np

B = 64


def slot(t):
    return t % 16 // 4 * 16 + t // 16 * 4 + t % 4


def attend(q, k, v, at, window, scale):
    """One head: queries [n][D] at positions at[n], keys / values [m][D]; results [n][D] and weights [n][m]."""
    o, w = np.zeros((len(q), v.shape[1])), np.zeros((len(q), len(k)))
    for i in range(len(q)):
        lo, hi = (max(0, at[i] - window + 1) if window else 0), min(at[i] + 1, len(k))
        if hi <= lo:
            continue
        s = k[lo:hi].astype(np.float64) @ q[i].astype(np.float64) * scale
        if np.all(s == -np.inf):
            continue
        e = np.exp(s - np.max(s))
        w[i, lo:hi] = e / e.sum()
        o[i] = w[i, lo:hi] @ v[lo:hi].astype(np.float64)
    return o, w


def prompt(q, k, v, qs, ks, window, scale):
    """q [nq][H][D], k, v [nk][KV][D] packed by qs, ks."""
    H, KV = q.shape[1], k.shape[1]
    o = np.zeros(q.shape)
    for s in range(len(qs) - 1):
        n, m = qs[s + 1] - qs[s], ks[s + 1] - ks[s]
        for h in range(H):
            kh = h // (H // KV)
            o[qs[s]:qs[s + 1], h] = attend(q[qs[s]:qs[s + 1], h], k[ks[s]:ks[s + 1], kh], v[ks[s]:ks[s + 1], kh],
                                           np.arange(n) + m - n, window, scale)[0]
    return o


class Cache:
    """Codes by token: k, v int8 [pages][heads][64][D]; scales fp32 [pages][heads]."""

    def __init__(self, pages, heads, D, rng):
        self.k, self.v = (rng.integers(-127, 128, (pages, heads, B, D)).astype(np.int8) for _ in range(2))
        self.ks, self.vs = (rng.uniform(0.01, 0.04, (pages, heads)).astype(np.float32) for _ in range(2))

    def device_v(self):
        out = np.empty((*self.v.shape[:2], self.v.shape[3], B), np.int8)
        for t in range(B):
            out[..., slot(t)] = self.v[:, :, t]
        return out

    @staticmethod
    def tokens_of(v):
        """The library's value layout back to token by token."""
        out = np.empty((*v.shape[:2], B, v.shape[2]), np.int8)
        for t in range(B):
            out[:, :, t] = v[..., slot(t)]
        return out

    def values(self, table, n):
        """Keys and values [n][heads][D] in 64 bits of a sequence's first n tokens, and which of them are held."""
        H, D = self.k.shape[1], self.k.shape[3]
        k, v, have = np.zeros((n, H, D)), np.zeros((n, H, D)), np.zeros(n, bool)
        for t in range(n):
            p = table[t // B] if t // B < len(table) else -1
            if 0 <= p < len(self.k):
                k[t] = self.k[p, :, t % B].astype(np.float64) * self.ks[p][:, None].astype(np.float64)
                v[t] = self.v[p, :, t % B].astype(np.float64) * self.vs[p][:, None].astype(np.float64)
                have[t] = True
        return k, v, have

    def append(self, table, length, k, v):
        """The last len(k) of `length` tokens."""
        drop = max(0, len(k) - length)
        k, v = k[drop:], v[drop:]
        old = length - len(k)
        if length == old:
            return
        for blk in range(old // B, (length - 1) // B + 1):
            if blk >= len(table) or not 0 <= table[blk] < len(self.k):
                continue
            p, had = table[blk], max(0, old - blk * B)
            end = min(length - blk * B, B)
            for codes, scale, x in ((self.k, self.ks, k), (self.v, self.vs, v)):
                new = x[blk * B + had - old:blk * B + end - old]
                for h in range(codes.shape[1]):
                    y = new[:, h].astype(np.float64)
                    was = scale[p, h] if had else np.float32(0)
                    if not np.all(np.isfinite(y)) or np.isnan(was):
                        scale[p, h] = np.nan
                        codes[p, h, :end] = 0
                        continue
                    now = np.float32(max(np.float64(was), np.float64(np.float32(np.abs(y).max() / 127))))
                    scale[p, h] = now
                    if had and now != was:
                        codes[p, h, :had] = np.rint(codes[p, h, :had] * (np.float64(was) / np.float64(now)))
                    codes[p, h, had:end] = np.clip(np.rint(y / np.float64(now)), -127, 127) if now > 0 else 0

    def evict(self, table, length, w, keep, sink, recent):
        """Per head: the kept tokens, and [kept][D] codes and scales by new block for k and v."""
        length = min(length, len(table) * B)
        out = []
        for h in range(self.k.shape[1]):
            kept = list(range(length))
            if length > keep:
                x = np.where(np.isnan(w[h]), -np.inf, w[h])
                inner = sorted(range(sink, length - recent), key=lambda i: (np.isnan(w[h][i]), -x[i], i))
                kept = sorted([*range(sink), *inner[:keep - sink - recent], *range(length - recent, length)])
            res = [kept]
            for codes, scale in ((self.k, self.ks), (self.v, self.vs)):
                new, tops = np.zeros((len(kept), codes.shape[3])), []
                for b in range(0, len(kept), B):
                    part = kept[b:b + B]
                    sc = np.array([scale[table[t // B], h] if 0 <= table[t // B] < len(codes) else 0 for t in part], np.float64)
                    top = sc.max()
                    tops.append(top)
                    for i, t in enumerate(part):
                        if sc[i] and top == top:
                            new[b + i] = np.rint(codes[table[t // B], h, t % B] * (sc[i] / top))
                res += [new, np.array(tops)]
            out.append(res)
        return out
