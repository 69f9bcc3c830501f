// okf_kv.h -- the paged 8-bit KV cache: its layout, quantizing new tokens into
// it (okf_kv_append), reading values back (okf_kv_read) and cutting sequences
// to their most attended tokens (okf_kv_evict).
//
// A page holds 64 tokens of every head as int8 codes with one fp32 scale a page
// and head.  Keys stand token by token ([64][dim]); values stand dimension by
// dimension ([dim][64]), a row's tokens in the order in which the attention
// kernel's matrix instruction takes them (kv_slot), so that it loads both
// without a transpose.
#pragma once
#include "okf_kv_seqs.h"

namespace okf {

// where token t of a page stands in a value row, and the token at byte b of
// 16-byte group g
__host__ __device__ constexpr uint32_t kv_slot(uint32_t t) { return t % 16 / 4 * 16 + t / 16 * 4 + t % 4; }
__host__ __device__ constexpr uint32_t kv_token(uint32_t g, uint32_t b) { return b / 4 * 16 + g * 4 + b % 4; }

// The page blocks that a sequence's last n rows touch: positions old .. len - 1.
struct KvSpan {
    uint32_t row;   // the row of position old
    uint32_t old, len;
    __device__ uint32_t blocks() const { return len > old ? (len - 1) / KV_B - old / KV_B + 1 : 0; }
};
__device__ __forceinline__ KvSpan kv_span(const KvSeqs &q, const int32_t *start, uint32_t s, uint32_t n) {
    const uint2 r = kv_rows(start, s, n);
    const uint32_t len = (uint32_t)max(q.len[s], 0), m = r.y - r.x;
    return m <= len ? KvSpan{r.x, len - m, len} : KvSpan{r.x + (m - len), 0, len};
}

// Largest |x| of a workgroup's values, NaN if one of them is NaN or infinite.
template <int NT>
__device__ __forceinline__ float kv_block_max(float m, bool bad, float *red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    const bool any = __ballot(bad) != 0;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = any ? __builtin_nanf("") : m;
    __syncthreads();
    float r = red[0];
#pragma unroll
    for (int w = 1; w < NT / 64; w++) r = red[w] != red[w] || r != r ? __builtin_nanf("") : fmaxf(r, red[w]);
    return r;
}

// The code of x under scale s: x / s rounded to the nearest whole number, ties
// to even, exactly.  r = rint(x * (1 / s)) is off by one at most, next to a
// half; d = x - r s is exact (r has 8 bits, and |d| is about s / 2 at most), so
// its comparison with s / 2 puts r right.  Scales so small that 1 / s or s / 2
// leaves the normal numbers divide in 64 bits.
__device__ __forceinline__ int kv_code(float x, float s, float inv) {
    float r;
    if (s > 1e-36f) {
        r = rintf(x * inv);
        const float d = fmaf(-r, s, x), a = 2.0f * fabsf(d);
        if (a > s || (a == s && ((int)r & 1))) r += d > 0 ? 1.0f : -1.0f;
    } else {
        r = s > 0 ? (float)rint((double)x / (double)s) : 0.0f;
    }
    return (int)fminf(fmaxf(r, -127.0f), 127.0f);  // (NaN scales: 0 below)
}

// A code under another scale: rint(c q), q the quotient of the scales in 64 bits.
__device__ __forceinline__ int kv_recode(int c, double q) {
    const double r = rint((double)c * q);
    return r == r ? (int)fmin(fmax(r, -127.0), 127.0) : 0;
}

constexpr int KV_NT = 256;

// okf_kv_append: workgroup (item, head, K or V); item: one page block that new
// tokens go to.  The block's new values stay in registers between the search
// for the largest and the rounding, so they are read once.
template <class T>
__global__ __launch_bounds__(KV_NT) void kv_append_kernel(KvCache c, KvSeqs q, const T *__restrict__ K,
                                                          const T *__restrict__ V, const int32_t *__restrict__ start,
                                                          uint32_t n, uint64_t kst, uint64_t vst) {
    __shared__ float red[KV_NT / 64];
    __shared__ __align__(16) uint8_t tile[256 * KV_B];  // V: [dim][slot]
    const SeqItem it = kv_find(blockIdx.x, q.count, [&](uint32_t s) { return kv_span(q, start, s, n).blocks(); });
    if (it.seq >= q.count) return;
    const KvSpan sp = kv_span(q, start, it.seq, n);
    const uint32_t blk = sp.old / KV_B + it.at;
    if (blk >= q.stride) return;
    const int32_t page = q.pages[(uint64_t)it.seq * q.stride + blk];
    if ((uint32_t)page >= c.pages) return;
    const bool isv = blockIdx.z;
    const uint32_t D = c.dim, h = blockIdx.y, tid = threadIdx.x;
    const uint32_t had = it.at == 0 ? sp.old % KV_B : 0;              // tokens held before
    const uint32_t end = min(sp.len - blk * KV_B, KV_B);              // tokens held after
    const T *src = (isv ? V : K) + ((uint64_t)sp.row + blk * KV_B + had - sp.old) * (isv ? vst : kst) + h * D;
    const uint64_t st = isv ? vst : kst;
    const uint32_t cpt = D / 8, chunks = (end - had) * cpt;  // 8-value chunks of the new tokens
    constexpr uint32_t MAXC = 256 / 8 * KV_B / KV_NT;
    float x[MAXC][8];
    float m = 0;
    bool bad = false;
#pragma unroll
    for (uint32_t i = 0; i < MAXC; i++) {
        const uint32_t e = tid + i * KV_NT;
        if (e >= chunks) break;
        const T *p = src + (uint64_t)(e / cpt) * st + e % cpt * 8;
        T raw[8];
        __builtin_memcpy(raw, __builtin_assume_aligned(p, 16), sizeof(raw));
#pragma unroll
        for (int j = 0; j < 8; j++) {
            x[i][j] = to_f32(raw[j]);
            m = fmaxf(m, fabsf(x[i][j]));
            bad |= !(fabsf(x[i][j]) <= 3.402823466e38f);
        }
    }
    const float top = kv_block_max<KV_NT>(m, bad, red);
    const uint64_t ph = (uint64_t)page * c.heads + h;
    float *sc = (isv ? c.vs : c.ks) + ph;
    const float was = had ? *sc : 0.0f;
    const float now = was != was || top != top ? __builtin_nanf("") : fmaxf(was, top / 127.0f);
    __syncthreads();  // (every thread has read the old scale)
    if (tid == 0) *sc = now;
    const float inv = 1.0f / now;
    const bool again = had && now != was;  // (a NaN scale too: its codes are cleared)
    const double ratio = (double)was / (double)now;
    int8_t *out = (isv ? c.v : c.k) + ph * KV_B * D;
    if (!isv) {
        if (again)
            for (uint32_t e = tid; e < had * cpt; e += KV_NT) {
                int8_t b[8];
                __builtin_memcpy(b, out + e * 8, 8);
#pragma unroll
                for (int j = 0; j < 8; j++) b[j] = (int8_t)kv_recode(b[j], ratio);
                __builtin_memcpy(out + e * 8, b, 8);
            }
#pragma unroll
        for (uint32_t i = 0; i < MAXC; i++) {
            const uint32_t e = tid + i * KV_NT;
            if (e >= chunks) break;
            int8_t b[8];
#pragma unroll
            for (int j = 0; j < 8; j++) b[j] = (int8_t)(now == now ? kv_code(x[i][j], now, inv) : 0);
            __builtin_memcpy(out + had * D + e * 8, b, 8);
        }
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < MAXC; i++) {
        const uint32_t e = tid + i * KV_NT;
        if (e >= chunks) break;
        const uint32_t slot = kv_slot(had + e / cpt), d = e % cpt * 8;
#pragma unroll
        for (int j = 0; j < 8; j++) tile[(d + j) * KV_B + slot] = (uint8_t)(now == now ? kv_code(x[i][j], now, inv) : 0);
    }
    __syncthreads();
    for (uint32_t e = tid; e < D * 4; e += KV_NT) {
        const uint32_t g = e & 3;
        uint8_t nb[16];
        int8_t ob[16];
        __builtin_memcpy(nb, tile + e * 16, 16);
        if (had) __builtin_memcpy(ob, out + e * 16, 16);
#pragma unroll
        for (int b = 0; b < 16; b++) {
            const uint32_t t = kv_token(g, b);
            if (t < had) nb[b] = (uint8_t)(again ? kv_recode(ob[b], ratio) : ob[b]);
            else if (t >= end) nb[b] = 0;
        }
        __builtin_memcpy(out + e * 16, nb, 16);
    }
}

template <class T>
__device__ __forceinline__ void kv_put(T *p, const float (&x)[8]) {
    T r[8];
#pragma unroll
    for (int j = 0; j < 8; j++) r[j] = (T)x[j];
    __builtin_memcpy(__builtin_assume_aligned(p, 16), r, sizeof(r));
}

// okf_kv_read: workgroup (item, head, K or V); item: one page block of a
// sequence's last rows.
template <class T>
__global__ __launch_bounds__(KV_NT) void kv_read_kernel(KvCache c, KvSeqs q, T *__restrict__ K, T *__restrict__ V,
                                                        const int32_t *__restrict__ start, uint32_t n, uint64_t kst,
                                                        uint64_t vst) {
    __shared__ __align__(16) uint8_t tile[KV_B * (256 + 16)];  // V: [token][dim]
    const SeqItem it = kv_find(blockIdx.x, q.count, [&](uint32_t s) {
        const uint2 r = kv_rows(start, s, n);
        const KvSpan sp = kv_span(q, start, s, n);
        return sp.blocks() + (r.y - r.x > sp.len);  // (one item more for rows before the sequence)
    });
    const bool isv = blockIdx.z;
    T *dst = isv ? V : K;
    if (it.seq >= q.count || !dst) return;
    const KvSpan sp = kv_span(q, start, it.seq, n);
    const uint64_t st = isv ? vst : kst;
    const uint32_t D = c.dim, h = blockIdx.y, tid = threadIdx.x, cpt = D / 8;
    if (it.at >= sp.blocks()) {
        const float zero[8] = {};
        const uint32_t a = kv_rows(start, it.seq, n).x;
        for (uint64_t e = tid; e < (uint64_t)(sp.row - a) * cpt; e += KV_NT)
            kv_put(dst + (a + e / cpt) * st + h * D + e % cpt * 8, zero);
        return;
    }
    const uint32_t blk = sp.old / KV_B + it.at;
    const uint32_t t0 = it.at == 0 ? sp.old % KV_B : 0, end = min(sp.len - blk * KV_B, KV_B);
    const int32_t page = blk < q.stride ? q.pages[(uint64_t)it.seq * q.stride + blk] : -1;
    const bool have = (uint32_t)page < c.pages;
    const uint64_t ph = have ? (uint64_t)page * c.heads + h : 0;
    const float sc = have ? (isv ? c.vs : c.ks)[ph] : 0.0f;
    const int8_t *codes = (isv ? c.v : c.k) + ph * KV_B * D;
    const uint32_t row = D + 16;
    if (isv && have) {
        for (uint32_t e = tid; e < D * 4; e += KV_NT) {
            uint8_t b[16];
            __builtin_memcpy(b, codes + e * 16, 16);
#pragma unroll
            for (int i = 0; i < 16; i++) tile[kv_token(e & 3, i) * row + (e >> 2)] = b[i];
        }
        __syncthreads();
    }
    for (uint32_t e = tid; e < (end - t0) * cpt; e += KV_NT) {
        const uint32_t t = t0 + e / cpt, d = e % cpt * 8;
        float x[8] = {};
        if (have) {
            int8_t b[8];
            __builtin_memcpy(b, isv ? (const int8_t *)tile + t * row + d : codes + t * D + d, 8);
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = (float)b[j] * sc;
        }
        kv_put(dst + ((uint64_t)sp.row + blk * KV_B + t - sp.old) * st + h * D + d, x);
    }
}

// A weight as an unsigned key of the same order (-0 as 0, NaN lowest).
__device__ __forceinline__ uint32_t kv_key(float w) {
    if (w != w) return 0;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return u >> 31 ? ~u : u | 0x80000000u;
}

// Inclusive sum over the workgroup's threads, in order.
template <int NT>
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t *red, uint32_t &total) {
    const uint32_t lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t u = __shfl_up(v, o);
        if (lane >= (uint32_t)o) v += u;
    }
    __syncthreads();
    if (lane == 63) red[w] = v;
    __syncthreads();
    uint32_t add = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < NT / 64; i++) {
        if (i < (int)w) add += red[i];
        total += red[i];
    }
    return v + add;
}

// okf_kv_evict, first launch: one workgroup per (sequence, head) finds the key
// of the last token that stays (four rounds of a 256-way count, from the top
// byte down) and lists the kept tokens in order.
constexpr int EV_NT = 1024;
__global__ __launch_bounds__(EV_NT) void kv_select_kernel(KvSeqs from, int32_t *__restrict__ new_len, uint32_t heads,
                                                          uint32_t keep, uint32_t sink, uint32_t recent,
                                                          const float *__restrict__ W, uint64_t wst, float *WO,
                                                          uint64_t wost, int32_t *__restrict__ kept) {
    __shared__ uint32_t hist[256], red[EV_NT / 64], pick[2];
    const uint32_t tid = threadIdx.x, s = blockIdx.x / heads, h = blockIdx.x % heads;
    const uint64_t sh = (uint64_t)s * heads + h;
    const uint32_t len = min((uint32_t)max(from.len[s], 0), (uint32_t)min((uint64_t)from.stride * KV_B, (uint64_t)0x7FFFFFFF));
    const float *w = W + sh * wst;
    int32_t *list = kept + sh * keep;
    if (h == 0 && tid == 0) new_len[s] = (int32_t)min(len, keep);
    if (len <= keep) {
        for (uint32_t i = tid; i < keep; i += EV_NT) {
            list[i] = i < len ? (int32_t)i : -1;
            if (WO && i < len) WO[sh * wost + i] = w[i];
        }
        return;
    }
    const uint32_t lo = sink, hi = len - recent;
    uint32_t want = keep - sink - recent;  // of [lo, hi)
    uint32_t key = 0, mask = 0;
    if (want) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (uint32_t i = lo + tid; i < hi; i += EV_NT) {
                const uint32_t k = kv_key(w[i]);
                if ((k & mask) == key) atomicAdd(&hist[k >> shift & 255], 1u);
            }
            __syncthreads();
            // the digit at which the count from the top reaches `want`
            uint32_t total;
            const uint32_t mine = tid < 256 ? hist[255 - tid] : 0;
            const uint32_t upto = block_scan<EV_NT>(mine, red, total);
            if (tid < 256 && upto >= want && upto - mine < want) {
                pick[0] = 255 - tid;
                pick[1] = want - (upto - mine);
            }
            __syncthreads();
            key |= pick[0] << shift;
            mask |= 255u << shift;
            want = pick[1];
        }
    }
    // in order: larger keys, the first `want` of equal ones, sink and recent
    uint32_t at = 0, ties = 0;
    const bool none = keep == sink + recent;
    for (uint32_t b = 0; b < len; b += EV_NT) {
        const uint32_t i = b + tid;
        const bool in = i < len, inner = in && i >= lo && i < hi;
        const float x = in ? w[i] : 0.0f;
        const uint32_t k = kv_key(x);
        const bool tie = inner && !none && k == key;
        uint32_t nt, nk;
        const uint32_t tr = block_scan<EV_NT>(tie, red, nt) + ties;
        const bool stay = in && (!inner || (!none && (k > key || (tie && tr <= want))));
        const uint32_t r = block_scan<EV_NT>(stay, red, nk) + at;
        if (stay) {
            list[r - 1] = (int32_t)i;
            if (WO) WO[sh * wost + r - 1] = x;
        }
        ties += nt;
        at += nk;
    }
}

// okf_kv_evict, second launch: workgroup (new block, head, sequence) gathers
// the listed tokens and rounds them to the block's scale.
__global__ __launch_bounds__(KV_NT) void kv_gather_kernel(KvCache c, KvSeqs from, KvCache o, KvSeqs to, uint32_t keep,
                                                          const int32_t *__restrict__ kept) {
    __shared__ double qk[KV_B], qv[KV_B];
    __shared__ uint64_t base[KV_B];
    __shared__ uint32_t pos[KV_B];
    const uint32_t blk = blockIdx.x, h = blockIdx.y % c.heads, tid = threadIdx.x;
    const uint64_t s = (uint64_t)blockIdx.z * (gridDim.y / c.heads) + blockIdx.y / c.heads;
    if (s >= from.count) return;
    const int32_t *list = kept + (s * c.heads + h) * keep + blk * KV_B;
    const uint32_t left = min(keep - blk * KV_B, KV_B), D = c.dim;
    const int32_t page = to.pages[s * to.stride + blk];
    if ((uint32_t)page >= o.pages || list[0] < 0) return;
    const uint64_t ph = (uint64_t)page * o.heads + h;
    if (tid < KV_B) {
        const int32_t i = tid < left ? list[tid] : -1;
        const int32_t p = i >= 0 ? from.pages[s * from.stride + i / KV_B] : -1;
        const bool have = (uint32_t)p < c.pages;
        const uint64_t sh = have ? (uint64_t)p * c.heads + h : 0;
        const float a = have ? c.ks[sh] : 0.0f, b = have ? c.vs[sh] : 0.0f;
        float ma = a, mb = b;
#pragma unroll
        for (int x = 32; x > 0; x >>= 1) {
            ma = fmaxf(ma, __shfl_xor(ma, x));
            mb = fmaxf(mb, __shfl_xor(mb, x));
        }
        if (__ballot(a != a)) ma = __builtin_nanf("");
        if (__ballot(b != b)) mb = __builtin_nanf("");
        qk[tid] = ma != 0 ? (double)a / (double)ma : 0.0;
        qv[tid] = mb != 0 ? (double)b / (double)mb : 0.0;
        base[tid] = have ? sh * KV_B * D : ~0ull;
        pos[tid] = i % KV_B;
        if (tid == 0) {
            o.ks[ph] = ma;
            o.vs[ph] = mb;
        }
    }
    __syncthreads();
    int8_t *ok = o.k + ph * KV_B * D, *ov = o.v + ph * KV_B * D;
    const uint32_t cpt = D / 16;
    for (uint32_t e = tid; e < KV_B * cpt; e += KV_NT) {
        const uint32_t t = e / cpt, d = e % cpt * 16;
        int8_t b[16] = {};
        if (base[t] != ~0ull) __builtin_memcpy(b, c.k + base[t] + pos[t] * D + d, 16);
        if (qk[t] != 1.0) {
#pragma unroll
            for (int j = 0; j < 16; j++) b[j] = (int8_t)kv_recode(b[j], qk[t]);
        }
        __builtin_memcpy(ok + e * 16, b, 16);
    }
    for (uint32_t e = tid; e < D * 4; e += KV_NT) {
        const uint32_t g = e & 3, d = e >> 2;
        int8_t b[16];
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const uint32_t t = kv_token(g, j);
            const int x = base[t] != ~0ull ? c.v[base[t] + d * KV_B + kv_slot(pos[t])] : 0;
            b[j] = (int8_t)(qv[t] != 1.0 ? kv_recode(x, qv[t]) : x);
        }
        __builtin_memcpy(ov + e * 16, b, 16);
    }
}

}  // namespace okf
