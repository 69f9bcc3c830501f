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

// Largest of a workgroup's unsigned values.
template <int NT>
__device__ __forceinline__ uint32_t kv_block_max(uint32_t m, uint32_t *red) {
    m = lanes_max(m);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64; w++) m = max(m, red[w]);
    return m;
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

// Four small integers' low bytes.
__device__ __forceinline__ uint32_t kv_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0C0C0400u), __builtin_amdgcn_perm(b, a, 0x0C0C0400u), 0x05040100u);
}

// The codes of 8 values.  x (1 / s) is off by 2^-23 of itself at most, 1.6e-5: where
// its distance to the whole number is not so close to a half, that number (taken from
// the sum with 1.5 2^23, whose low bits it is) is the code; else, one value in ten
// thousand, kv_code tells.
__device__ __forceinline__ uint2 kv_codes(const float (&x)[8], float s, float inv) {
    constexpr float MAGIC = 12582912.0f;
    uint32_t c[8];
    float off = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float y = fmaf(x[j], inv, MAGIC);
        off = fmaxf(off, fabsf(fmaf(x[j], inv, MAGIC - y)));
        c[j] = __float_as_uint(y);
    }
    if (!(off < 0.4999f) || !(s > 1e-36f)) {
#pragma unroll
        for (int j = 0; j < 8; j++) c[j] = s == s ? (uint32_t)kv_code(x[j], s, inv) : 0;
    }
    return {kv_bytes(c[0], c[1], c[2], c[3]), kv_bytes(c[4], c[5], c[6], c[7])};
}

// A code under another scale: rint(c q), q the quotient of the scales in 64 bits.  The
// product with q in fp32 is off by 2^-23 of itself at most: only next to a half does
// the one in 64 bits tell.
struct KvRatio {
    double q;
    float f;
    __device__ __forceinline__ explicit KvRatio(double x) : q(x), f((float)x) {}
};
__device__ __forceinline__ int kv_recode(int c, const KvRatio &q) {
    const float x = (float)c * q.f, r = rintf(x);
    if (fabsf(x - r) < 0.4999f) return (int)fminf(fmaxf(r, -127.0f), 127.0f);
    const double y = rint((double)c * q.q);
    return y == y ? (int)fmin(fmax(y, -127.0), 127.0) : 0;
}

// The same for the four codes of a dword: their whole numbers in low bytes (the sum with
// 1.5 2^23), and in `off` how near to a half they came.  Right where off < 0.4999 and f is
// a number.
__device__ __forceinline__ float kv_near(float c, float f, float &off) {
    constexpr float MAGIC = 12582912.0f;
    const float y = fmaf(c, f, MAGIC);
    off = fmaxf(off, fabsf(fmaf(c, f, MAGIC - y)));
    return y;
}
__device__ __forceinline__ u32x4 kv_recode16(u32x4 x, double q) {
    const float f = (float)q;
    float off = 0;
    u32x4 r;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        uint32_t y[4];
#pragma unroll
        for (int n = 0; n < 4; n++) y[n] = __float_as_uint(kv_near((float)(int8_t)(x[j] >> 8 * n), f, off));
        r[j] = kv_bytes(y[0], y[1], y[2], y[3]);
    }
    if (!(off < 0.4999f) || f != f) {
        const KvRatio all(q);
#pragma unroll 1
        for (int j = 0; j < 4; j++) {
            const uint32_t from = j == 0 ? x[0] : j == 1 ? x[1] : j == 2 ? x[2] : x[3];
            uint32_t y[4];
#pragma unroll
            for (int n = 0; n < 4; n++) y[n] = (uint32_t)kv_recode((int8_t)(from >> 8 * n), all);
            const uint32_t to = kv_bytes(y[0], y[1], y[2], y[3]);
            r[0] = j == 0 ? to : r[0], r[1] = j == 1 ? to : r[1], r[2] = j == 2 ? to : r[2], r[3] = j == 3 ? to : r[3];
        }
    }
    return r;
}

// The 4 x 4 bytes of four dwords, transposed.
__device__ __forceinline__ void kv_transpose(uint32_t (&x)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u), b = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u);
    const uint32_t c = __builtin_amdgcn_perm(x[1], x[0], 0x07030602u), d = __builtin_amdgcn_perm(x[3], x[2], 0x07030602u);
    x[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    x[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    x[2] = __builtin_amdgcn_perm(d, c, 0x05040100u);
    x[3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}

// A page's values in LDS: rows of a dimension's 64 codes, a dword apart more than they
// are long, so that sixteen rows' dwords at a time lie in different banks.
constexpr uint32_t KV_PITCH = KV_B / 4 + 1;

constexpr int KV_NT = 256;

// Row and column of unit e in rows of n, for e = first, first + KV_NT, ... (one division
// in all).
struct KvWalk {
    uint32_t n, row, col, drow, dcol;
    __device__ __forceinline__ KvWalk(uint32_t first, uint32_t n) : n(n), row(first / n), col(first - row * n),
                                                                    drow((uint32_t)KV_NT / n), dcol((uint32_t)KV_NT - drow * n) {}
    __device__ __forceinline__ void next() {
        row += drow, col += dcol;
        if (col >= n) col -= n, row++;
    }
};

// okf_kv_append: workgroup (item, head, K or V); item: one page block that new
// tokens go to.  The block's new values stay in registers between the search
// for the largest and the rounding, so they are read once.  Bound by latency: for one
// token by the chain of dependent loads (sequence, page, scale), 5 us; for long prompts by each
// workgroup's wait for its loads, its largest value and the codes' way through LDS byte by
// byte (4 bf16 prompts of up to 2500 x 8 heads of 128: 43 MB in 18.8 us, 2.3 TB/s, under half of
// a copy's rate).
template <class T, int ND>  // ND: 64s of dimensions
__global__ __launch_bounds__(KV_NT) void kv_append_kernel(KvCache c, KvSeqs q, const T *__restrict__ K,
                                                          const T *__restrict__ V, const int32_t *__restrict__ start,
                                                          uint32_t n, uint64_t kst, uint64_t vst) {
    __shared__ uint32_t red[KV_NT / 64];
    __shared__ uint32_t tile[64 * ND * KV_PITCH];  // V: [dim][slot]
    const SeqItem it = kv_find(blockIdx.x, q.count, [&](uint32_t s) { return kv_span(q, start, s, n).blocks(); });
    if (it.seq >= q.count) return;
    const KvSpan sp = kv_span(q, start, it.seq, n);
    const uint32_t blk = sp.old / KV_B + it.at;
    if (blk >= q.stride) return;
    const int32_t page = q.pages[(uint64_t)it.seq * q.stride + blk];
    const bool isv = blockIdx.z;
    const uint32_t D = c.dim, h = blockIdx.y, tid = threadIdx.x;
    const uint32_t had = it.at == 0 ? sp.old % KV_B : 0;              // tokens held before
    const uint32_t end = min(sp.len - blk * KV_B, KV_B);              // tokens held after
    const T *src = (isv ? V : K) + ((uint64_t)sp.row + blk * KV_B + had - sp.old) * (isv ? vst : kst) + h * D;
    const uint64_t st = isv ? vst : kst;
    const uint32_t cpt = D / 8, chunks = (end - had) * cpt;  // 8-value chunks of the new tokens
    constexpr uint32_t MAXC = 64 * ND / 8 * KV_B / KV_NT;
    T raw[MAXC][8];
    const KvWalk at0(tid, cpt);
    KvWalk at = at0;
#pragma unroll
    for (uint32_t i = 0; i < MAXC; i++) {
        if (tid + i * KV_NT >= chunks) break;
        __builtin_memcpy(raw[i], __builtin_assume_aligned(src + (uint64_t)at.row * st + at.col * 8, 16), sizeof(raw[i]));
        at.next();
    }
    if ((uint32_t)page >= c.pages) return;
    const uint64_t ph = (uint64_t)page * c.heads + h;
    float *sc = (isv ? c.vs : c.ks) + ph;
    const float was = had ? *sc : 0.0f;
    uint32_t m = 0;  // the largest magnitude's bits: infinities and NaN above all others
#pragma unroll
    for (uint32_t i = 0; i < MAXC; i++) {
        if (tid + i * KV_NT >= chunks) break;
#pragma unroll
        for (int j = 0; j < 8; j++) m = max(m, __float_as_uint(to_f32(raw[i][j])) & 0x7FFFFFFFu);
    }
    m = kv_block_max<KV_NT>(m, red);
    const float now = was != was || m >= 0x7F800000u ? __builtin_nanf("") : fmaxf(was, __uint_as_float(m) / 127.0f);
    __syncthreads();  // (every thread has read the old scale)
    if (tid == 0) *sc = now;
    const float inv = 1.0f / now;
    const bool again = had && now != was;  // (a NaN scale too: its codes are cleared)
    const double ratio = again ? (double)was / (double)now : 1.0;
    int8_t *out = (isv ? c.v : c.k) + ph * KV_B * D;
    if (!isv && again)
        for (uint32_t e = tid; e < had * (D / 16); e += KV_NT)
            *(u32x4 *)(out + e * 16) = kv_recode16(*(const u32x4 *)(out + e * 16), ratio);
    // few new values beside ones that stay as they are: byte by byte
    const bool few = had && !again && end - had <= 8;
    at = at0;
#pragma unroll
    for (uint32_t i = 0; i < MAXC; i++, at.next()) {
        const uint32_t e = tid + i * KV_NT;
        if (e >= chunks) break;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = to_f32(raw[i][j]);
        const uint2 b = kv_codes(x, now, inv);
        if (!isv) {
            *(uint2 *)(out + had * D + e * 8) = b;
            continue;
        }
        const uint32_t slot = kv_slot(had + at.row), d = at.col * 8;
        if (few) {
#pragma unroll
            for (int j = 0; j < 8; j++) out[(d + j) * KV_B + slot] = (int8_t)((j < 4 ? b.x : b.y) >> j % 4 * 8);
        } else {
            uint8_t *to = (uint8_t *)tile + d * KV_PITCH * 4 + slot;
#pragma unroll
            for (int j = 0; j < 8; j++) to[j * KV_PITCH * 4] = (uint8_t)((j < 4 ? b.x : b.y) >> j % 4 * 8);
        }
    }
    if (!isv || few) return;
    __syncthreads();
    for (uint32_t e = tid; e < D * 4; e += KV_NT) {
        const uint32_t g = e & 3;
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = tile[(e >> 2) * KV_PITCH + g * 4 + i];
        if (had || end < KV_B) {
            u32x4 x = {0, 0, 0, 0};
            if (had) {
                x = *(const u32x4 *)(out + e * 16);
                if (again) x = kv_recode16(x, ratio);
            }
#pragma unroll
            for (int b = 0; b < 16; b++) {
                const uint32_t t = kv_token(g, b), m = 255u << b % 4 * 8;
                if (t < had) w[b / 4] = (w[b / 4] & ~m) | (x[b / 4] & m);
                else if (t >= end) w[b / 4] &= ~m;
            }
        }
        *(u32x4 *)(out + e * 16) = u32x4{w[0], w[1], w[2], w[3]};
    }
}

// Four codes' values.
template <class T>
__device__ __forceinline__ void kv_put4(T *p, uint32_t codes, float sc) {
    T r[4];
    const uint32_t u = codes ^ 0x80808080u;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        float x = ((float)(u >> 8 * j & 255u) - 128.0f) * sc;
        asm("" : "+v"(x));  // (the fp32 product, not one that is rounded to T alone)
        r[j] = (T)x;
    }
    __builtin_memcpy(__builtin_assume_aligned(p, sizeof(r)), r, sizeof(r));
}

// okf_kv_read: workgroup (item, head, K or V); item: one page block of a
// sequence's last rows.  Bound by memory, most of it the values written.
template <class T, int ND>
__global__ __launch_bounds__(KV_NT) void kv_read_kernel(KvCache c, KvSeqs q, T *__restrict__ K, T *__restrict__ V,
                                                        const int32_t *__restrict__ start, uint32_t n, uint64_t kst,
                                                        uint64_t vst) {
    __shared__ uint32_t tile[64 * ND * KV_PITCH];  // V: [dim][slot]
    const bool isv = blockIdx.z;
    T *dst = isv ? V : K;
    if (!dst) return;
    const SeqItem it = kv_find(blockIdx.x, q.count, [&](uint32_t s) {
        const uint2 r = kv_rows(start, s, n);
        const KvSpan sp = kv_span(q, start, s, n);
        return sp.blocks() + (r.y - r.x > sp.len);  // (one item more for rows before the sequence)
    });
    if (it.seq >= q.count) return;
    const KvSpan sp = kv_span(q, start, it.seq, n);
    const uint64_t st = isv ? vst : kst;
    const uint32_t D = c.dim, h = blockIdx.y, tid = threadIdx.x, q4 = D / 4;
    if (it.at >= sp.blocks()) {
        const uint32_t a = kv_rows(start, it.seq, n).x;
        for (uint64_t e = tid; e < (uint64_t)(sp.row - a) * q4; e += KV_NT)
            kv_put4(dst + (a + e / q4) * st + h * D + e % q4 * 4, 0, 0.0f);
        return;
    }
    const uint32_t blk = sp.old / KV_B + it.at;
    const uint32_t t0 = it.at == 0 ? sp.old % KV_B : 0, end = min(sp.len - blk * KV_B, KV_B);
    const int32_t page = blk < q.stride ? q.pages[(uint64_t)it.seq * q.stride + blk] : -1;
    const bool have = (uint32_t)page < c.pages;
    const uint64_t ph = have ? (uint64_t)page * c.heads + h : 0;
    const float sc = have ? (isv ? c.vs : c.ks)[ph] : 0.0f;
    const int8_t *codes = (isv ? c.v : c.k) + ph * KV_B * D;
    T *out = dst + ((uint64_t)sp.row + blk * KV_B - sp.old) * st + h * D;  // (token 0 of the block's; rows from t0)
    if (!have) {
        for (uint32_t e = tid; e < (end - t0) * q4; e += KV_NT) kv_put4(out + (uint64_t)(t0 + e / q4) * st + e % q4 * 4, 0, 0.0f);
        return;
    }
    if (!isv) {
        constexpr uint32_t IN = 4 * ND;  // loads under way: up to the page's
        const uint32_t all = end * q4;
        KvWalk at(t0 * q4 + tid, q4);
        for (uint32_t e0 = t0 * q4 + tid; e0 < all; e0 += IN * KV_NT) {
            uint32_t x[IN];
#pragma unroll
            for (uint32_t i = 0; i < IN; i++) x[i] = e0 + i * KV_NT < all ? ((const uint32_t *)codes)[e0 + i * KV_NT] : 0;
#pragma unroll
            for (uint32_t i = 0; i < IN; i++, at.next())
                if (e0 + i * KV_NT < all) kv_put4(out + (uint64_t)at.row * st + at.col * 4, x[i], sc);
        }
        return;
    }
    u32x4 x[ND];
#pragma unroll
    for (uint32_t i = 0; i < ND; i++)
        if (tid + i * KV_NT < D * 4) x[i] = ((const u32x4 *)codes)[tid + i * KV_NT];
#pragma unroll
    for (uint32_t i = 0; i < ND; i++) {
        const uint32_t e = tid + i * KV_NT;
        if (e >= D * 4) break;
#pragma unroll
        for (int j = 0; j < 4; j++) tile[(e >> 2) * KV_PITCH + (e & 3) * 4 + j] = x[i][j];
    }
    __syncthreads();
    // units of four tokens and four dimensions, sixteen of the latter side by side
    for (uint32_t e = tid; e < (q4 + 15) / 16 * 256; e += KV_NT) {
        const uint32_t d = (e % 16 + e / 256 * 16) * 4, t = e / 16 % 16 * 4;
        if (d >= D || t >= end || t + 4 <= t0) continue;
        uint32_t y[4];
#pragma unroll
        for (int j = 0; j < 4; j++) y[j] = tile[(d + j) * KV_PITCH + kv_slot(t) / 4];
        kv_transpose(y);
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (t + j >= t0 && t + j < end) kv_put4(out + (uint64_t)(t + j) * st + d, y[j], sc);
    }
}

// The tokens that sequence s of an eviction holds in its table.
__device__ __forceinline__ uint32_t kv_held(const KvSeqs &q, uint64_t s) {
    return min((uint32_t)max(q.len[s], 0), (uint32_t)min((uint64_t)q.stride * KV_B, (uint64_t)0x7FFFFFFF));
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
    v = lanes_sum(v);
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
// of the last token that stays (a count by the top 11 bits, then by the next 11 and the
// last 10) and lists the kept tokens in order.  A wavefront takes 1024 tokens side by
// side, 64 at a time, so that a token's place among its wavefront's is a count of lanes;
// up to EV_ALL tokens' keys stay in registers from count to count.  Always three counts with
// their barriers: 8 heads of 4096 tokens 12 us, on as many CUs; 128 of up to 16000 26.  The weights may be W's own
// rows: a kept one goes to its own place or to a lower one, which no later round reads, and
// those of one round are all read before the first of them is written.
constexpr int EV_NT = 1024;
constexpr uint32_t EV_PER = 16, EV_ALL = EV_NT * EV_PER;
__global__ __launch_bounds__(EV_NT) void kv_select_kernel(KvSeqs from, uint32_t heads, uint32_t keep, uint32_t sink,
                                                          uint32_t recent, const float *W, uint64_t wst, float *WO,
                                                          uint64_t wost, int32_t *__restrict__ kept) {
    __shared__ uint32_t hist[2048], red[EV_NT / 64], pick[2];
    const uint32_t tid = threadIdx.x, s = blockIdx.x / heads, h = blockIdx.x % heads, lane = tid & 63;
    const uint64_t sh = (uint64_t)s * heads + h;
    const uint32_t len = kv_held(from, s);
    const float *w = W + sh * wst;
    int32_t *list = kept + sh * keep;
    if (len <= keep) {
        for (uint32_t i = tid; i < keep; i += EV_NT) {
            list[i] = i < len ? (int32_t)i : -1;
            if (WO && i < len) WO[sh * wost + i] = w[i];
        }
        return;
    }
    // The tokens that stay anyway have keys above all weights', so that the `keep` largest are
    // looked for; places past the end have 0 and come last among those (NaN) of 0.
    const uint32_t lo = sink, hi = len - recent;
    // tokens of a wavefront, in 64s; this lane's first one of a round of EV_ALL
    const uint32_t per = min((len + EV_NT - 1) / EV_NT, EV_PER), mine = tid / 64 * 64 * per + lane;
    uint32_t k[EV_PER];
    auto load = [&](uint32_t b) {
#pragma unroll
        for (uint32_t u = 0; u < EV_PER; u++) {
            const uint32_t i = b + mine + u * 64;
            k[u] = u < per && i < len ? (i >= lo && i < hi ? kv_key(w[i]) : 0xFFFFFFFFu) : 0;
        }
    };
    auto below = [](uint64_t who) { return __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0)); };
    load(0);
    uint32_t want = keep, key = 0, mask = 0;
#pragma unroll 1
    for (int round = 0; round < 3; round++) {
        const uint32_t shift = round == 0 ? 21 : round == 1 ? 10 : 0, bits = round == 2 ? 1023 : 2047;
        hist[tid] = hist[tid + EV_NT] = 0;
        __syncthreads();
        for (uint32_t b = 0; b < len; b += EV_ALL) {
            if (len > EV_ALL) load(b);
#pragma unroll
            for (uint32_t u = 0; u < EV_PER; u++)
                if (u < per) {
                    const bool in = (k[u] & mask) == key;
                    const uint64_t who = __ballot(in);
                    if (who) {
                        const uint32_t d = k[u] >> shift & bits;
                        const int first = __ffsll((unsigned long long)who) - 1;
                        const uint32_t d0 = __builtin_amdgcn_readlane(d, first);
                        // (all in one bin, as equal weights are: one addition)
                        if (__ballot(in && d == d0) == who) {
                            if ((int)lane == first) atomicAdd(&hist[d0], (uint32_t)__popcll(who));
                        } else if (in) {
                            atomicAdd(&hist[d], 1u);
                        }
                    }
                }
        }
        __syncthreads();
        // the digit at which the count from the top reaches `want`: two a thread
        const bool on = 2 * tid < bits;
        const uint32_t top = bits - 2 * tid, h0 = on ? hist[top] : 0, h1 = on ? hist[top - 1] : 0;
        uint32_t total;
        const uint32_t upto = block_scan<EV_NT>(h0 + h1, red, total), before = upto - h0 - h1;
        if (upto >= want && before < want) {
            const bool one = before + h0 >= want;
            pick[0] = one ? top : top - 1;
            pick[1] = want - before - (one ? 0 : h0);
        }
        __syncthreads();
        key |= pick[0] << shift;
        mask |= bits << shift;
        want = pick[1];
    }
    // in order: larger keys and the first `want` of equal ones
    uint32_t at = 0, ties = 0;
    for (uint32_t b = 0; b < len; b += EV_ALL) {
        if (len > EV_ALL) load(b);
        // what a wavefront has, from `have`, to what all have before it
        auto share = [&](uint32_t have, uint32_t &all) {
            __syncthreads();
            if (lane == 0) red[tid >> 6] = have;
            __syncthreads();
            uint32_t before = 0;
            all = 0;
#pragma unroll
            for (uint32_t i = 0; i < EV_NT / 64; i++) {
                if (i < tid >> 6) before += red[i];
                all += red[i];
            }
            return before;
        };
        uint32_t nt = 0, ns = 0, all;
#pragma unroll
        for (uint32_t u = 0; u < EV_PER; u++)
            if (u < per) nt += __popcll(__ballot(k[u] == key));
        uint32_t tie = ties + share(nt, all);
        ties += all;
        uint32_t stays = 0;  // bit u: token u stays
#pragma unroll
        for (uint32_t u = 0; u < EV_PER; u++)
            if (u < per) {
                const uint64_t who = __ballot(k[u] == key);
                bool stay = k[u] > key;
                if (who) {
                    stay |= k[u] == key && tie + below(who) < want;
                    tie += __popcll(who);
                }
                stays |= (uint32_t)stay << u;
                ns += __popcll(__ballot(stay));
            }
        uint32_t to = at + share(ns, all);
        at += all;
        float x[EV_PER];
        if (WO) {
#pragma unroll
            for (uint32_t u = 0; u < EV_PER; u++) x[u] = w[stays >> u & 1 ? b + mine + u * 64 : 0];
            __syncthreads();  // (the other wavefronts' too, before the first is written: WO may be W)
        }
#pragma unroll
        for (uint32_t u = 0; u < EV_PER; u++)
            if (u < per) {
                const bool stay = stays >> u & 1;
                const uint64_t who = __ballot(stay);
                if (stay) {
                    const uint32_t r = to + below(who);
                    list[r] = (int32_t)(b + mine + u * 64);
                    if (WO) WO[sh * wost + r] = x[u];
                }
                to += __popcll(who);
            }
    }
}

// okf_kv_evict, second launch: workgroup (new block, head, sequence) gathers
// the listed tokens and rounds them to the block's scale.  It also writes the new lengths,
// which may stand in the old ones' array: no workgroup here reads a length but the one that
// writes it.  Keys are rows; a value is a
// byte in each of a page's rows.  Wavefront g takes the tokens of byte group g (kv_slot)
// of every source page: a lane loads the group's 16 bytes of its rows, which is all of
// the page's lines that hold kept tokens, and puts each kept byte to its new place in
// LDS.  Bound by memory latency and those lines: 16 sequences of up to 16000 tokens x 8
// heads of 128 to 2000 each read nearly all of their values' 144 MB.
template <int ND>  // 64s of dimensions
__global__ __launch_bounds__(KV_NT) void kv_gather_kernel(KvCache c, KvSeqs from, KvCache o, KvSeqs to, uint32_t keep,
                                                          const int32_t *__restrict__ kept) {
    __shared__ uint32_t tile[64 * ND * KV_PITCH];  // the block's values, [dim][slot]
    __shared__ double qk[KV_B], qv[KV_B];
    __shared__ uint64_t base[KV_B], run_base[KV_B];
    __shared__ unsigned long long run_has[KV_B];  // the page's tokens that stay
    __shared__ uint32_t pos[KV_B], run_at[KV_B], runs;
    const uint32_t blk = blockIdx.x, h = blockIdx.y % c.heads, tid = threadIdx.x;
    const uint64_t s = (uint64_t)blockIdx.z * (gridDim.y / c.heads) + blockIdx.y / c.heads;
    if (s >= from.count) return;
    // (by the last wavefront: the first one has loads enough to wait for)
    if (blk == 0 && h == 0 && tid == KV_NT - 1) to.len[s] = (int32_t)min(kv_held(from, s), keep);
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
        // the runs of tokens from one page
        const int32_t mine = i >= 0 ? i / (int32_t)KV_B : -1, last = __shfl_up(mine, 1);
        const bool first = tid == 0 || mine != last;
        const uint64_t who = __ballot(first);
        const uint32_t r = __popcll(who & ((2ull << tid) - 1)) - 1;
        const uint64_t at = have ? sh * KV_B * D : ~0ull;
        run_has[tid] = 0;
        if (first) run_at[r] = tid, run_base[r] = at;
        if (tid == 0) runs = __popcll(who);
        base[tid] = at;
        pos[tid] = i % KV_B;
        if (have) atomicOr(&run_has[r], 1ull << i % KV_B);
        // (scales are 0 or more: their bits' order is theirs, NaN above all)
        const float ma = __uint_as_float(lanes_max(__float_as_uint(a))), mb = __uint_as_float(lanes_max(__float_as_uint(b)));
        qk[tid] = ma != 0 ? (double)a / (double)ma : 0.0;
        qv[tid] = mb != 0 ? (double)b / (double)mb : 0.0;
        if (tid == 0) {
            o.ks[ph] = ma;
            o.vs[ph] = mb;
        }
    }
    for (uint32_t e = tid; e < D * KV_PITCH; e += KV_NT) tile[e] = 0;  // (tokens without a page)
    __syncthreads();
    int8_t *ok = o.k + ph * KV_B * D, *ov = o.v + ph * KV_B * D;
    constexpr uint32_t KC = ND * 4 * KV_B / KV_NT;
    u32x4 kx[KC];
    const KvWalk at0(tid, D / 16);
    KvWalk at = at0;
#pragma unroll
    for (uint32_t i = 0; i < KC; i++, at.next())
        if (at.row < KV_B)
            kx[i] = base[at.row] != ~0ull ? *(const u32x4 *)(c.k + base[at.row] + pos[at.row] * D + at.col * 16) : u32x4{0, 0, 0, 0};

    const uint32_t lane = tid & 63, g = __builtin_amdgcn_readfirstlane(tid >> 6), nr = __builtin_amdgcn_readfirstlane(runs);
    auto uniform = [](uint64_t x) {
        return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(x >> 32)) << 32 |
               (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)x);
    };
    const float qf = (float)qv[lane];
    struct Run {
        uint64_t has;
        uint32_t at;
        u32x4 x[ND];
    };
    // the next run from r on with tokens of group g, and its bytes on their way
    uint32_t r = 0;
    auto next = [&](Run &n) {
        for (; r < nr; r++) {
            n.has = uniform(run_has[r]);
            if (!(n.has >> 4 * g & 0x000F000F000F000Full)) continue;
            n.at = __builtin_amdgcn_readfirstlane(run_at[r]);
            const int8_t *p = c.v + uniform(run_base[r]) + 16 * g;
#pragma unroll
            for (int d = 0; d < ND; d++) n.x[d] = *(const u32x4 *)(p + min(64u * d + lane, D - 1) * KV_B);
            r++;
            return true;
        }
        return false;
    };
    uint8_t *put = (uint8_t *)tile + lane * KV_PITCH * 4;
    auto place = [&](const Run &n) {
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const uint32_t p = j / 4 * 16 + 4 * g + j % 4;  // kv_token(g, j)
            if (!(n.has >> p & 1)) continue;
            const uint32_t t = n.at + __popcll(n.has & ((1ull << p) - 1));
            const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(qf), t));
            float off = 0;
            uint32_t y[ND];
#pragma unroll
            for (int d = 0; d < ND; d++) y[d] = __float_as_uint(kv_near((float)(int8_t)(n.x[d][j / 4] >> 8 * (j % 4)), f, off));
            if (!(off < 0.4999f) || f != f) {
#pragma unroll
                for (int d = 0; d < ND; d++) y[d] = (uint32_t)kv_recode((int8_t)(n.x[d][j / 4] >> 8 * (j % 4)), KvRatio(qv[t]));
            }
            uint8_t *dst = put + kv_slot(t);
#pragma unroll
            for (int d = 0; d < ND; d++) dst[64 * d * KV_PITCH * 4] = (uint8_t)y[d];  // (rows past the last: LDS of their own)
        }
    };
    Run a, b;
    bool more = next(a);
    while (more) {
        more = next(b);
        place(a);
        if (!more) break;
        more = next(a);
        place(b);
    }
    at = at0;
#pragma unroll
    for (uint32_t i = 0; i < KC; i++, at.next()) {
        if (at.row >= KV_B) break;
        kx[i] = kv_recode16(kx[i], qk[at.row]);
        *(u32x4 *)(ok + (tid + i * KV_NT) * 16) = kx[i];
    }
    __syncthreads();
    for (uint32_t e = tid; e < D * 4; e += KV_NT) {
        const uint32_t *x = tile + (e >> 2) * KV_PITCH + (e & 3) * 4;
        *(u32x4 *)(ov + e * 16) = u32x4{x[0], x[1], x[2], x[3]};
    }
}

}  // namespace okf
