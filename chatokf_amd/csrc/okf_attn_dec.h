// okf_attn_dec.h -- attention of a sequence's last tokens to the paged 8-bit
// cache (okf_attn_decode) on the integer matrix cores.
//
// Arithmetic.  A cached key is code * scale, so q k = scale_k f (Q code) with
// Q = rint(q / f), f a power of two for each query row such that |Q| < 2^23:
// three signed byte digits Q = Q2 2^16 + Q1 2^8 + Q0, each a column operand of
// v_mfma_i32_16x16x64_i8 against the codes as they lie in memory.  Their sums
// are exact in 32 bits ((Q1 code << 8) + Q0 code too), so a score's roundings
// are Q's (2^-24 of the row's largest) and a few in fp32.  The softmax weights p
// <= 1 of the page's largest score become P = rint(p (2^23 - 2^15 - 2^7 - 1)) the
// same way for the product with the value codes (against the running maximum, one
// token that takes nearly all would leave the others' integers no digits).  No code
// is ever unpacked.
//
// Layout.  A wavefront takes one page (64 tokens) at a time and 16 query rows
// (row = query token * group + query head of the group); where there are more, two
// wavefronts of a workgroup take a page each with 16 rows of their own.  Scores: A = 16 tokens
// x 64 dimensions of K, B = a digit plane of the queries; a lane then holds,
// for the query row lane % 16, tokens 16 t + 4 (lane / 16) + i.  Values: A = 16
// dimensions x the page's 64 tokens, B = a digit plane of P, whose 16 bytes a lane
// are just the tokens whose scores it holds, in the order that kv_slot gives
// the value rows: no exchange between lanes, and no LDS, until the wavefronts
// of a workgroup join their results at the end.
//
// Bound by the cache's bytes for batches (32 sequences of up to 8192 tokens, 8 kv heads of
// 128: this launch 56 us again and again on one cache, 5.2 TB/s, as fast as a copy; a call on a
// cache not read before 69 us, 6 of them the join's), by the chain of loads (length, page, scale, keys)
// and the second launch for one short sequence (1999 tokens 7.3 + 4.0 us), by latency and the
// vector units for wide heads (100003 tokens x 4 x 256, 20 rows each: 57 us, the call 64, 3.2 TB/s:
// one wavefront a SIMD; two, with the values in the keys' registers, spill: 100 us).
#pragma once
#include "okf_ffn_mfma.h"
#include "okf_kv_seqs.h"

namespace okf {

constexpr uint32_t DEC_NT = 256, DEC_W = DEC_NT / 64;
constexpr float DEC_P = 8355711.0f;      // 0x7F7F7F: the largest 3-digit number with signed byte digits
constexpr double LOG2E = 1.4426950408889634;

struct DecArgs {
    KvCache c;
    KvSeqs s;
    const float *q;
    float *o;
    uint32_t tokens, heads;
    float scale;
    uint32_t window;
    const float *w_in;
    float *w_out;
    uint64_t wst;
    uint32_t splits, rb;   // page ranges a sequence; blocks of 16 NR query rows
    float *part, *ml;      // [row block][split][16 NR][dim], [row block][split][16 NR][2]
    float *sc;             // scores [sequence][kv head][row][64 stride] for the weights, or null: they are made again
};

// Four integers + 0x808080 -> the dwords of their three digit planes.
__device__ __forceinline__ void dec_digits(uint32_t a, uint32_t b, uint32_t c, uint32_t d, int &p0, int &p1, int &p2) {
    const uint32_t ab = perm(b, a, 0x05010400u), cd = perm(d, c, 0x05010400u);  // a0 b0 a1 b1
    const uint32_t ah = perm(b, a, 0x0C0C0602u), ch = perm(d, c, 0x0C0C0602u);  // a2 b2
    p0 = (int)(perm(cd, ab, 0x05040100u) ^ 0x80808080u);
    p1 = (int)(perm(cd, ab, 0x07060302u) ^ 0x80808080u);
    p2 = (int)(perm(ch, ah, 0x05040100u) ^ 0x80808080u);
}

// A block of 16 NR query rows of a sequence and kv head, as the B operands.
template <int KS, int NR>
struct DecQuery {
    int32x4 d[NR][3][KS];
    float f[NR];                // f 2^fe: score of one unit of Q code, times log2 e (without a
    int fe[NR];                 // page's scale it may leave the range of fp32)
    uint32_t hi[NR], lo[NR];
    uint32_t hi_min, hi_max, lo_min, lo_max;   // over the workgroup's rows

    __device__ __forceinline__ void load(const DecArgs &a, uint32_t s, uint32_t kh, uint32_t rb) {
        const uint32_t lane = threadIdx.x & 63, g4 = lane >> 4, D = a.c.dim;
        const uint32_t G = a.heads / a.c.heads, rows = a.tokens * G;
        const int64_t len = max(a.s.len[s], 0);
        const uint32_t cap = (uint32_t)min(len, (int64_t)a.s.stride * KV_B);
        auto see = [&](uint32_t t, uint32_t &h, uint32_t &l) {
            const int64_t end = max(len - a.tokens + t + 1, (int64_t)0);
            h = (uint32_t)min(end, (int64_t)cap);
            l = a.window && end > a.window ? (uint32_t)(end - a.window) : 0;
        };
        const uint32_t r0 = rb * 16 * NR, r1 = min(r0 + 16 * NR, rows) - 1;
        see(r0 / G, hi_min, lo_min);
        see(r1 / G, hi_max, lo_max);
#pragma unroll
        for (int n = 0; n < NR; n++) {
            const uint32_t r = min(r0 + 16 * n + (lane & 15), r1), t = r / G, h = kh * G + r % G;
            see(t, hi[n], lo[n]);
            const float *q = a.q + (((uint64_t)s * a.tokens + t) * a.heads + h) * D;
            floatx4 x[KS][4];
            float m = 0, bad = 0;
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t d = 64 * k + 16 * g4;
                    x[k][i] = d < D ? *(const floatx4 *)(q + d + 4 * i) : floatx4{0, 0, 0, 0};
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        m = fmaxf(m, fabsf(x[k][i][j]));
                        bad = fmaf(x[k][i][j], 0.0f, bad);  // NaN for an infinity or NaN
                    }
                }
            m = fmaxf(m, __shfl_xor(m, 16));
            m = fmaxf(m, __shfl_xor(m, 32));
            bad += __shfl_xor(bad, 16);
            bad += __shfl_xor(bad, 32);
            // m = c 2^e, c < 1: units of 2^(e - 23) where c 2^23 fits three digits (by exponents: no
            // fp32 number is the unit's inverse for every m)
            int e = __builtin_amdgcn_frexp_expf(m);
            e += __builtin_amdgcn_ldexpf(m, 23 - e) > DEC_P;
            const double c = (double)a.scale * LOG2E;
            f[n] = (float)__builtin_amdgcn_frexp_mant(c) + bad;
            fe[n] = __builtin_amdgcn_frexp_exp(c) + e - 23;
#pragma unroll
            for (int k = 0; k < KS; k++) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    uint32_t y[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) y[j] = (uint32_t)(__float2int_rn(__builtin_amdgcn_ldexpf(x[k][i][j], 23 - e)) + 0x808080);
                    int p0, p1, p2;
                    dec_digits(y[0], y[1], y[2], y[3], p0, p1, p2);
                    d[n][0][k][i] = p0;
                    d[n][1][k][i] = p1;
                    d[n][2][k][i] = p2;
                }
            }
        }
    }
};

// The keys of a page as the A operand: tile t, dimensions 64 k + 16 (lane / 16) ..
template <int KS>
__device__ __forceinline__ void dec_load_tile(int32x4 (&kk)[KS], int t, const int8_t *page, uint32_t D) {
    const uint32_t lane = threadIdx.x & 63;
    const int8_t *p = page + ((lane & 15) + 16 * t) * D;
#pragma unroll
    for (int k = 0; k < KS; k++)  // (past the end: bytes of the row that meet zero digits)
        kk[k] = *(const int32x4 *)(p + min(64 * k + 16 * (lane >> 4), D - 16));
}
template <int KS>
__device__ __forceinline__ void dec_load_k(int32x4 (&kk)[4][KS], const int8_t *page, uint32_t D) {
#pragma unroll
    for (int t = 0; t < 4; t++) dec_load_tile<KS>(kk[t], t, page, D);
}

// Scores of a page in units of log2, masked where the page is not wholly visible.
template <int KS, int NR>
__device__ __forceinline__ void dec_scores(float (&s)[NR][16], const int32x4 (&kk)[4][KS], const DecQuery<KS, NR> &q,
                                           float ks, uint32_t j0) {
    const uint32_t g4 = (threadIdx.x & 63) >> 4;
    const bool whole = j0 + KV_B <= q.hi_min && j0 >= q.lo_max;
#pragma unroll
    for (int n = 0; n < NR; n++) {
        const float f = __builtin_amdgcn_ldexpf(q.f[n] * ks, q.fe[n]);
#pragma unroll
        for (int t = 0; t < 4; t++) {
            int32x4 c0 = {0, 0, 0, 0}, c1 = c0, c2 = c0;
#pragma unroll
            for (int k = 0; k < KS; k++) {
                c0 = __builtin_amdgcn_mfma_i32_16x16x64_i8(kk[t][k], q.d[n][0][k], c0, 0, 0, 0);
                c1 = __builtin_amdgcn_mfma_i32_16x16x64_i8(kk[t][k], q.d[n][1][k], c1, 0, 0, 0);
                c2 = __builtin_amdgcn_mfma_i32_16x16x64_i8(kk[t][k], q.d[n][2][k], c2, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
                s[n][4 * t + i] = fmaf((float)c2[i], 65536.0f, (float)((c1[i] << 8) + c0[i])) * f;
        }
        if (!whole) {
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t j = j0 + 16 * t + 4 * g4 + i;
                    if (j < q.lo[n] || j >= q.hi[n]) s[n][4 * t + i] = -__builtin_inff();
                }
        }
    }
}

// The pages that the splits share out: those that some row of the block sees.
__device__ __forceinline__ uint2 dec_pages(uint32_t lo_min, uint32_t hi_max) {
    return {lo_min / KV_B, (hi_max + KV_B - 1) / KV_B};
}
__device__ __forceinline__ uint32_t dec_chunk(uint2 pg, uint32_t splits) {
    return pg.y > pg.x ? (pg.y - pg.x + splits - 1) / splits : 0;
}

// Grid: (row block, split, kv head, sequence) in one dimension, the row block
// slowest: blocks that read the same pages lie a multiple of 8 apart.
struct DecAt {
    uint32_t s, kh, split, rb;
    bool ok;
};
__device__ __forceinline__ DecAt dec_at(const DecArgs &a, uint32_t id) {
    const uint32_t per = (a.s.count * a.c.heads * a.splits + 7) / 8 * 8, rb = id / per, i = id % per;
    const uint32_t sh = i / a.splits;
    return {sh / a.c.heads, sh % a.c.heads, i % a.splits, rb, sh < a.s.count * a.c.heads};
}

// Visible pages of a block of rows, as its first and last row see them.
__device__ __forceinline__ uint2 dec_block_pages(const DecArgs &a, uint32_t s, uint32_t r0, uint32_t r1) {
    const uint32_t G = a.heads / a.c.heads;
    const int64_t len = max(a.s.len[s], 0);
    const uint32_t cap = (uint32_t)min(len, (int64_t)a.s.stride * KV_B);
    const int64_t e0 = max(len - a.tokens + r0 / G + 1, (int64_t)0), e1 = max(len - a.tokens + r1 / G + 1, (int64_t)0);
    return dec_pages(a.window && e0 > a.window ? (uint32_t)(e0 - a.window) : 0, (uint32_t)min(e1, (int64_t)cap));
}

// RB: the blocks of 16 rows that a workgroup's wavefronts are dealt to (1 or 2); the
// wavefronts of a block take its pages in turn.  (Both blocks in each wavefront, which
// reads every page once, takes 490 registers and the same time, 59 us for the longest
// case above.)
template <int KS, int RB>
__global__ __launch_bounds__(DEC_NT, KS <= 2 ? 2 : 1) void attn_dec_kernel(DecArgs a) {
    extern __shared__ __align__(16) float dec_lds[];  // [wave][16][dim + 4], then m and l [wave][16]
    float *const lds = dec_lds;
    constexpr uint32_t PW = DEC_W / RB;
    const DecAt at = dec_at(a, blockIdx.x);
    if (!at.ok) return;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), D = a.c.dim, g4 = lane >> 4;
    const uint32_t G = a.heads / a.c.heads, rows = a.tokens * G, r0 = at.rb * 16 * RB;
    DecQuery<KS, 1> q;
    q.load(a, at.s, at.kh, at.rb * RB + wave % RB);
    const uint2 pg = dec_block_pages(a, at.s, r0, min(r0 + 16 * RB, rows) - 1);
    const uint32_t chunk = dec_chunk(pg, a.splits);
    const uint32_t p0 = pg.x + at.split * chunk, p1 = min(p0 + chunk, pg.y);
    if (a.splits > 1 && p0 >= p1) return;  // (the joining kernel knows)
    floatx4 o[4 * KS] = {};
    float m = -__builtin_inff(), l = 0;
    const int32_t *pages = a.s.pages + (uint64_t)at.s * a.s.stride;
    const uint64_t pbytes = (uint64_t)KV_B * D;
    for (uint32_t b = p0 + wave / RB; b < p1; b += 64 * PW) {
        // page ids and scales of this wavefront's next 64 pages, one a lane
        const uint32_t mine = b + lane * PW;
        const int32_t id = mine < p1 ? pages[mine] : -1;
        const bool have = (uint32_t)id < a.c.pages;
        const uint64_t ph = have ? (uint64_t)id * a.c.heads + at.kh : 0;
        const float lks = have ? a.c.ks[ph] : 0, lvs = have ? a.c.vs[ph] : 0;
        uint64_t todo = __ballot(have);
        if (!todo) continue;
        int at_lane = __ffsll((unsigned long long)todo) - 1;
        auto base = [&](int ln) {
            const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)ph, ln), hi = __builtin_amdgcn_readlane((uint32_t)(ph >> 32), ln);
            return (((uint64_t)hi << 32) | lo) * pbytes;
        };
        int32x4 kk[4][KS];
        uint64_t off = base(at_lane);
        dec_load_k<KS>(kk, a.c.k + off, D);
        while (todo) {
            const uint32_t j0 = (b + at_lane * PW) * KV_B;
            const float ks = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(lks), at_lane));
            const float vs = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(lvs), at_lane));
            int32x4 vv[4 * KS];
            const int8_t *vp = a.c.v + off + (lane & 15) * KV_B + g4 * 16;
#pragma unroll
            for (int d = 0; d < 4 * KS; d++)
                if (16u * d < D) vv[d] = *(const int32x4 *)(vp + d * 1024);
            float s[1][16];
            dec_scores<KS, 1>(s, kk, q, ks, j0);
            todo &= todo - 1;
            if (todo) {
                at_lane = __ffsll((unsigned long long)todo) - 1;
                off = base(at_lane);
                dec_load_k<KS>(kk, a.c.k + off, D);
            }
            if (RB == 1 && a.sc && (lane & 15) < rows) {
                float *to = a.sc + (((uint64_t)at.s * a.c.heads + at.kh) * rows + (lane & 15)) * ((uint64_t)a.s.stride * KV_B) + j0 + 4 * g4;
#pragma unroll
                for (int t = 0; t < 4; t++) *(floatx4 *)(to + 16 * t) = floatx4{s[0][4 * t], s[0][4 * t + 1], s[0][4 * t + 2], s[0][4 * t + 3]};
            }
            float x = s[0][0];
#pragma unroll
            for (int i = 1; i < 16; i++) x = fmaxf(x, s[0][i]);
            x = fmaxf(x, __shfl_xor(x, 16));
            x = fmaxf(x, __shfl_xor(x, 32));
            const float nm = fmaxf(m, x), ref = nm == -__builtin_inff() ? 0.0f : nm;
            if (__ballot(nm > m)) {
                const float f = __builtin_amdgcn_exp2f(m - ref);
                l *= f;
#pragma unroll
                for (int d = 0; d < 4 * KS; d++) o[d] *= f;
            }
            m = nm;
            // weights of the page's own largest score, which g brings to the running one
            const float own = x == -__builtin_inff() ? 0.0f : x, g = __builtin_amdgcn_exp2f(x - ref);
            float lp = 0;
            int32x4 pd[3];
#pragma unroll
            for (int t = 0; t < 4; t++) {
                uint32_t y[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float p = __builtin_amdgcn_exp2f(s[0][4 * t + i] - own);
                    lp += p;
                    // (2^23 + P: P's rounding is the addition's, its digits the low three bytes)
                    y[i] = __float_as_uint(fmaf(p, DEC_P, 8388608.0f)) + 0x808080u;
                }
                int d0, d1, d2;
                dec_digits(y[0], y[1], y[2], y[3], d0, d1, d2);
                pd[0][t] = d0, pd[1][t] = d1, pd[2][t] = d2;
            }
            // (a row that sees nothing of the page takes nothing from it, a NaN scale neither)
            const float f = j0 < q.hi[0] && j0 + KV_B > q.lo[0] ? vs * g : 0.0f;
            l = fmaf(lp, g, l);
#pragma unroll
            for (int d = 0; d < 4 * KS; d++)
                if (16u * d < D) {
                    const int32x4 z = {0, 0, 0, 0};
                    const int32x4 c0 = __builtin_amdgcn_mfma_i32_16x16x64_i8(vv[d], pd[0], z, 0, 0, 0);
                    const int32x4 c1 = __builtin_amdgcn_mfma_i32_16x16x64_i8(vv[d], pd[1], z, 0, 0, 0);
                    const int32x4 c2 = __builtin_amdgcn_mfma_i32_16x16x64_i8(vv[d], pd[2], z, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        o[d][i] += fmaf((float)c2[i], 65536.0f, (float)((c1[i] << 8) + c0[i])) * f;
                }
        }
    }
    // the wavefronts' results joined
    const uint32_t row = D + 4;
    float *lm = lds + DEC_W * 16 * row;
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (lane < 16) {
        lm[wave * 32 + lane] = m;
        lm[wave * 32 + 16 + lane] = l;
    }
    float *p = lds + (wave * 16 + (lane & 15)) * row + 4 * g4;
#pragma unroll
    for (int d = 0; d < 4 * KS; d++)
        if (16u * d < D) *(floatx4 *)(p + 16 * d) = o[d];
    __syncthreads();
    const uint32_t n_rows = min(rows - r0, 16u * RB);
    const uint64_t seg = ((uint64_t)at.rb * a.s.count * a.c.heads + at.s * a.c.heads + at.kh) * a.splits + at.split;
    for (uint32_t e = threadIdx.x; e < n_rows * (D / 4); e += DEC_NT) {
        const uint32_t r = e / (D / 4), d = e % (D / 4) * 4;
        float top = -__builtin_inff();
#pragma unroll
        for (uint32_t w = 0; w < PW; w++) top = fmaxf(top, lm[(w * RB + r / 16) * 32 + r % 16]);
        const float ref = top == -__builtin_inff() ? 0.0f : top;
        floatx4 sum = {0, 0, 0, 0};
        float ls = 0;
#pragma unroll
        for (uint32_t w = 0; w < PW; w++) {
            const uint32_t n = w * RB + r / 16;
            const float f = __builtin_amdgcn_exp2f(lm[n * 32 + r % 16] - ref);
            sum += *(const floatx4 *)(lds + (n * 16 + r % 16) * row + d) * f;
            ls += lm[n * 32 + 16 + r % 16] * f;
        }
        sum *= 1.0f / DEC_P;
        if (a.ml && d == 0) {
            a.ml[(seg * 16 * RB + r) * 2] = top;
            a.ml[(seg * 16 * RB + r) * 2 + 1] = ls;
        }
        if (a.splits > 1) {
            *(floatx4 *)(a.part + (seg * 16 * RB + r) * D + d) = sum;
        } else {
            const uint32_t rr = r0 + r;
            float *out = a.o + (((uint64_t)at.s * a.tokens + rr / G) * a.heads + at.kh * G + rr % G) * D + d;
            *(floatx4 *)out = ls != 0 ? sum * (1.0f / ls) : floatx4{0, 0, 0, 0};
        }
    }
}

// Joins the splits: one workgroup a query row (query token and head).  The splits'
// factors first, a thread each; then threads take four dimensions of every (1024 /
// dim)-th split, four of them under way.
constexpr uint32_t DEC_SPLITS = 1024;
__device__ __forceinline__ void dec_join(const DecArgs &a, uint32_t rpb) {
    __shared__ __align__(16) float acc[DEC_NT * 4];
    __shared__ float w[DEC_SPLITS], red[2 * DEC_W];
    const uint32_t G = a.heads / a.c.heads, rows = a.tokens * G, D = a.c.dim, tid = threadIdx.x;
    const uint32_t r = blockIdx.x % rows, sh = blockIdx.x / rows, s = sh / a.c.heads, kh = sh % a.c.heads;
    const uint32_t rb = r / rpb, r0 = rb * rpb;
    const uint2 pg = dec_block_pages(a, s, r0, min(r0 + rpb, rows) - 1);
    const uint32_t chunk = dec_chunk(pg, a.splits), ns = chunk ? (pg.y - pg.x + chunk - 1) / chunk : 0;
    const uint64_t seg = ((uint64_t)rb * a.s.count * a.c.heads + sh) * a.splits;
    const float2 *ml = (const float2 *)a.ml + seg * rpb + (r - r0);
    float2 x[DEC_SPLITS / DEC_NT];
    float top = -__builtin_inff(), ls = 0;
#pragma unroll
    for (uint32_t i = 0; i < DEC_SPLITS / DEC_NT; i++) {
        const uint32_t j = tid + i * DEC_NT;
        x[i] = j < ns ? ml[(uint64_t)j * rpb] : float2{-__builtin_inff(), 0};
        top = fmaxf(top, x[i].x);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if ((tid & 63) == 0) red[tid >> 6] = top;
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < DEC_W; i++) top = fmaxf(top, red[i]);
    const float ref = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
    for (uint32_t i = 0; i < DEC_SPLITS / DEC_NT; i++) {
        const float f = __builtin_amdgcn_exp2f(x[i].x - ref);
        w[tid + i * DEC_NT] = f;
        ls += x[i].y * f;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) ls += __shfl_xor(ls, o);
    if ((tid & 63) == 0) red[DEC_W + (tid >> 6)] = ls;
    __syncthreads();
    ls = red[DEC_W];
#pragma unroll
    for (uint32_t i = 1; i < DEC_W; i++) ls += red[DEC_W + i];
    const uint32_t q4 = D / 4, groups = DEC_NT / q4, g = tid / q4, d = tid % q4 * 4;
    floatx4 sum = {0, 0, 0, 0};
    if (g < groups) {
        const float *part = a.part + (seg * rpb + (r - r0)) * D + d;
        for (uint32_t i = g; i < ns; i += 4 * groups) {
            floatx4 y[4];
#pragma unroll
            for (uint32_t u = 0; u < 4; u++) y[u] = *(const floatx4 *)(part + (uint64_t)min(i + u * groups, ns - 1) * rpb * D);
#pragma unroll
            for (uint32_t u = 0; u < 4; u++)
                if (i + u * groups < ns) sum += y[u] * w[i + u * groups];
        }
    }
    *(floatx4 *)(acc + tid * 4) = sum;
    __syncthreads();
    if (tid < q4) {
        for (uint32_t i = 1; i < groups; i++) sum += *(const floatx4 *)(acc + (i * q4 + tid) * 4);
        float *out = a.o + (((uint64_t)s * a.tokens + r / G) * a.heads + kh * G + r % G) * D + d;
        *(floatx4 *)out = ls != 0 ? sum * (1.0f / ls) : floatx4{0, 0, 0, 0};
    }
}

__global__ __launch_bounds__(DEC_NT) void attn_dec_join_kernel(DecArgs a, uint32_t rpb) { dec_join(a, rpb); }

// x of the lane N before this one in its row of 16, around.
template <int N>
__device__ __forceinline__ float dec_ror(float x) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), 0x120 + N, 0xF, 0xF, false));
}

// Accumulated attention weights from the scores that attn_dec_kernel has left (up to 16
// query rows): the rows' maxima and sums over the splits first, a wavefront a row, then a
// thread a token.
__global__ __launch_bounds__(DEC_NT) void attn_dec_sum_kernel(DecArgs a, uint32_t parts, uint32_t joins) {
    if (blockIdx.x < joins) return dec_join(a, 16);  // (the splits' results beside them)
    __shared__ float top_of[16], inv_of[16];
    const uint32_t id_ = blockIdx.x - joins, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t sh = id_ / parts, s = sh / a.c.heads, part = id_ % parts;
    const uint32_t cap = (uint32_t)min((uint64_t)max(a.s.len[s], 0), (uint64_t)a.s.stride * KV_B);
    const uint32_t rows = a.tokens * (a.heads / a.c.heads);
    const uint2 pg = dec_block_pages(a, s, 0, rows - 1);
    const uint32_t ch = dec_chunk(pg, a.splits), ns = ch ? (pg.y - pg.x + ch - 1) / ch : 0;
    for (uint32_t r = wave; r < rows; r += DEC_W) {
        const float2 *ml = (const float2 *)a.ml + (uint64_t)sh * a.splits * 16 + r;
        float top = -__builtin_inff(), ls = 0;
        for (uint32_t i = lane; i < ns; i += 64) top = fmaxf(top, ml[i * 16].x);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        const float ref = top == -__builtin_inff() ? 0.0f : top;
        for (uint32_t i = lane; i < ns; i += 64) ls += ml[i * 16].y * __builtin_amdgcn_exp2f(ml[i * 16].x - ref);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) ls += __shfl_xor(ls, o);
        if (lane == 0) top_of[r] = ref, inv_of[r] = ls != 0 ? 1.0f / ls : 0.0f;
    }
    __syncthreads();
    const uint64_t row = (uint64_t)a.s.stride * KV_B;
    const int32_t *pages = a.s.pages + (uint64_t)s * a.s.stride;
    const float *sc = a.sc + (uint64_t)sh * rows * row, *wi = a.w_in ? a.w_in + (uint64_t)sh * a.wst : nullptr;
    float *wo = a.w_out + (uint64_t)sh * a.wst;
    for (uint64_t j = part * DEC_NT + threadIdx.x; j < cap; j += (uint64_t)parts * DEC_NT) {
        const uint32_t p = j / KV_B;
        float w = 0;
        if ((uint32_t)pages[p] < a.c.pages && p >= pg.x && p < pg.y)
            for (uint32_t r = 0; r < rows; r++) {
                const float x = sc[r * row + j];
                // (unseen tokens get nothing of a row whose sum is NaN)
                w += x != -__builtin_inff() ? __builtin_amdgcn_exp2f(x - top_of[r]) * inv_of[r] : 0.0f;
            }
        wo[j] = (wi ? wi[j] : 0.0f) + w;
    }
}

// Accumulated attention weights: a wavefront a page, the scores computed again
// from the keys, for every block of query rows: where the scores have not been kept.
template <int KS, int NR>
__global__ __launch_bounds__(DEC_NT, KS <= 2 ? 2 : 1) void attn_dec_weights_kernel(DecArgs a, uint32_t parts, uint32_t joins) {
    if (blockIdx.x < joins) return dec_join(a, 16 * NR);  // (the splits' results beside them)
    const uint32_t id_ = blockIdx.x - joins;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, D = a.c.dim, g4 = lane >> 4;
    const uint32_t sh = id_ / parts, s = sh / a.c.heads, kh = sh % a.c.heads, part = id_ % parts;
    const uint32_t cap = (uint32_t)min((uint64_t)max(a.s.len[s], 0), (uint64_t)a.s.stride * KV_B);
    const uint32_t np = (cap + KV_B - 1) / KV_B, chunk = (np + parts - 1) / parts;
    const uint32_t rows = a.tokens * (a.heads / a.c.heads);
    const int32_t *pages = a.s.pages + (uint64_t)s * a.s.stride;
    const float *wi = a.w_in ? a.w_in + (uint64_t)sh * a.wst : nullptr;
    float *wo = a.w_out + (uint64_t)sh * a.wst;
    for (uint32_t rb = 0; rb < a.rb; rb++) {
        DecQuery<KS, NR> q;
        q.load(a, s, kh, rb);
        // maximum and sum over the splits, for this lane's rows
        const uint2 pg = dec_pages(q.lo_min, q.hi_max);
        const uint32_t ch = dec_chunk(pg, a.splits), ns = ch ? (pg.y - pg.x + ch - 1) / ch : 0;
        const uint64_t seg = ((uint64_t)rb * a.s.count * a.c.heads + sh) * a.splits;
        float ref[NR], inv[NR];
#pragma unroll
        for (int n = 0; n < NR; n++) {
            const bool valid = rb * 16 * NR + 16 * n + (lane & 15) < rows;
            const float *ml = a.ml + (seg * 16 * NR + 16 * n + (lane & 15)) * 2;
            float top = -__builtin_inff(), ls = 0;
            if (valid)
                for (uint32_t i = g4; i < ns; i += 4) top = fmaxf(top, ml[(uint64_t)i * 32 * NR]);
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            ref[n] = top == -__builtin_inff() ? 0.0f : top;
            if (valid)
                for (uint32_t i = g4; i < ns; i += 4)
                    ls += ml[(uint64_t)i * 32 * NR + 1] * __builtin_amdgcn_exp2f(ml[(uint64_t)i * 32 * NR] - ref[n]);
            ls += __shfl_xor(ls, 16);
            ls += __shfl_xor(ls, 32);
            inv[n] = valid && ls != 0 ? 1.0f / ls : 0.0f;
        }
        const uint32_t p1 = min((part + 1) * chunk, np);
        for (uint32_t b = part * chunk + wave; b < p1; b += 64 * DEC_W) {
            // page ids and scales of this wavefront's next 64 pages, one a lane
            const uint32_t mine = b + lane * DEC_W, pages_here = min((p1 - b + DEC_W - 1) / DEC_W, 64u);
            const int32_t id = mine < p1 ? pages[mine] : -1;
            const bool have = (uint32_t)id < a.c.pages && mine * KV_B < q.hi_max && mine * KV_B + KV_B > q.lo_min;
            const uint64_t ph = have ? (uint64_t)id * a.c.heads + kh : 0;
            const float lks = have ? a.c.ks[ph] : 0;
            const uint64_t live = __ballot(have);
            auto keys = [&](int32x4 (&kk)[4][KS], uint32_t u) {
                if (u >= pages_here || !(live >> u & 1)) return;
                const uint64_t at = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(ph >> 32), u) << 32 | (uint32_t)__builtin_amdgcn_readlane((uint32_t)ph, u);
                dec_load_k<KS>(kk, a.c.k + at * KV_B * D, D);
            };
            int32x4 kk[4][KS];
            keys(kk, 0);
            for (uint32_t u = 0; u < pages_here; u++) {
                // lane (g, r) has the token 16 (r / 4) + 4 g + r % 4 of the page
                const uint32_t j0 = (b + u * DEC_W) * KV_B, r = lane & 15, j = j0 + 16 * (r / 4) + 4 * g4 + r % 4;
                const bool here = j < cap;
                const float was = !here ? 0.0f : rb ? wo[j] : wi ? wi[j] : 0.0f;
                float w = 0;
                if (live >> u & 1) {
                    float sc[NR][16];
                    dec_scores<KS, NR>(sc, kk, q, __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(lks), u)), j0);
                    keys(kk, u + 1);
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        float sum = 0;
#pragma unroll
                        for (int n = 0; n < NR; n++) {
                            const float e = __builtin_amdgcn_exp2f(sc[n][i] - ref[n]) * inv[n];
                            // (unseen tokens get nothing of a row whose sum is NaN; rows that are not there count 0)
                            sum += inv[n] != 0 && sc[n][i] != -__builtin_inff() ? e : 0.0f;
                        }
                        // the sixteen lanes of the group added up, in all of them
                        sum += dec_ror<8>(sum);
                        sum += dec_ror<4>(sum);
                        sum += dec_ror<2>(sum);
                        sum += dec_ror<1>(sum);
                        w = (int)r == i ? sum : w;
                    }
                } else {
                    keys(kk, u + 1);
                }
                if (here) wo[j] = was + w;
            }
        }
    }
}

}  // namespace okf
