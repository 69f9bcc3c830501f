// okf_delta_scan.h -- the gated delta rule in chunks of 32 tokens on the matrix cores
// (okf_delta_prompt).
//
// With G the running sum of g in a chunk, S the state in front of it and
//   A_ij = beta_i e^(G_i - G_j) k_i.k_j (j < i),   T = (I + A)^-1 diag(beta),
//   P_ij = e^(G_i - G_j) q_i.k_j (j <= i)
// the chunk's corrections, outputs and the state behind it are
//   U = T (V - e^G K S),   O = scale (e^G Q S + P U),   S' = e^G_last S + K^T (e^(G_last - G) U).
// delta_prepare_kernel computes T and P of every chunk at once and leaves them, with K, Q and K^T, in
// scratch as the operands of the matrix instruction; delta_scan_kernel goes through each
// sequence's chunks one behind the other with the state in registers.
//
// Precision: every product has fp32's.  An fp32 value is three bf16 parts (x = x0 + x1 + x2
// exactly, each what is left rounded to nearest), f16 inputs are two, bf16 one; of the products of parts those that
// come to less than 2^-24 of the whole, of either sign, are left out: |x1| <= 2^-8 and |x2| <= 2^-17 of a power of two
// that |x| reaches, so x1 y2 + x2 y1 + x2 y2.  (Parts that are cut off have the sign of x, and what is left out
// reaches 2^-21, 0.7 2^-24 on average.)  G and its differences are in 64 bits, so that
// decays far apart keep their ratios.  (I + A)^-1 comes from forward substitution, which
// is as stable as the recurrence; powers of A are not.
//
// Where something is not finite, 0 times it in the places that a mask or the order of tokens
// leaves out would spread it to earlier tokens: columns whose corrections show any are gone through
// again token by token.  (A chunk whose queries are not finite has its T spoilt, so that it shows.  Values
// from 2^127 on count as not finite: those next to the type's end have no first part.)
#pragma once
#include <utility>

#include "okf_delta.h"

namespace okf {

constexpr uint32_t DC = 32;                     // tokens a chunk
constexpr uint32_t DV_BYTES = 12 * 1024 + 256;  // scratch of a chunk and value head: T, P; e^G, e^(G_last - G)

typedef __bf16 bf16x8d __attribute__((ext_vector_type(8)));

template <class T>
__host__ __device__ constexpr int dl_parts() { return sizeof(T) == 4 ? 3 : std::is_same<T, _Float16>::value ? 2 : 1; }
// scratch of a chunk and key head: K, Q and K^T in their parts, 32 dimensions 6 KB
__host__ __device__ constexpr uint32_t dl_kq_bytes(int parts, uint32_t k_dim) { return parts * ((k_dim + 31) / 32) * 6144; }

struct ScanArgs {
    DeltaArgs a;
    uint8_t *k_work, *v_work;  // of the chunks c0 .. c1 - 1: [k_heads][at_once][kq], [v_heads][at_once][DV_BYTES]: a head's
                               // chunks, which a workgroup goes through, side by side
    uint32_t kq, passes;       // passes: pairs of value heads of a key head
    uint32_t c0, c1, at_once;
    const float *carry_in;  // the state of the sequence that chunk c0 - 1 belongs to
    float *carry_out;       // that of the one that goes on behind c1
};

__device__ __forceinline__ uint32_t dl_chunks(const StateSeqs &s, uint32_t i) {
    const uint2 r = kv_rows(s.start, i, s.n);
    return (r.y - r.x + DC - 1) / DC;
}
// The chunks of the sequences before sequence `seq`.
__device__ __forceinline__ uint32_t dl_before(const StateSeqs &s, uint32_t seq) {
    uint32_t sum = 0;
    for (uint32_t b = 0; b < seq; b += 64) {
        const uint32_t i = b + (threadIdx.x & 63);
        sum += (uint32_t)__builtin_amdgcn_readlane(lanes_sum(i < seq ? dl_chunks(s, i) : 0), 63);
    }
    return sum;
}

// Two floats as bf16, rounded to nearest even, a in the lower half; and the lower's and the upper's value.
typedef __bf16 bf16x2d __attribute__((ext_vector_type(2)));
typedef float floatx2d __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t dl_round(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((floatx2d{a, b}), bf16x2d));
}
__device__ __forceinline__ float dl_lower(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float dl_upper(uint32_t p) { return __uint_as_float(p & 0xFFFF0000u); }

// Eight floats -> NP bf16 parts of each.
template <int NP>
__device__ __forceinline__ void dl_split(const float (&x)[8], bf16x8d (&p)[NP]) {
    u32x4 out[NP];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        float a = x[2 * j], b = x[2 * j + 1];
#pragma unroll
        for (int n = 0; n < NP; n++) {
            out[n][j] = dl_round(a, b);
            if (n < NP - 1) a -= dl_lower(out[n][j]), b -= dl_upper(out[n][j]);
        }
    }
#pragma unroll
    for (int n = 0; n < NP; n++) p[n] = __builtin_bit_cast(bf16x8d, out[n]);
}

// The parts of two results below each other, as the B operand of the next product, step by step: dl_top rounds
// every value to its first part, what that leaves is the value less it, for one of the four
// values of both in dl_rest; or from the matrix cores, -1 times the part added to the value (exact: the
// difference has fewer bits).
struct DlMinus {
    bf16x8d a[2];  // -1 times the identity: of the upper and of the lower result's rows
    __device__ __forceinline__ DlMinus(uint32_t m, uint32_t h) {
#pragma unroll
        for (uint32_t j = 0; j < 8; j++)
#pragma unroll
            for (uint32_t t = 0; t < 2; t++) a[t][j] = (__bf16)(j / 4 == t && 4 * h + j % 4 == m ? -1.0f : 0.0f);
    }
};
__device__ __forceinline__ bf16x8d dl_top(floatx4 x, floatx4 y) {
    u32x4 p;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float a = j < 2 ? x[2 * j] : y[2 * j - 4], b = j < 2 ? x[2 * j + 1] : y[2 * j - 3];
        p[j] = dl_round(a, b);
    }
    return __builtin_bit_cast(bf16x8d, p);
}
__device__ __forceinline__ void dl_rest(floatx4 &x, floatx4 &y, bf16x8d part, int j) {
    const u32x4 p = __builtin_bit_cast(u32x4, part);
    const uint32_t px = p[j / 2], py = p[2 + j / 2];
    x[j] -= j % 2 ? dl_upper(px) : dl_lower(px);
    y[j] -= j % 2 ? dl_upper(py) : dl_lower(py);
}
__device__ __forceinline__ void dl_split(floatx4 x, floatx4 y, bf16x8d (&p)[3]) {
#pragma unroll
    for (int n = 0; n < 3; n++) {
        p[n] = dl_top(x, y);
#pragma unroll
        for (int j = 0; n < 2 && j < 4; j++) dl_rest(x, y, p[n], j);
    }
}
__device__ __forceinline__ floatx4 dl_mfma(bf16x8d a, bf16x8d b, floatx4 d) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, d, 0, 0, 0); }
// the parts of an operand of NP whose products with the other's part j count
template <int NP>
__host__ __device__ constexpr int dl_with(int j) { return NP < 3 - j ? NP : 3 - j; }

// f of every constant below N.
template <class F, int... I>
__device__ __forceinline__ void dl_each_of(F f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void dl_each(F f) {
    dl_each_of(f, std::make_integer_sequence<int, N>{});
}

// M matrix instructions and V bundles of vector instructions in turn, in this very order.  A wavefront issues
// in order, and a matrix instruction runs for as long as four vector instructions take to issue; the compiler's
// own order left the chain of products at twice the time.
template <int M, int V, class FM, class FV>
__device__ __forceinline__ void dl_zip(FM matrix, FV vector) {
    if constexpr (M == 0) {
#pragma unroll
        for (int v = 0; v < V; v++) vector(v);
    } else {
#pragma unroll
        for (int i = 0; i < M; i++) {
            matrix(i);
#pragma unroll
            for (int v = i * V / M; v < (i + 1) * V / M; v++) vector(v);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
}

// d + a b over the parts of both whose product counts.
template <int NA, int NB>
__device__ __forceinline__ floatx4 dl_mma(const bf16x8d (&a)[NA], const bf16x8d (&b)[NB], floatx4 d) {
#pragma unroll
    for (int i = 0; i < NA; i++)
#pragma unroll
        for (int j = 0; j < NB; j++)
            if (i + j <= 2) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[j], d, 0, 0, 0);
    return d;
}

// The operand layout (v_mfma_f32_16x16x32): lane l holds row (A) or column (B) l % 16 and, h = l / 16, of 32
// terms those at 4 h + 0..3 and 16 + 4 h + 0..3; the result's column l % 16 and rows 4 h + 0..3.
// So two results below each other are the B operand of the next product as they lie.

// Two fours of T, as parts.
template <class T, int NP>
__device__ __forceinline__ void dl_operand(const T *lo, const T *hi, bool on_lo, bool on_hi, bf16x8d (&p)[NP]) {
    typedef T vec __attribute__((ext_vector_type(4)));
    vec a, b;
#pragma unroll
    for (int j = 0; j < 4; j++) a[j] = b[j] = (T)0.0f;
    if (on_lo) a = *(const vec *)lo;
    if (on_hi) b = *(const vec *)hi;
    if constexpr (NP == 1) {
#pragma unroll
        for (int j = 0; j < 4; j++) p[0][j] = a[j], p[0][4 + j] = b[j];
    } else {
        float x[8];
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = to_f32(a[j]), x[4 + j] = to_f32(b[j]);
        dl_split<NP>(x, p);
    }
}

// The parts of four terms, and d + a b over 16 of them (v_mfma_f32_16x16x16: lane l holds the terms 4 h + 0..3).
typedef short shortx4d __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void dl_split4(floatx4 x, shortx4d (&p)[3]) {
#pragma unroll
    for (int n = 0; n < 3; n++) {
        const uint2 t = {dl_round(x[0], x[1]), dl_round(x[2], x[3])};
        p[n] = __builtin_bit_cast(shortx4d, t);
        x -= floatx4{dl_lower(t.x), dl_upper(t.x), dl_lower(t.y), dl_upper(t.y)};
    }
}
__device__ __forceinline__ floatx4 dl_mma16(floatx4 x, floatx4 y) {
    shortx4d a[3], b[3];
    dl_split4(x, a);
    dl_split4(y, b);
    floatx4 d = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 3; i++)
#pragma unroll
        for (int j = 0; i + j <= 2; j++) d = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a[i], b[j], d, 0, 0, 0);
    return d;
}

constexpr int DP_NT = 256;
constexpr uint32_t DP_ROW = 20;  // floats from a row of a 16 x 16 matrix in LDS to the next: 16-byte rows on different banks

// A wavefront takes a chunk, a key head and two of its value heads.  k k^T and q k^T come from the matrix cores
// with the later token in the lane's column, so that P lies as the next product takes it; K^T is K
// times the identity, whose result lies as an operand too.  (I + A)^-1 in 2 x 2 blocks of 16: those on the diagonal by
// substitution from the right (t_j = delta_ij - sum_l>j t_l A_lj), both of both heads at once, a row a lane; the lower one
// as -T22 (A21 T11).  Many chunks are bound by memory: 8192 tokens of 16 key and 48 value heads of 128, bf16, 76 us for 128 MB in
// and 255 MB of scratch out (fp32 113, 456 MB out); few by the chain itself, 15 us (K, Q and K^T laid out by other wavefronts: 14, many chunks 88 for 77).
template <class T, int KS>
__global__ __launch_bounds__(DP_NT) void delta_prepare_kernel(const ScanArgs p) {
    constexpr int NP = dl_parts<T>();
    const DeltaArgs &a = p.a;
    __shared__ __align__(16) float mat[DP_NT / 64][2][2][2][16 * DP_ROW];  // [A^T, T][value head][block]
    __shared__ __align__(16) double gam[DP_NT / 64][2][DC];
    __shared__ __align__(16) float bet[DP_NT / 64][2][DC];
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63, m = lane & 15, h = lane >> 4;
    const uint32_t w = blockIdx.x * (DP_NT / 64) + wave, pass = w % p.passes, kh = w / p.passes % a.k_heads;
    const uint32_t chunk = p.c0 + w / p.passes / a.k_heads;
    if (chunk >= p.c1) return;
    const SeqItem it = kv_find(chunk, a.s.count, [&](uint32_t s) { return dl_chunks(a.s, s); });
    if (it.seq >= a.s.count) return;
    const uint2 r = kv_rows(a.s.start, it.seq, a.s.n);
    const uint32_t first = r.x + it.at * DC, n = min(r.y - first, DC);
    if (first >= r.y) return;  // (not with starts that rise)
    bf16x8d *kq = (bf16x8d *)(p.k_work + ((uint64_t)kh * p.at_once + (chunk - p.c0)) * p.kq);
    auto vb = [&](uint32_t head) { return p.v_work + ((uint64_t)head * p.at_once + (chunk - p.c0)) * DV_BYTES; };
    const T *q = (const T *)a.q + kh * a.k_dim, *k = (const T *)a.k + kh * a.k_dim;
    // running decays: each half of the lanes a value head
    const uint32_t half = lane >> 5, j = lane & 31, group = a.v_heads / a.k_heads, heads = min(group - pass * 2, 2u);
    const uint32_t vh = kh * group + pass * 2;
    double G = 0;
    float beta = 0;
    if (j < n && half < heads) {
        const double g = (double)a.g[(uint64_t)(first + j) * a.gs + vh + half] * 1.4426950408889634;
        G = g < -1e5 ? -1e5 : g;  // (2^-1e5 is 0; -inf would leave inf - inf behind it)
        beta = a.beta[(uint64_t)(first + j) * a.bs + vh + half];
    }
    floatx4 kk[3] = {}, qk[3] = {};  // earlier and later tokens of tiles (0, 0), (0, 1), (1, 1)
#pragma unroll 1
    for (int ks = 0; ks < KS; ks++) {
        bf16x8d kp[2][NP], qp[2][NP];
#pragma unroll
        for (int mt = 0; mt < 2; mt++) {
            const uint32_t row = mt * 16 + m, d = 32 * ks + 4 * h;
            const bool lo = row < n && d < a.k_dim, hi = row < n && d + 16 < a.k_dim;
            const uint64_t at = first + row;
            dl_operand<T, NP>(k + at * a.ks + d, k + at * a.ks + d + 16, lo, hi, kp[mt]);
            dl_operand<T, NP>(q + at * a.qs + d, q + at * a.qs + d + 16, lo, hi, qp[mt]);
            if (pass == 0) {
#pragma unroll
                for (int i = 0; i < NP; i++) {
                    kq[((i * 2 + mt) * KS + ks) * 64 + lane] = kp[mt][i];
                    kq[(((NP + i) * 2 + mt) * KS + ks) * 64 + lane] = qp[mt][i];
                }
            }
        }
#pragma unroll
        for (int t = 0; t < 3; t++) {
            kk[t] = dl_mma(kp[t > 1], kp[t > 0], kk[t]);
            qk[t] = dl_mma(kp[t > 1], qp[t > 0], qk[t]);
        }
        if (pass == 0) {  // K^T
#pragma unroll
            for (int t = 0; t < 2; t++) {
                bf16x8d one;
#pragma unroll
                for (uint32_t l = 0; l < 8; l++) one[l] = (__bf16)(l / 4 == (uint32_t)t && 4 * h + l % 4 == m ? 1.0f : 0.0f);
#pragma unroll
                for (int i = 0; i < NP; i++) {
                    const floatx4 zero = {0, 0, 0, 0};
                    kq[NP * 4 * KS * 64 + (i * 2 * KS + 2 * ks + t) * 64 + lane] = dl_top(dl_mfma(kp[0][i], one, zero), dl_mfma(kp[1][i], one, zero));
                }
            }
        }
    }
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const double up = __shfl_up(G, o, 32);
        if (j >= (uint32_t)o) G += up;
    }
    gam[wave][half][j] = G;
    bet[wave][half][j] = beta;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (half < heads) {
        float *eg = (float *)(vb(vh + half) + 12 * 1024);
        eg[j] = __builtin_amdgcn_exp2f((float)G);
        eg[DC + j] = __builtin_amdgcn_exp2f((float)(gam[wave][half][DC - 1] - G));
    }
    floatx4 a21[2], P[2][3];
#pragma unroll
    for (uint32_t z = 0; z < 2; z++) {
        const double *gz = gam[wave][z];
        const float *bz = bet[wave][z];
#pragma unroll
        for (int t = 0; t < 3; t++) {
            const uint32_t late = (t > 0) * 16 + m, early = (t > 1) * 16 + 4 * h;
            const double gl = gz[late];
            const float bl = bz[late];
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
                const float e = __builtin_amdgcn_exp2f((float)(gl - gz[early + i]));
                const bool before = t == 1 || 4 * h + i < m;
                const float A = before ? bl * (e * kk[t][i]) : 0.0f;
                P[z][t][i] = before || (t != 1 && 4 * h + i == m) ? e * qk[t][i] : 0.0f;
                if (t == 1) a21[z][i] = A;
                else mat[wave][0][z][t > 1][(4 * h + i) * DP_ROW + m] = A;
            }
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    {
        const uint32_t z = lane >> 5, blk = lane >> 4 & 1;
        const float *At = mat[wave][0][z][blk];
        float t[16];
#pragma unroll
        for (int c = 15; c >= 0; c--) {
            float s = m == (uint32_t)c ? 1.0f : 0.0f;
#pragma unroll
            for (int l4 = (c + 1) / 4; l4 < 4; l4++) {
                const floatx4 x = *(const floatx4 *)(At + c * DP_ROW + 4 * l4);
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (4 * l4 + i > c) s = fmaf(-t[4 * l4 + i], x[i], s);
            }
            t[c] = s;
        }
        float *to = mat[wave][1][z][blk] + m * DP_ROW;
#pragma unroll
        for (int c = 0; c < 16; c += 4) *(floatx4 *)(to + c) = floatx4{t[c], t[c + 1], t[c + 2], t[c + 3]};
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (uint32_t z = 0; z < 2; z++) {
        if (z >= heads) break;
        const float *t11 = mat[wave][1][z][0], *t22 = mat[wave][1][z][1], *bz = bet[wave][z];
        const floatx4 r11 = *(const floatx4 *)(t11 + m * DP_ROW + 4 * h), r22 = *(const floatx4 *)(t22 + m * DP_ROW + 4 * h);
        floatx4 c11;
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) c11[i] = t11[(4 * h + i) * DP_ROW + m];
        const floatx4 x = dl_mma16(r22, dl_mma16(a21[z], c11));  // (rows of results to columns, through LDS)
        float *turn = mat[wave][0][z][0];
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) turn[(4 * h + i) * DP_ROW + m] = -x[i];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const floatx4 r21 = *(const floatx4 *)(turn + m * DP_ROW + 4 * h);
        const floatx4 b0 = *(const floatx4 *)(bz + 4 * h), b1 = *(const floatx4 *)(bz + 16 + 4 * h), zero = {0, 0, 0, 0};
        float bad = 0;
#pragma unroll
        for (int t = 0; t < 3; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) bad = fmaf(2 * P[z][t][i], 0.0f, bad);
        floatx4 lo = r11 * b0;
        if (__ballot(bad != bad)) lo[0] = __builtin_nanf("");
        bf16x8d *to = (bf16x8d *)vb(vh + z) + lane;
        bf16x8d part[4][3];
        dl_split(lo, zero, part[0]);
        dl_split(r21 * b0, r22 * b1, part[1]);
        dl_split(P[z][0], zero, part[2]);
        dl_split(P[z][1], P[z][2], part[3]);
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < 3; i++) to[(t / 2 * 6 + i * 2 + t % 2) * 64] = part[t][i];
    }
}

// The tokens first .. first + n - 1 one by one: S of a lane in the layout of results (rows dt * 16 + 4 h + i,
// column `col`).
template <class T, int KS>
__device__ __forceinline__ void dl_tokens(const DeltaArgs &a, uint32_t kh, uint32_t vh, uint32_t col, uint32_t h, uint32_t first, uint32_t n,
                                          floatx4 (&S)[2 * KS]) {
    const T *q = (const T *)a.q + kh * a.k_dim + 4 * h, *k = (const T *)a.k + kh * a.k_dim + 4 * h;
#pragma unroll 1
    for (uint64_t t = first; t < (uint64_t)first + n; t++) {
        const float e = expf(a.g[t * a.gs + vh]), beta = a.beta[t * a.bs + vh], v = to_f32(((const T *)a.v)[t * a.vs + vh * a.v_dim + col]);
        float kr = 0, qr = 0;
#pragma unroll
        for (int dt = 0; dt < 2 * KS; dt++)
            if (dt * 16 < (int)a.k_dim)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    S[dt][i] = e == 0 ? 0.0f : e * S[dt][i];
                    kr = fmaf(to_f32(k[t * a.ks + dt * 16 + i]), S[dt][i], kr);
                }
        const float u = beta * (v - dl_sum_rows(kr));
#pragma unroll
        for (int dt = 0; dt < 2 * KS; dt++)
            if (dt * 16 < (int)a.k_dim)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    S[dt][i] = fmaf(to_f32(k[t * a.ks + dt * 16 + i]), u, S[dt][i]);
                    qr = fmaf(to_f32(q[t * a.qs + dt * 16 + i]), S[dt][i], qr);
                }
        qr = dl_sum_rows(qr);
        if (h == 0) ((T *)a.o)[t * a.os + vh * a.v_dim + col] = (T)(qr * a.scale);
    }
}

constexpr int DN_NT = 256;
// What the two wavefronts of a pair hand each other in LDS, for a chunk of even and of odd number each: the
// state's parts and the corrections with a word (to the outputs'), the values (to the state's).
template <int KS>
struct DlHand {
    bf16x8d parts[KS][3][64];
    floatx4 u[2][64], v[2][64];
    uint32_t bad, pad[3];  // (of even numbers:) not all corrections were finite
};
template <int KS>
constexpr uint32_t dl_scan_lds() { return 2 * 2 * sizeof(DlHand<KS>); }

__device__ __forceinline__ void dl_meet() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Two wavefronts a SIMD where the registers of one fit in half of them (192 bf16 dimensions, which nearly do: 352 us for 440
// with 8 sequences of 2048 tokens, 16 heads; 160 dimensions, which do: 489 for 376 at 32 heads if they had all).
template <class T, int KS>
constexpr bool dl_two() { return KS * dl_parts<T>() <= 6 && KS < 6; }

// A workgroup takes 32 columns of a value head's state through its sequence's chunks, two wavefronts 16 of
// them.  The first carries the state from chunk to chunk; the second makes the outputs from the
// state's parts and the corrections that the first leaves in LDS, and brings it the values.  They meet once a
// chunk, when its corrections are there.
//
// Bound by the first wavefront's chain, chunk after chunk: 8192 tokens of 48 heads of 128 x 128, bf16, 366 us; without
// any loads 280, 1.1 us a chunk of 68 matrix and some 250 vector instructions in order.  Tried and not faster: the operands brought to LDS once
// for both halves (434 us, with Q S in the first wavefront then), what a part leaves of a value always by the
// matrix cores (363).  fp32, three parts of K, Q and K^T for one: 116 matrix instructions a chunk in that chain and three times
// the operands, 758 us; f16 597.
template <class T, int KS>
__global__ __launch_bounds__(DN_NT, (dl_two<T, KS>() ? 2 : 1)) void delta_scan_kernel(const ScanArgs p) {
    constexpr int NP = dl_parts<T>();
    const DeltaArgs &a = p.a;
    extern __shared__ __align__(16) uint8_t dn_mem[];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 15, h = lane >> 4;
    const uint32_t tiles = a.v_dim / 16, pairs = (tiles + 1) / 2, group = a.v_heads / a.k_heads;
    // a key head's workgroups on one XCD, whose L2 then holds its K and Q (XCDs take workgroups in turn)
    uint32_t id = blockIdx.x;
    const uint32_t each = group * pairs, sets = a.s.count * a.k_heads;
    if (sets % 8 == 0) id = (id / 8 / each * 8 + id % 8) * each + id / 8 % each;
    const uint32_t tile = id % pairs * 2 + (wave >> 1), vh = id / pairs % a.v_heads, seq = id / pairs / a.v_heads, kh = vh / group;
    const uint2 r = kv_rows(a.s.start, seq, a.s.n);
    const uint32_t own = (r.y - r.x + DC - 1) / DC, c_own = dl_before(a.s, seq);
    const uint32_t cb = max(c_own, p.c0), ce = min(c_own + own, p.c1);
    const bool begins = !own || c_own >= p.c0, ends = !own || c_own + own <= p.c1;
    if (own ? cb >= ce : p.c0 != 0) return;
    const uint32_t n = own ? ce - cb : 0;
    if (tile >= tiles) {  // (an odd number of column tiles)
        for (uint32_t c = 0; n && c < n + 2; c++) dl_meet();
        return;
    }
    const uint32_t col = tile * 16 + m, row0 = r.x + (cb - c_own) * DC;  // (row0 is not used without chunks)
    DlHand<KS> *hand = (DlHand<KS> *)dn_mem + (wave >> 1) * 2;
    const uint8_t *k_work = p.k_work + ((uint64_t)kh * p.at_once + (cb - p.c0)) * p.kq;
    const uint8_t *v_work = p.v_work + ((uint64_t)vh * p.at_once + (cb - p.c0)) * DV_BYTES;
    auto kq_of = [&](uint32_t c) { return (const bf16x8d *)(k_work + (uint64_t)c * p.kq) + lane; };
    auto vb_of = [&](uint32_t c) { return v_work + (uint64_t)c * DV_BYTES; };
    // Loads of the next chunk stand where this one's are used up and stay there: they take their place, and waits
    // are for the oldest only.
    auto fix = [] { __builtin_amdgcn_sched_barrier(0); };
    auto wait = [] {
        __builtin_amdgcn_s_waitcnt(0x0F70);  // (all loads from memory)
        __builtin_amdgcn_sched_barrier(0);
    };
    const DlMinus minus(m, h);
    const int64_t slot = a.s.state(seq);
    if ((wave & 1) == 0) {
        floatx4 S[2 * KS];
        const uint64_t each_state = (uint64_t)a.v_heads * a.k_dim * a.v_dim, at = ((uint64_t)vh * a.k_dim + 4 * h) * a.v_dim + col;
        const float *from = !begins ? p.carry_in : a.si && slot >= 0 ? a.si + slot * each_state : nullptr;
        auto load_state = [&] {
#pragma unroll
            for (int dt = 0; dt < 2 * KS; dt++)
#pragma unroll
                for (int i = 0; i < 4; i++) S[dt][i] = from && dt * 16 < (int)a.k_dim ? from[at + (uint64_t)(dt * 16 + i) * a.v_dim] : 0.0f;
        };
        load_state();
        // Operands of wide fp32 keys do not fit in registers beside each other: there K^T is loaded while T R is made and K when
        // K^T is used up (2048 tokens, 16 heads of 256 x 256: 465 us for 750; 192 dimensions, which fit, 259 for 253).
        constexpr bool LATE = KS * NP > 18;
        bf16x8d ka[2][KS][NP], tp[2][3], kt[2 * KS][NP];
        floatx4 eg[2], el[2], v[2], ks0[2];
        float e_last;
        auto load_k = [&](uint32_t c) {
            const bf16x8d *kq = kq_of(c);
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int mt = 0; mt < 2; mt++)
#pragma unroll
                    for (int i = 0; i < NP; i++) ka[mt][ks][i] = kq[((i * 2 + mt) * KS + ks) * 64];
            fix();
        };
        auto load_eg = [&](uint32_t c) {
            const floatx4 *e = (const floatx4 *)(vb_of(c) + 12 * 1024) + h;
            eg[0] = e[0], eg[1] = e[4];
            fix();
        };
        auto load_t = [&](uint32_t c) {
            const bf16x8d *to = (const bf16x8d *)vb_of(c) + lane;
#pragma unroll
            for (int i = 0; i < 3; i++)
#pragma unroll
                for (int mt = 0; mt < 2; mt++) tp[mt][i] = to[(i * 2 + mt) * 64];
            const float *e = (const float *)(vb_of(c) + 12 * 1024);
            el[0] = ((const floatx4 *)(e + DC))[h], el[1] = ((const floatx4 *)(e + DC))[4 + h];
            e_last = e[DC - 1];
            fix();
        };
        auto load_kt = [&](uint32_t c) {
            const bf16x8d *kq = kq_of(c) + NP * 4 * KS * 64;
#pragma unroll
            for (int i = NP - 1; i >= 0; i--)
#pragma unroll
                for (int dt = 0; dt < 2 * KS; dt++) kt[dt][i] = kq[(i * 2 * KS + dt) * 64];
            fix();
        };
        auto load_v = [&](uint32_t c) { v[0] = hand[c & 1].v[0][lane], v[1] = hand[c & 1].v[1][lane]; };
        // The state's parts, which go to LDS, and K S of chunk c, 32 rows of the state behind each other in five stages; stage
        // st does what stands there for rows st, st - 1, ... at once.
        bf16x8d sp[KS][3];
        floatx4 x[KS][2];
        auto read_state = [&](uint32_t c) __attribute__((always_inline)) {
            auto &to = hand[c & 1].parts;
            ks0[0] = ks0[1] = floatx4{0, 0, 0, 0};
            dl_each<KS + 4>([&](auto stage) __attribute__((always_inline)) {
                constexpr int st = decltype(stage)::value;
                constexpr bool in0 = st < KS, in1 = st >= 1 && st - 1 < KS, in2 = st >= 2 && st - 2 < KS, in3 = st >= 3 && st - 3 < KS,
                               in4 = st >= 4 && st - 4 < KS;
                constexpr int h0 = in1 ? 2 * dl_with<NP>(0) : 0, h1 = in2 ? 2 * dl_with<NP>(1) : 0, h2 = in4 ? 2 * dl_with<NP>(2) : 0, m1 = in2 ? 2 : 0;
                auto top = [&](int ks, int j) __attribute__((always_inline)) {
                    sp[ks][j] = j ? dl_top(x[ks][0], x[ks][1]) : dl_top(S[2 * ks], S[2 * ks + 1]);
                    to[ks][j][lane] = sp[ks][j];
                };
                auto by_k = [&](int ks, int j, int i) __attribute__((always_inline)) { ks0[i % 2] = dl_mfma(ka[i % 2][ks][i / 2], sp[ks][j], ks0[i % 2]); };
                dl_zip<m1 + h2 + h1 + h0, (in3 ? 1 : 0) + (in1 ? 1 : 0) + (in0 ? 5 : 0)>(
                    [&](int i) __attribute__((always_inline)) {
                        if constexpr (in2)
                            if (i < m1) x[st - 2][i] = dl_mfma(minus.a[i], sp[st - 2][1], x[st - 2][i]);
                        if constexpr (in4)
                            if (i >= m1 && i < m1 + h2) by_k(st - 4, 2, i - m1);
                        if constexpr (in2)
                            if (i >= m1 + h2 && i < m1 + h2 + h1) by_k(st - 2, 1, i - m1 - h2);
                        if constexpr (in1)
                            if (i >= m1 + h2 + h1) by_k(st - 1, 0, i - m1 - h2 - h1);
                    },
                    [&](int i) __attribute__((always_inline)) {
                        if constexpr (in3)
                            if (i-- == 0) top(st - 3, 2);
                        if constexpr (in1)
                            if (i-- == 0) top(st - 1, 1);
                        if constexpr (in0) {
                            if (i == 0) {
                                top(st, 0);
                                x[st][0] = S[2 * st], x[st][1] = S[2 * st + 1];
                            }
                            if (i > 0) dl_rest(x[st][0], x[st][1], sp[st][0], i - 1);
                        }
                    });
            });
        };
        if (n) {
            wait();
            load_k(0), load_eg(0), load_t(0);
            if (!LATE) load_kt(0);
            read_state(0);
            wait();
            if (!LATE) load_k(min(1u, n - 1));
            dl_meet();  // (the first values)
            load_v(0);
        }
        for (uint32_t c = 0; c < n; c++) {
            const uint32_t next = min(c + 1, n - 1);
            DlHand<KS> &to = hand[c & 1];
            floatx4 u[2];
            bf16x8d part[3];
            auto scale = [&](int dt) { S[dt] *= e_last; };
            if (LATE) load_kt(c);
            // R = V - e^G K S and its parts; T R, the state's decay beside it
            constexpr int EARLY = KS;  // (decays until K S is there)
#pragma unroll
            for (int dt = 0; dt < EARLY; dt++) scale(dt);
            fix();
            v[0] -= eg[0] * ks0[0], v[1] -= eg[1] * ks0[1];
            part[0] = dl_top(v[0], v[1]);
            fix();
            load_eg(next);
            u[0] = u[1] = floatx4{0, 0, 0, 0};
            auto rest = [&](int n) {
                return [&, n](int i) {
                    if (i < 4) dl_rest(v[0], v[1], part[n - 1], i);
                    else part[n] = dl_top(v[0], v[1]);
                };
            };
            auto by_t = [&](int j) {
                return [&, j](int i) { u[i % 2] = dl_mfma(tp[i % 2][i / 2], part[j], u[i % 2]); };
            };
            dl_zip<6, 5>(by_t(0), rest(1));
            dl_zip<4, 5>(by_t(1), rest(2));
            dl_zip<2, 2>(by_t(2), [&](int i) { scale(EARLY + i); });
#pragma unroll
            for (int dt = EARLY + 2; dt < 2 * KS; dt++) scale(dt);
            fix();
            // U; K^T (e^(G_last - G) U)
            to.u[0][lane] = u[0], to.u[1][lane] = u[1];
            v[0] = el[0] * u[0], v[1] = el[1] * u[1];
            part[0] = dl_top(v[0], v[1]);
            fix();
            load_t(next);
            auto by_kt = [&](int j) {
                return [&, j](int i) {
                    const int dt = i % (2 * KS);
                    S[dt] = dl_mfma(kt[dt][i / (2 * KS)], part[j], S[dt]);
                };
            };
            dl_zip<2 * KS * dl_with<NP>(0), 5>(by_kt(0), rest(1));
            dl_zip<2 * KS * dl_with<NP>(1), 5>(by_kt(1), rest(2));
            dl_meet();
            load_v(c + 1);
            dl_zip<2 * KS, 0>(by_kt(2), [](int) {});
            if (LATE) load_k(next);
            else load_kt(next);
            read_state(c + 1);
            if (!LATE) load_k(min(c + 2, n - 1));
        }
        if (n) {
            dl_meet();  // (the outputs are written)
            if (hand->bad) {
                load_state();
                dl_tokens<T, KS>(a, kh, vh, col, h, row0, min(r.y - row0, n * DC), S);
            }
        }
        float *to = !ends ? p.carry_out : a.so && slot >= 0 ? a.so + slot * each_state : nullptr;
        if (to) {
#pragma unroll
            for (int dt = 0; dt < 2 * KS; dt++)
                if (dt * 16 < (int)a.k_dim)
#pragma unroll
                    for (int i = 0; i < 4; i++) to[at + (uint64_t)(dt * 16 + i) * a.v_dim] = S[dt][i];
        }
    } else {
        if (!n) return;
        bf16x8d qa[2][KS][NP], pp[2][3];
        floatx4 eg[2];
        T vv[8];
        const T *vp = (const T *)a.v + vh * a.v_dim + col;
        auto load_v = [&](uint32_t c) {
#pragma unroll
            for (uint32_t j = 0; j < 8; j++)
                vv[j] = vp[min((uint64_t)row0 + (uint64_t)c * DC + j / 4 * 16 + 4 * h + j % 4, (uint64_t)r.y - 1) * a.vs];
            fix();
        };
        auto give_v = [&](uint32_t c) {  // (0 behind the sequence's end)
            const uint64_t first = (uint64_t)row0 + (uint64_t)c * DC + 4 * h;
#pragma unroll
            for (uint32_t j = 0; j < 8; j++)
                ((float *)&hand[c & 1].v[j / 4][lane])[j % 4] = first + j / 4 * 16 + j % 4 < r.y ? to_f32(vv[j]) : 0.0f;
        };
        auto load_q = [&](uint32_t c) {
            const bf16x8d *kq = kq_of(c) + NP * 2 * KS * 64;
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int mt = 0; mt < 2; mt++)
#pragma unroll
                    for (int i = 0; i < NP; i++) qa[mt][ks][i] = kq[((i * 2 + mt) * KS + ks) * 64];
            fix();
        };
        auto load_p = [&](uint32_t c) {
            const bf16x8d *to = (const bf16x8d *)vb_of(c) + 6 * 64 + lane;
#pragma unroll
            for (int mt = 0; mt < 2; mt++)
#pragma unroll
                for (int i = 0; i < 3; i++) pp[mt][i] = to[(i * 2 + mt) * 64];
            const floatx4 *e = (const floatx4 *)(vb_of(c) + 12 * 1024) + h;
            eg[0] = e[0], eg[1] = e[4];
            fix();
        };
        load_v(0);
        give_v(0);
        load_v(1);
        give_v(1);
        dl_meet();
        wait();
        load_v(2), load_q(0), load_p(0);
        float bad = 0;
        for (uint32_t c = 0; c < n; c++) {
            dl_meet();
            const uint32_t next = min(c + 1, n - 1), first = row0 + c * DC, left = r.y - first;
            const DlHand<KS> &from = hand[c & 1];
            give_v(c + 2);
            fix();
            load_v(c + 3);
            floatx4 o[2] = {};
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const bf16x8d part[3] = {from.parts[ks][0][lane], from.parts[ks][1][lane], from.parts[ks][2][lane]};
#pragma unroll
                for (int mt = 0; mt < 2; mt++) o[mt] = dl_mma(qa[mt][ks], part, o[mt]);
            }
            fix();
            load_q(next);
            bf16x8d part[3];
            dl_split(from.u[0][lane], from.u[1][lane], part);
#pragma unroll
            for (int j = 0; j < 8; j++) bad = fmaf(2 * from.u[j / 4][lane][j % 4], 0.0f, bad);
#pragma unroll
            for (int mt = 0; mt < 2; mt++) o[mt] = dl_mma(pp[mt], part, o[mt] * eg[mt]);
            fix();
            load_p(next);
            T *to = (T *)a.o + (uint64_t)(first + 4 * h) * a.os + vh * a.v_dim + col;
            if (left >= DC) {
#pragma unroll
                for (uint32_t j = 0; j < 8; j++) to[(j / 4 * 16 + j % 4) * a.os] = (T)(o[j / 4][j % 4] * a.scale);
            } else {
#pragma unroll
                for (uint32_t j = 0; j < 8; j++)
                    if (j / 4 * 16 + 4 * h + j % 4 < left) to[(j / 4 * 16 + j % 4) * a.os] = (T)(o[j / 4][j % 4] * a.scale);
            }
        }
        hand->bad = __ballot(bad != bad) != 0;
        wait();
        dl_meet();
    }
}

}  // namespace okf
