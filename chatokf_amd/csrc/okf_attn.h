// okf_attn.h -- causal attention over packed prompts (okf_attn_prompt) on the
// matrix cores.
//
// One pass over a row's keys with the running maximum and sum of its softmax.  A
// wavefront takes 32 query rows of a head, a workgroup 64 or 128 (launch_prompt_d),
// tile by tile of keys.  Both products are computed transposed (v_mfma_f32_32x32x16):
//   S^T = K Q^T: A = 32 keys x 16 dimensions, B = the queries (in registers
//     throughout); a lane then holds, for query row lane % 32, the keys
//     8 (i / 4) + 4 (lane / 32) + i % 4, so that a row's maximum and sum are the
//     lane's own but for one exchange with lane ^ 32;
//   O^T = V^T P^T: B = the weights as they lie in those registers, two fours of keys
//     a lane and instruction, and A = 32 dimensions x the same keys, which
//     ds_read_b64_tr_b16 takes out of the row-major V tile.
// No weight passes through LDS, and the row's factors are the lane's own.
//
// 16-bit inputs go from memory to LDS without registers (buffer loads with the LDS
// as target), double-buffered; rows are read in an order such that 16-byte chunk c
// of row r stands at c ^ at_fk(r) / at_fv(r), which spreads the reads of both
// products over the banks.  fp32 inputs are split into three bf16 parts on their way
// to LDS (x = x0 + x1 + x2 exactly from 2^-110 up, each part the next eight bits), and so
// are the weights: six of the nine products of parts, the others are below 2^-22 of the
// whole.
//
// Measured (MI355X): f16, 8192 rows x 40 heads of 128 682-705 us, 975-1010 TFLOP/s; a matrix
// product of 8192 in f16 runs at 1119-1157 there, both at the 2.0 GHz or less that the card's
// power leaves.  Without its loads from memory the variant named at the pass took 14 %
// less, without its reads of LDS 11 %: no one of matrix cores (57 % of their time), vector
// units (50 %) and LDS bounds it alone.  8 packed bf16 prompts of up to 1111 x 16 heads 34-36 us; with the
// last sequence's tiles first 47.
//
// Registers: the second, careful pass is part of the kernel and sets what the first one
// runs with.  A lane's (bf16, f16 alike; without that pass): 64 wide 186 to 190 (112 to 118), 128 wide
// 237, and 256 with 3 spilled for 128 rows (156, 167), 256 wide 512 with 36 to 44 spilled (404, 439): one
// wavefront a SIMD there, two elsewhere.  Widths that are not compiled for spill more: 68 for 112 with
// 128 rows, 468 to 677 past 128.  fp32: two wavefronts a SIMD at up to 64 wide with 128 rows or
// eight wavefronts, else one; 200 registers spilled at 256 wide, 1907 at the other widths past 128.
#pragma once
#include <type_traits>

#include "okf_kv_seqs.h"

namespace okf {

struct AttnArgs {
    const void *q, *k, *v;
    void *o;
    uint32_t heads, kv_heads, dim, seqs, nq, nk;
    const int32_t *q_start, *k_start;
    uint64_t qs, ks, vs, os, qh, kh, vh, oh;
    float scale;
    uint32_t window;
    uint32_t tiles;   // bound of the query tiles of all sequences
};

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2v __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4v __attribute__((ext_vector_type(4)));
typedef short shortx4 __attribute__((ext_vector_type(4)));

// A kernel's shape.  DH: the head width, or 0 for one that is known at the launch
// only; DP: the width that its rows have in LDS.  A workgroup has RG x KG wavefronts:
// RG groups of 32 query rows, and KG groups that the keys are dealt to.
template <class T, int DP_, int DH_, int RG_, int KG_>
struct AtShape {
    using E = T;
    static constexpr int DP = DP_, DH = DH_, RG = RG_, KG = KG_, BM = 32 * RG, NT = 64 * RG * KG;
    static constexpr int NP = 1, NB = 2;  // parts of a value; buffers
    static constexpr int BN = DP * KG <= 128 || (DP == 256 && KG == 1) ? 64 : 32;  // keys of a wavefront's tile
    static constexpr int WAVES = DP <= 128 || NT > 256 ? 2 : 1;  // a SIMD
};
template <int DP_, int DH_, int RG_, int KG_>
struct AtShape<float, DP_, DH_, RG_, KG_> {
    using E = __bf16;
    static constexpr int DP = DP_, DH = DH_, RG = RG_, KG = KG_, BM = 32 * RG, NT = 64 * RG * KG;
    static constexpr int NP = 3, NB = 1, BN = 32, WAVES = NT > 256 ? 2 : 1;
};
// bytes of LDS: the tiles, or the key groups' results
template <class S>
constexpr uint32_t at_lds() {
    constexpr uint32_t tiles = S::NB * 2 * S::NP * S::KG * S::BN * S::DP * 2;
    constexpr uint32_t join = (S::KG - 1) * S::RG * 64 * (16 * (((S::DH ? S::DH : S::DP) + 31) / 32) + 2) * 4;
    return tiles > join ? tiles : join;
}
template <class S>
constexpr bool at_fits() { return at_lds<S>() <= 160 * 1024; }

template <class E>
__device__ __forceinline__ floatx16 at_mfma(u32x4v a, u32x4v b, floatx16 c) {
    if constexpr (sizeof(E) == 2 && __is_same(E, _Float16))
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// two fp32 values as two 16-bit ones, to nearest even
template <class E>
__device__ __forceinline__ uint32_t at_pack(float a, float b) {
    const floatx2 x = {a, b};
    if constexpr (__is_same(E, _Float16)) return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, half2v));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2));
}

// fp32 pair -> the bf16 pairs of its three parts.  An infinity is its first part,
// the others 0.
__device__ __forceinline__ void at_split(float a, float b, uint32_t &p0, uint32_t &p1, uint32_t &p2) {
    const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
    p0 = __builtin_amdgcn_perm(ub, ua, 0x07060302u);
    float ra = a - __uint_as_float(ua & 0xFFFF0000u), rb = b - __uint_as_float(ub & 0xFFFF0000u);
    if ((ua & 0x7F800000u) == 0x7F800000u) ra = 0;
    if ((ub & 0x7F800000u) == 0x7F800000u) rb = 0;
    const uint32_t va = __float_as_uint(ra), vb = __float_as_uint(rb);
    p1 = __builtin_amdgcn_perm(vb, va, 0x07060302u);
    ra -= __uint_as_float(va & 0xFFFF0000u);
    rb -= __uint_as_float(vb & 0xFFFF0000u);
    p2 = __builtin_amdgcn_perm(__float_as_uint(rb), __float_as_uint(ra), 0x07060302u);
}

// the low half of x
template <class E>
__device__ __forceinline__ float at_half(uint32_t x) {
    if constexpr (__is_same(E, _Float16)) return (float)__builtin_bit_cast(_Float16, (uint16_t)x);
    else return __uint_as_float(x << 16);
}

// the larger of x here and in lane ^ 32
__device__ __forceinline__ float at_max32(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Where a row's 16-byte chunks stand (see above): K's 16 rows of a quarter
// wavefront read the same chunk, V's four rows four chunks each.
template <int CPR>
__device__ __forceinline__ uint32_t at_fk(uint32_t r) { return CPR == 8 ? (r & 7) ^ (r >> 3 & 1) : r & 15; }
template <int CPR>
__device__ __forceinline__ uint32_t at_fv(uint32_t r) { return (r & 1) * (CPR == 8 ? 2 : 10) ^ (r & 2) * 2; }

// The idx-th tile of up to 64 sequences, those of the most keys first: level L holds the
// tiles whose rows end about L tiles behind their sequence's first key.  More sequences:
// the last first.
template <int BM>
__device__ __forceinline__ SeqItem at_tile(const AttnArgs &a, uint32_t idx) {
    auto tiles = [&](uint32_t s) {
        const uint2 r = kv_rows(a.q_start, s, a.nq);
        return (r.y - r.x + BM - 1) / BM;
    };
    if (a.seqs == 1) {
        const uint32_t n = tiles(0);
        return {idx < n ? 0u : 1u, n - 1 - idx};
    }
    if (a.seqs > 64) return kv_find(a.tiles - 1 - idx, a.seqs, tiles);
    const uint32_t lane = threadIdx.x & 63;
    uint32_t n = 0, before = 0;
    if (lane < a.seqs) {
        n = tiles(lane);
        const uint2 rq = kv_rows(a.q_start, lane, a.nq), rk = kv_rows(a.k_start, lane, a.nk);
        before = rk.y - rk.x > rq.y - rq.x ? (rk.y - rk.x - (rq.y - rq.x)) / BM : 0;
    }
    auto count = [&](uint32_t level) {  // tiles of this level and above
        uint32_t v = level < before + n ? min(before + n - level, n) : 0;
        return (uint32_t)__builtin_amdgcn_readlane(lanes_sum(v), 63);
    };
    uint32_t lo = 0, hi = lanes_max(before + n);  // count(lo) > idx >= count(hi)
    if (count(0) <= idx) return {a.seqs, 0};
    uint32_t above = 0;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2, c = count(mid);
        if (c > idx) lo = mid;
        else hi = mid, above = c;
    }
    const bool here = lo >= before && lo < before + n;
    const uint64_t who = __ballot(here);
    const bool mine = here && __popcll(who & ((1ull << lane) - 1)) == idx - above;
    const int l = __ffsll((unsigned long long)__ballot(mine)) - 1;
    return {(uint32_t)l, lo - (uint32_t)__builtin_amdgcn_readlane(before, l)};
}

template <class T, class S>
__global__ __launch_bounds__(S::NT, S::WAVES) void attn_prompt_kernel(AttnArgs a) {
    using E = typename S::E;
    constexpr int DP = S::DP, DH = S::DH, KG = S::KG, RG = S::RG, NP = S::NP, BN = S::BN, BM = S::BM;
    constexpr int KS = (DH ? DH : DP) / 16, DT = ((DH ? DH : DP) + 31) / 32, TT = BN / 32, CPR = DP / 8;
    constexpr uint32_t ROW = DP * 2, PB = KG * BN * ROW;  // bytes of a row and of a part's tiles in LDS
    constexpr int STEP = KG * BN;
    extern __shared__ __align__(16) uint8_t at_mem[];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), D = DH ? DH : a.dim;
    const uint32_t rg = wave % RG, kg = wave / RG, h = lane >> 5;
    // A kv head's workgroups on as few XCDs (workgroups a multiple of 8 apart) as there are for
    // it, tiles in order: kv heads that divide 8 have 8 / kv_heads XCDs each; else heads that 8
    // divides lie side by side on one.
    uint32_t head = blockIdx.x % a.heads, rank = blockIdx.x / a.heads;
    if (8 % a.kv_heads == 0) {
        const uint32_t x = blockIdx.x % 8, group = a.heads / a.kv_heads;
        const uint32_t at = blockIdx.x / 8 * (8 / a.kv_heads) + x / a.kv_heads;
        head = x % a.kv_heads * group + at % group;
        rank = at / group;
    } else if (a.heads % 8 == 0) {
        head = head % 8 * (a.heads / 8) + head / 8;
    }
    const SeqItem it = at_tile<BM>(a, rank);
    if (it.seq >= a.seqs) return;
    const uint2 rq = kv_rows(a.q_start, it.seq, a.nq), rk = kv_rows(a.k_start, it.seq, a.nk);
    // (a window of all keys is none; a smaller one taken from a position, which is below zero where
    // there are more queries than keys, is above -nq and so within 32 bits)
    const int nq = rq.y - rq.x, nk = rk.y - rk.x, i0 = it.at * BM, w = a.window && a.window < (uint32_t)nk ? (int)a.window : 0;
    const int kh = head / (a.heads / a.kv_heads);
    // positions: of the workgroup's first and last row, the wavefront's, the lane's
    const int p_first = nk - nq + i0, p_last = nk - nq + min(i0 + BM, nq) - 1;
    const int w_first = p_first + 32 * (int)rg, w_last = min(w_first + 31, p_last);
    const int row = i0 + 32 * (int)rg + (int)(lane & 31), pos = nk - nq + row;
    const int j_end = p_last + 1, j_begin = w ? max(p_first - w + 1, 0) / BN * BN : 0;

    const T *kp = (const T *)a.k + rk.x * a.ks + (uint64_t)kh * a.kh, *vp = (const T *)a.v + rk.x * a.vs + (uint64_t)kh * a.vh;
    // queries: parts of dimensions 16 k + 8 h .. + 7 of the lane's row.  The scale's sign goes to them.
    float c = a.scale * 1.4426950408889634f;
    const uint32_t flip = c < 0 ? 0x80008000u : 0;
    // (a factor of 0 would make NaN of a masked -inf; the smallest number there is takes any two
    // scores less than 2^-19 apart)
    c = c == 0 ? 0x1p-149f : fabsf(c);
    u32x4v q[NP][KS];
    const T *qrow = (const T *)a.q + (uint64_t)(rq.x + min(row, nq - 1)) * a.qs + (uint64_t)head * a.qh;
#pragma unroll
    for (int k = 0; k < KS; k++) {
        if (!DH && 16 * k >= (int)D) break;
        const T *qp = qrow + 16 * k + 8 * h;
        if constexpr (NP == 1) {
            q[0][k] = *(const u32x4v *)qp ^ flip;
        } else {
            const floatx4 x = *(const floatx4 *)qp, y = *(const floatx4 *)(qp + 4);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                uint32_t s0, s1, s2;
                at_split(i < 2 ? x[2 * i] : y[2 * i - 4], i < 2 ? x[2 * i + 1] : y[2 * i - 3], s0, s1, s2);
                q[0][k][i] = s0 ^ flip, q[1][k][i] = s1 ^ flip, q[2][k][i] = s2 ^ flip;
            }
        }
    }

    // staging
    constexpr uint32_t RPP = 1024 / ROW;               // rows of a 1 KB piece: one instruction of a wavefront
    constexpr int WAVES = RG * KG, PIECES = (int)(PB / 1024 / WAVES);  // a wavefront's, K and V each
    constexpr int XV = STEP * DP / 4 / S::NT;          // fp32: 16-byte loads a thread, K and V each
    uint32_t koff[2], voff;
    floatx4 xk[NP == 3 ? XV : 1], xv[NP == 3 ? XV : 1];
    if constexpr (NP == 1) {
        const uint32_t r = wave * RPP + lane / CPR, cc = lane % CPR;
#pragma unroll
        for (int p = 0; p < 2; p++)
            koff[p] = r * (uint32_t)(a.ks * 2) + min(cc ^ at_fk<CPR>(r + p * WAVES * RPP), D / 8 - 1) * 16;
        voff = r * (uint32_t)(a.vs * 2) + min(cc ^ at_fv<CPR>(r), D / 8 - 1) * 16;
    }
    // LDS: K in NB buffers, then V.  16-bit: memory to LDS; fp32: memory to registers, `put` to LDS.
    auto issue = [&](int j, int buf, bool isv) __attribute__((always_inline)) {
        const T *from = isv ? vp : kp;
        const uint64_t st = isv ? a.vs : a.ks;
        if constexpr (NP == 1) {
            // rows past the sequence's end lie past the buffer's (whole offsets in the lanes: the
            // range check may leave the scalar one out)
            const uint32_t rows = (uint32_t)min(nk - j, STEP);
            auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)(from + (uint64_t)j * st), 0,
                                                          (rows - 1) * (uint32_t)(st * 2) + D * 2, 0x00027000);
            using lds_t = __attribute__((address_space(3))) void;
            uint8_t *to = at_mem + ((isv ? 2 : 0) + buf) * PB + wave * 1024;
#pragma unroll
            for (int p = 0; p < PIECES; p++)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_t *)(to + p * WAVES * 1024), 16,
                                                         (isv ? voff : koff[p & 1]) + p * WAVES * RPP * (uint32_t)(st * 2), 0, 0, 0);
        } else {
#pragma unroll
            for (int i = 0; i < XV; i++) {
                const uint32_t e = threadIdx.x + i * S::NT, r = e / (DP / 4), d = min(e % (DP / 4) * 4, D - 4);
                const uint64_t rr = (uint32_t)min(j + (int)r, nk - 1);
                (isv ? xv : xk)[i] = *(const floatx4 *)(from + rr * st + d);
            }
        }
    };
    auto put = [&](bool isv) __attribute__((always_inline)) {
        if constexpr (NP == 3) {
#pragma unroll
            for (int i = 0; i < XV; i++) {
                const uint32_t e = threadIdx.x + i * S::NT, r = e / (DP / 4), c4 = e % (DP / 4);
                uint8_t *to = at_mem + (isv ? NP * PB : 0) + r * ROW +
                              ((c4 / 2) ^ (isv ? at_fv<CPR>(r) : at_fk<CPR>(r))) * 16 + c4 % 2 * 8;
                const floatx4 x = (isv ? xv : xk)[i];
                u32x2v s[3];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    uint32_t s0, s1, s2;
                    at_split(x[2 * u], x[2 * u + 1], s0, s1, s2);
                    s[0][u] = s0, s[1][u] = s1, s[2][u] = s2;
                }
#pragma unroll
                for (int p = 0; p < 3; p++) *(u32x2v *)(to + p * PB) = s[p];
            }
        }
    };
    // (buffers by constants, so that they are part of the loads' immediate offsets)
    auto kbuf = [&](auto n) __attribute__((always_inline)) -> const uint8_t * { return at_mem + (NP == 1 ? (n & 1) * PB : 0); };
    auto vbuf = [&](auto n) __attribute__((always_inline)) -> const uint8_t * { return at_mem + NP * PB + (NP == 1 ? PB + (n & 1) * PB : 0); };
    constexpr std::integral_constant<int, 0> B0{};
    constexpr std::integral_constant<int, 1> B1{};

    floatx16 o[DT];
    // the running maximum; the scores that move it; what their exponents lose (f16: weights of up to
    // 2^8 2^7, so that those 2^-30 of the largest are still normal or nearly so); the weights' sum
    constexpr float UP = __is_same(E, _Float16) ? 7.0f : 0.0f;
    float m, limit, mc, l;
    // this lane's part of the LDS addresses: K row lane % 32, V row and chunk of the transposed read
    const uint32_t kl = kg * BN * ROW + (lane & 31) * ROW, kx = h ^ at_fk<CPR>(lane & 31);
    const uint32_t vr = 4 * h + (lane & 15) / 4, vl = (kg * BN + vr) * ROW + (lane & 1) * 8, vx = ((lane >> 4 & 1) * 2 + (lane & 3) / 2);
    const uint32_t vf = at_fv<CPR>(vr);
    auto read_v = [&](const uint8_t *v, int kk, int dt) __attribute__((always_inline)) {
        const uint8_t *p = v + vl + kk * 16 * ROW + ((4 * dt + vx) ^ vf) * 16;
        using lds4 = __attribute__((address_space(3))) shortx4;
        const u32x2v x = __builtin_bit_cast(u32x2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)p));
        const u32x2v y = __builtin_bit_cast(u32x2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)(p + 8 * ROW)));
        return u32x4v{x[0], x[1], y[0], y[1]};
    };

    auto product = [&](const u32x4v (&x)[NP], const u32x4v &y0, const u32x4v &y1, const u32x4v &y2, floatx16 &s) __attribute__((always_inline)) {
        if constexpr (NP == 3) {
            s = at_mfma<E>(x[2], y0, s);
            s = at_mfma<E>(x[0], y2, s);
            s = at_mfma<E>(x[1], y1, s);
            s = at_mfma<E>(x[1], y0, s);
            s = at_mfma<E>(x[0], y1, s);
        }
        s = at_mfma<E>(x[0], y0, s);
    };
    // scores of the wavefront's tile; the weighted sum of its values
    auto qk = [&](const uint8_t *K, floatx16 (&s)[TT]) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < TT; t++) s[t] = floatx16{};
#pragma unroll
        for (int k = 0; k < KS; k++) {
            if (!DH && 16 * k >= (int)D) break;
#pragma unroll
            for (int t = 0; t < TT; t++) {
                u32x4v x[NP];
#pragma unroll
                for (int i = 0; i < NP; i++) x[i] = *(const u32x4v *)(K + i * PB + t * 32 * ROW + kl + ((2 * k) ^ kx) * 16);
                product(x, q[0][k], q[NP / 2][k], q[NP - 1][k], s[t]);
            }
        }
    };
    struct Weights {
        u32x4v x[NP][2 * TT];
    };
    auto pv = [&](const Weights &p, const uint8_t *V) __attribute__((always_inline)) {
#pragma unroll
        for (int kk = 0; kk < 2 * TT; kk++)
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
                if (!DH && 32 * dt >= (int)D) break;
                u32x4v x[NP];
#pragma unroll
                for (int i = 0; i < NP; i++) x[i] = read_v(V + i * PB, kk, dt);
                product(x, p.x[0][kk], p.x[NP / 2][kk], p.x[NP - 1][kk], o[dt]);
            }
    };
    auto sees = [&](int jj) __attribute__((always_inline)) { return jj <= pos && (!w || jj > pos - w); };
    auto is_whole = [&](int j) __attribute__((always_inline)) { return j + BN - 1 <= w_first && (!w || j >= w_last - w + 1); };
    auto mask = [&](floatx16 (&s)[TT], int j) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < TT; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) s[t][i] = sees(j + 32 * t + 8 * (i / 4) + 4 * (int)h + i % 4) ? s[t][i] : -__builtin_inff();
    };
    // A tile's weights from its scores.  The running maximum moves only when it is passed by a
    // factor of 2^8 (limit): weights of up to 256 lose nothing, and most tiles need no new factors.
    const float slack = 8.0f / c;
    // (careful: see below)
    auto weights = [&](const floatx16 (&s)[TT], Weights &p, auto careful) __attribute__((always_inline)) {
        float x = s[0][0];
#pragma unroll
        for (int t = 0; t < TT; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) x = fmaxf(x, s[t][i]);
        x = at_max32(x);
        if (__ballot(x > limit)) {
            const float nm = fmaxf(m, x);
            const float f = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((m - nm) * c);
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; d++) o[d] *= f;
            m = nm;
            limit = nm + slack;
            mc = (nm == -__builtin_inff() ? 0.0f : nm * c) - UP;
        }
        float l1 = 0;
        [[maybe_unused]] const float ref = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
        for (int t = 0; t < TT; t++)
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const float e0 = __builtin_amdgcn_exp2f(careful ? fmaf(s[t][i] - ref, c, UP) : fmaf(s[t][i], c, -mc));
                const float e1 = __builtin_amdgcn_exp2f(careful ? fmaf(s[t][i + 1] - ref, c, UP) : fmaf(s[t][i + 1], c, -mc));
                l += e0, l1 += e1;
                const int kk = 2 * t + i / 8, at = i % 8 / 2;
                if constexpr (NP == 1) {
                    // (rounded to the inputs' type, half a step each: the second product at the first
                    // one's rate.  Their sum is kept of the unrounded ones.  bf16 2.0e-3 from 64 bits, with
                    // fp32 weights 1.6e-3, the output's own rounding; f16 2.8e-4 and 2.1e-4.  In two
                    // parts the product would take twice as long.)
                    p.x[0][kk][at] = at_pack<E>(e0, e1);
                } else {
                    uint32_t s0, s1, s2;
                    at_split(e0, e1, s0, s1, s2);
                    p.x[0][kk][at] = s0;
                    p.x[NP / 2][kk][at] = s1;
                    p.x[NP - 1][kk][at] = s2;
                }
            }
        l += l1;
    };
    auto start = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int d = 0; d < DT; d++) o[d] = floatx16{};
        m = limit = -__builtin_inff(), l = 0, mc = -UP;
    };
    const int steps = j_end > j_begin ? (j_end - j_begin + STEP - 1) / STEP : 0;
    auto at_key = [&](int n) __attribute__((always_inline)) { return j_begin + n * STEP + (int)kg * BN; };

    // The pass over the keys.  The wavefronts of a SIMD overlap one's products with another's
    // weights.  (Three blocks of 32 keys under way in each wavefront, its products in between
    // its weights' instructions, measured no better: 8192 x 40 heads of 128 731 us against 713,
    // 300 x 32 heads behind 3000 81 against 67; 64 rows a wavefront, which halves the reads of
    // LDS, 1725: their registers leave one wavefront a SIMD and spill.)
    start();
    if (steps) {
        issue(j_begin, 0, false);
        issue(j_begin, 0, true);
        auto turn = [&](int n, auto here, auto there) __attribute__((always_inline)) {
            if constexpr (NP == 1) {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();  // (this tile is whole, the other buffer's readers are done)
            } else {
                __syncthreads();
                put(false);
                put(true);
                __syncthreads();
            }
            if (n + 1 < steps) {
                issue(j_begin + (n + 1) * STEP, there, false);
                issue(j_begin + (n + 1) * STEP, there, true);
            }
            const int j = at_key(n);
            if (j > w_last || (w && j + BN <= w_first - w + 1)) return;  // nothing for this wavefront
            floatx16 s[TT];
            Weights p;
            qk(kbuf(here), s);
            if (!is_whole(j)) mask(s, j);
            weights(s, p, std::false_type{});
            pv(p, vbuf(here));
        };
        for (int n = 0; n < steps; n += 2) {
            turn(n, B0, B1);
            if (n + 1 < steps) turn(n + 1, B1, B0);
        }
    }

    // A value that is not finite makes NaN of rows that do not see it (0 * NaN), and an
    // infinity's parts of a score; both show in the results.  Where the maximum is large, its
    // product's rounding (half of 2^-23 of it) is a factor of its own on all of a row's weights, up
    // to one that no 16-bit, then no fp32 number holds.  Then the workgroup makes the pass again,
    // carefully: such values key by key, such scores in fp32, weights from the scores' differences.
    float nan = l * 0.0f;
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) nan = fmaf(o[d][i], 0.0f, nan);
    const bool large = m > -__builtin_inff() && fabsf(m) * c >= 0x1p20f;
    if (__syncthreads_or(nan != 0 || large)) {
        start();
#pragma unroll 1
        for (int n = 0; n < steps; n++) {
            __syncthreads();
            issue(j_begin + n * STEP, 0, false);
            issue(j_begin + n * STEP, 0, true);
            put(false);
            put(true);
            if constexpr (NP == 1) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            const uint8_t *V = vbuf(B0);
            const int j = at_key(n);
            floatx16 s[TT];
            qk(kbuf(B0), s);
            if constexpr (NP == 3) {
#pragma unroll 1
                for (int i = 0; i < 16; i++) {
                    const int jj = j + 8 * (i / 4) + 4 * (int)h + i % 4;
                    float old = 0;
#pragma unroll
                    for (int u = 0; u < 16; u++) old = u == i ? s[0][u] : old;
                    if (old != old && sees(jj)) {
                        float x = 0;
                        for (uint32_t d = 0; d < D; d++) x = fmaf((float)qrow[d], (float)kp[(uint64_t)jj * a.ks + d], x);
#pragma unroll
                        for (int u = 0; u < 16; u++) s[0][u] = u == i ? (flip ? -x : x) : s[0][u];
                    }
                }
            }
            const bool whole = is_whole(j);
            if (!whole) mask(s, j);
            Weights p;
            weights(s, p, std::true_type{});
            bool bad = false;
            if (!whole) {
                constexpr uint32_t EXP = __is_same(E, _Float16) ? 0x7C007C00u : 0x7F807F80u, ONE = __is_same(E, _Float16) ? 0x04000400u : 0x00800080u;
                uint32_t any = 0;
#pragma unroll 1
                for (uint32_t e = lane; e < BN * ROW / 16; e += 64) {
                    const u32x4v x = *(const u32x4v *)(V + kg * BN * ROW + e * 16);
#pragma unroll
                    for (int i = 0; i < 4; i++) any |= (x[i] & EXP) + ONE;
                }
                bad = __ballot((any & 0x80008000u) != 0) != 0;
            }
            if (!bad) {
                pv(p, V);
                continue;
            }
#pragma unroll 1
            for (int key = 0; key < BN; key++) {
                const int el = (key & 3) + (key & 8 ? 4 : 0), at = key / 16 * 4 + el / 2;  // (key & 4: the lane's half)
                float wt = 0;
#pragma unroll
                for (int pp = 0; pp < NP; pp++) {
                    uint32_t y = 0;
#pragma unroll
                    for (int u = 0; u < 8 * TT; u++) y = u == at ? p.x[pp][u / 4][u % 4] : y;
                    wt += at_half<E>(el & 1 ? y >> 16 : y);
                }
                wt = __shfl(wt, (int)(lane & 31) + 8 * (key & 4));
                const bool seen = sees(j + key);
                const uint8_t *vrow = V + (kg * BN + key) * ROW + h * 8;
#pragma unroll
                for (int u = 0; u < 4 * DT; u++) {
                    float v[4] = {};
#pragma unroll
                    for (int pp = 0; pp < NP; pp++) {
                        const u32x2v y = *(const u32x2v *)(vrow + pp * PB + (u ^ at_fv<CPR>(key)) * 16);
#pragma unroll
                        for (int i = 0; i < 4; i++) v[i] += at_half<E>(i & 1 ? y[i / 2] >> 16 : y[i / 2]);
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (seen) o[u / 4][4 * (u % 4) + i] = fmaf(wt, v[i], o[u / 4][4 * (u % 4) + i]);
                }
            }
        }
    }

    if constexpr (KG > 1) {
        // the key groups' results joined by the first
        constexpr uint32_t EACH = 64 * (16 * DT + 2);
        __syncthreads();
        if (kg) {
            float *to = (float *)at_mem + ((kg - 1) * RG + rg) * EACH + lane;
            to[0] = m, to[64] = l;
#pragma unroll
            for (int e = 0; e < 16 * DT; e++) to[64 * (2 + e)] = o[e / 16][e % 16];
        }
        __syncthreads();
        if (kg) return;
#pragma unroll 1
        for (int g = 1; g < KG; g++) {
            const float *from = (const float *)at_mem + ((g - 1) * RG + rg) * EACH + lane;
            const float m1 = from[0], nm = fmaxf(m, m1);
            const float f = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((m - nm) * c);
            const float f1 = m1 == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((m1 - nm) * c);
            l = l * f + from[64] * f1;
            m = nm;
#pragma unroll
            for (int e = 0; e < 16 * DT; e++) o[e / 16][e % 16] = o[e / 16][e % 16] * f + from[64 * (2 + e)] * f1;
        }
    }
    l += __shfl_xor(l, 32);
    if (row >= nq) return;
    const float inv = l != 0 ? 1.0f / l : 0.0f;
    T *out = (T *)a.o + (uint64_t)(rq.x + row) * a.os + (uint64_t)head * a.oh + 4 * h;
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const uint32_t d = 32 * dt + 2 * i;
            if (d >= D) break;
            const floatx16 &x = o[dt];
            if constexpr (NP == 1) {
                u32x2v y = {at_pack<E>(x[i] * inv, x[i + 1] * inv), at_pack<E>(x[i + 2] * inv, x[i + 3] * inv)};
                if (l == 0) y = {0, 0};
                *(u32x2v *)(out + d) = y;
            } else {
                *(floatx4 *)(out + d) = l != 0 ? floatx4{x[i] * inv, x[i + 1] * inv, x[i + 2] * inv, x[i + 3] * inv}
                                               : floatx4{0, 0, 0, 0};
            }
        }
}

}  // namespace okf
