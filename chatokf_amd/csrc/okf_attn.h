// okf_attn.h -- causal attention over packed prompts (okf_attn_prompt) on the
// matrix cores.
//
// One pass over a row's keys with the running maximum and sum of its softmax.  A
// workgroup takes 128 query rows of a head, a wavefront 32 of them, tile by tile of
// keys.  Both products are computed transposed (v_mfma_f32_32x32x16):
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
// to LDS (x = x0 + x1 + x2 exactly, each part the next eight bits), and so are the
// weights: six of the nine products of parts, the others are below 2^-22 of the
// whole.
#pragma once
#include "okf_kv.h"

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

constexpr int AT_NT = 256;
constexpr uint32_t AT_BM = 128;  // query rows a workgroup

template <class T>
struct AtType {
    using E = T;
    static constexpr int NP = 1, BN = 64;  // parts of a value; keys a tile
};
template <>
struct AtType<float> {
    using E = __bf16;
    static constexpr int NP = 3, BN = 32;
};

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

// Where a row's 16-byte chunks stand (see above): K's 16 rows of a quarter
// wavefront read the same chunk, V's four rows four chunks each.
template <int CPR>
__device__ __forceinline__ uint32_t at_fk(uint32_t r) { return CPR == 8 ? (r & 7) ^ (r >> 3 & 1) : r & 15; }
template <int CPR>
__device__ __forceinline__ uint32_t at_fv(uint32_t r) { return (r & 1) * (CPR == 8 ? 2 : 10) ^ (r & 2) * 2; }

template <class T, int DP>
constexpr uint32_t at_lds() { return (AtType<T>::NP == 1 ? 2 : 1) * 2 * AtType<T>::NP * AtType<T>::BN * DP * 2; }

// DP: the head width rounded up to 64, 128 or 256; FULL: it is that.  Dimensions
// past it are not multiplied; their V rows make output rows that are not stored.
template <class T, int DP, bool FULL>
__global__ __launch_bounds__(AT_NT, AtType<T>::NP == 1 && DP <= 128 ? 2 : 1) void attn_prompt_kernel(AttnArgs a) {
    using E = typename AtType<T>::E;
    constexpr int NP = AtType<T>::NP, BN = AtType<T>::BN, KS = DP / 16, DT = DP / 32, TT = BN / 32, CPR = DP / 8;
    constexpr uint32_t ROW = DP * 2, PB = BN * ROW;  // bytes of a row and of a part's tile in LDS
    extern __shared__ __align__(16) uint8_t at_mem[];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, D = FULL ? DP : a.dim;
    // heads of one kv head on one XCD where they divide over the eight
    uint32_t head = blockIdx.x % a.heads;
    const uint32_t tile = a.tiles - 1 - blockIdx.x / a.heads;  // (a sequence's last tiles take longest: first)
    if (a.heads % 8 == 0) head = head % 8 * (a.heads / 8) + head / 8;
    const SeqItem it = kv_find(tile, a.seqs, [&](uint32_t s) {
        const uint2 r = kv_rows(a.q_start, s, a.nq);
        return (r.y - r.x + AT_BM - 1) / AT_BM;
    });
    if (it.seq >= a.seqs) return;
    const uint2 rq = kv_rows(a.q_start, it.seq, a.nq), rk = kv_rows(a.k_start, it.seq, a.nk);
    const int nq = rq.y - rq.x, nk = rk.y - rk.x, i0 = it.at * AT_BM, w = (int)min(a.window, 0x7FFFFFFFu);
    const int kh = head / (a.heads / a.kv_heads);
    // positions: of the workgroup's first and last row, the wavefront's, the lane's
    const int p_first = nk - nq + i0, p_last = nk - nq + min(i0 + (int)AT_BM, nq) - 1;
    const int w_first = p_first + 32 * (int)wave, w_last = min(w_first + 31, p_last);
    const int row = i0 + 32 * (int)wave + (int)(lane & 31);
    const int pos = nk - nq + row, hi = pos + 1, lo = w ? pos - w + 1 : 0;
    const int j_end = p_last + 1, j_begin = w ? max(p_first - w + 1, 0) / BN * BN : 0;

    const T *kp = (const T *)a.k + rk.x * a.ks + (uint64_t)kh * a.kh, *vp = (const T *)a.v + rk.x * a.vs + (uint64_t)kh * a.vh;
    const uint32_t h = lane >> 5;
    // queries: parts of dimensions 16 k + 8 h .. + 7 of the lane's row.  The scale's sign goes to them.
    float c = a.scale * 1.4426950408889634f;
    const uint32_t flip = c < 0 ? 0x80008000u : 0;
    c = fabsf(c) < 1e-30f ? 1e-30f : fabsf(c);  // (a factor of 0 would make NaN of a masked -inf)
    u32x4v q[NP][KS];
    {
        const T *qp = (const T *)a.q + (uint64_t)(rq.x + min(row, nq - 1)) * a.qs + (uint64_t)head * a.qh + 8 * h;
#pragma unroll
        for (int k = 0; k < KS; k++) {
            if (!FULL && 16 * k >= (int)D) break;
            if constexpr (NP == 1) {
                q[0][k] = *(const u32x4v *)(qp + 16 * k) ^ flip;
            } else {
                const floatx4 x = *(const floatx4 *)(qp + 16 * k), y = *(const floatx4 *)(qp + 16 * k + 4);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    uint32_t s0, s1, s2;
                    at_split(i < 2 ? x[2 * i] : y[2 * i - 4], i < 2 ? x[2 * i + 1] : y[2 * i - 3], s0, s1, s2);
                    q[0][k][i] = s0 ^ flip, q[1][k][i] = s1 ^ flip, q[2][k][i] = s2 ^ flip;
                }
            }
        }
    }

    // staging
    constexpr uint32_t RPP = 1024 / ROW;              // rows of a 1 KB piece: one instruction of a wavefront
    constexpr int PIECES = (int)(PB / 1024 / 4);      // a wavefront's, K and V each
    constexpr int XV = BN * DP / 4 / AT_NT;           // fp32: 16-byte loads a thread, K and V each
    uint32_t koff[2], voff;
    floatx4 xk[NP == 3 ? XV : 1], xv[NP == 3 ? XV : 1];
    if constexpr (NP == 1) {
        const uint32_t r = wave * RPP + lane / CPR, cc = lane % CPR;
#pragma unroll
        for (int p = 0; p < 2; p++)
            koff[p] = r * (uint32_t)(a.ks * 2) + min(cc ^ at_fk<CPR>(r + p * 4 * RPP), D / 8 - 1) * 16;
        voff = r * (uint32_t)(a.vs * 2) + min(cc ^ at_fv<CPR>(r), D / 8 - 1) * 16;
    }
    auto issue = [&](int j, int buf) {
        if constexpr (NP == 1) {
            // rows past the sequence's end lie past the buffer's (whole offsets in the lanes: the
            // range check may leave the scalar one out)
            const uint32_t rows = (uint32_t)min(nk - j, BN);
            auto rk_ = __builtin_amdgcn_make_buffer_rsrc((void *)(kp + (uint64_t)j * a.ks), 0,
                                                         (rows - 1) * (uint32_t)(a.ks * 2) + D * 2, 0x00027000);
            auto rv_ = __builtin_amdgcn_make_buffer_rsrc((void *)(vp + (uint64_t)j * a.vs), 0,
                                                         (rows - 1) * (uint32_t)(a.vs * 2) + D * 2, 0x00027000);
            using lds_t = __attribute__((address_space(3))) void;
            uint8_t *to = at_mem + buf * 2 * PB + wave * 1024;
#pragma unroll
            for (int p = 0; p < PIECES; p++)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rk_, (lds_t *)(to + p * 4096), 16,
                                                         koff[p & 1] + p * 4 * RPP * (uint32_t)(a.ks * 2), 0, 0, 0);
#pragma unroll
            for (int p = 0; p < PIECES; p++)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rv_, (lds_t *)(to + PB + p * 4096), 16,
                                                         voff + p * 4 * RPP * (uint32_t)(a.vs * 2), 0, 0, 0);
        } else {
#pragma unroll
            for (int i = 0; i < XV; i++) {
                const uint32_t e = threadIdx.x + i * AT_NT, r = e / (DP / 4), d = min(e % (DP / 4) * 4, D - 4);
                const uint64_t rr = (uint32_t)min(j + (int)r, nk - 1);
                xk[i] = *(const floatx4 *)(kp + rr * a.ks + d);
                xv[i] = *(const floatx4 *)(vp + rr * a.vs + d);
            }
        }
    };
    auto store = [&]() {
        if constexpr (NP == 3) {
#pragma unroll
            for (int i = 0; i < XV; i++) {
                const uint32_t e = threadIdx.x + i * AT_NT, r = e / (DP / 4), c4 = e % (DP / 4);
                uint8_t *pk = at_mem + r * ROW + ((c4 / 2) ^ at_fk<CPR>(r)) * 16 + c4 % 2 * 8;
                uint8_t *pv = at_mem + NP * PB + r * ROW + ((c4 / 2) ^ at_fv<CPR>(r)) * 16 + c4 % 2 * 8;
                u32x2v s[3];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    uint32_t s0, s1, s2;
                    at_split(xk[i][2 * u], xk[i][2 * u + 1], s0, s1, s2);
                    s[0][u] = s0, s[1][u] = s1, s[2][u] = s2;
                }
#pragma unroll
                for (int p = 0; p < 3; p++) *(u32x2v *)(pk + p * PB) = s[p];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    uint32_t s0, s1, s2;
                    at_split(xv[i][2 * u], xv[i][2 * u + 1], s0, s1, s2);
                    s[0][u] = s0, s[1][u] = s1, s[2][u] = s2;
                }
#pragma unroll
                for (int p = 0; p < 3; p++) *(u32x2v *)(pv + p * PB) = s[p];
            }
        }
    };

    floatx16 o[DT] = {};
    float m = -__builtin_inff(), l = 0;
    // this lane's part of the LDS addresses: K row lane % 32, V row and chunk of the transposed read
    const uint32_t kl = (lane & 31) * ROW, kx = h ^ at_fk<CPR>(lane & 31);
    const uint32_t vr = 4 * h + (lane & 15) / 4, vl = vr * ROW + (lane & 1) * 8, vx = ((lane >> 4 & 1) * 2 + (lane & 3) / 2);
    const uint32_t vf = at_fv<CPR>(vr);
    auto read_v = [&](const uint8_t *v, int kk, int dt) {
        const uint8_t *p = v + vl + kk * 16 * ROW + ((4 * dt + vx) ^ vf) * 16;
        using lds4 = __attribute__((address_space(3))) shortx4;
        const u32x2v x = __builtin_bit_cast(u32x2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)p));
        const u32x2v y = __builtin_bit_cast(u32x2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)(p + 8 * ROW)));
        return u32x4v{x[0], x[1], y[0], y[1]};
    };

    if (j_begin < j_end) issue(j_begin, 0);
    int buf = 0;
    for (int j = j_begin; j < j_end; j += BN) {
        if constexpr (NP == 1) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();  // (this tile is whole, the other buffer's readers are done)
            if (j + BN < j_end) issue(j + BN, buf ^ 1);
        } else {
            __syncthreads();
            store();
            __syncthreads();
            if (j + BN < j_end) issue(j + BN, 0);
        }
        const uint8_t *K = at_mem + (NP == 1 ? buf * 2 * PB : 0), *V = K + NP * PB;
        buf ^= 1;
        if (j > w_last || (w && j + BN <= w_first - w + 1)) continue;  // nothing for this wavefront
        const bool whole = j + BN - 1 <= w_first && (!w || j >= w_last - w + 1);

        floatx16 s[TT];
#pragma unroll
        for (int t = 0; t < TT; t++) {
            floatx16 acc = {};
#pragma unroll
            for (int k = 0; k < KS; k++) {
                if (!FULL && 16 * k >= (int)D) break;
                const uint8_t *p = K + t * 32 * ROW + kl + ((2 * k) ^ kx) * 16;
                if constexpr (NP == 1) {
                    acc = at_mfma<E>(*(const u32x4v *)p, q[0][k], acc);
                } else {
                    const u32x4v k0 = *(const u32x4v *)p, k1 = *(const u32x4v *)(p + PB), k2 = *(const u32x4v *)(p + 2 * PB);
                    acc = at_mfma<E>(k2, q[0][k], acc);
                    acc = at_mfma<E>(k0, q[NP - 1][k], acc);
                    acc = at_mfma<E>(k1, q[NP / 2][k], acc);
                    acc = at_mfma<E>(k1, q[0][k], acc);
                    acc = at_mfma<E>(k0, q[NP / 2][k], acc);
                    acc = at_mfma<E>(k0, q[0][k], acc);
                }
            }
            s[t] = acc;
        }
        if constexpr (NP == 3) {
            // 0 * infinity between parts makes NaN of a score that is infinite: such ones again, in fp32
            bool nan = false;
#pragma unroll
            for (int i = 0; i < 16; i++) nan |= s[0][i] != s[0][i];
            if (__ballot(nan)) {
                const T *qp = (const T *)a.q + (uint64_t)(rq.x + min(row, nq - 1)) * a.qs + (uint64_t)head * a.qh;
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int jj = j + 8 * (i / 4) + 4 * (int)h + i % 4;
                    if (s[0][i] != s[0][i] && jj < hi && jj >= lo) {
                        float x = 0;
                        for (uint32_t d = 0; d < D; d++) x = fmaf((float)qp[d], (float)kp[(uint64_t)jj * a.ks + d], x);
                        s[0][i] = flip ? -x : x;
                    }
                }
            }
        }
        if (!whole) {
#pragma unroll
            for (int t = 0; t < TT; t++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int jj = j + 32 * t + 8 * (i / 4) + 4 * (int)h + i % 4;
                    if (jj >= hi || jj < lo) s[t][i] = -__builtin_inff();
                }
        }
        float x = s[0][0];
#pragma unroll
        for (int t = 0; t < TT; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) x = fmaxf(x, s[t][i]);
        x = fmaxf(x, __shfl_xor(x, 32));
        // The running maximum moves only when it is passed by a factor of 2^8: weights of up to
        // 256 lose nothing, and most tiles need no new factors.
        if (__ballot((x - m) * c > 8.0f || (m == -__builtin_inff() && x > m))) {
            const float nm = fmaxf(m, x);
            const float f = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((m - nm) * c);
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; d++) o[d] *= f;
            m = nm;
        }
        // (f16: weights up to 2^8 2^7, so that those 2^-30 of the largest are still normal or nearly so)
        const float mc = (m == -__builtin_inff() ? 0.0f : m * c) - (__is_same(E, _Float16) ? 7.0f : 0.0f);
        u32x4v p[NP][2 * TT];
#pragma unroll
        for (int t = 0; t < TT; t++)
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const float e0 = __builtin_amdgcn_exp2f(fmaf(s[t][i], c, -mc)), e1 = __builtin_amdgcn_exp2f(fmaf(s[t][i + 1], c, -mc));
                l += e0 + e1;
                if constexpr (NP == 1) {
                    p[0][2 * t + i / 8][i % 8 / 2] = at_pack<E>(e0, e1);
                } else {
                    uint32_t s0, s1, s2;
                    at_split(e0, e1, s0, s1, s2);
                    p[0][2 * t + i / 8][i % 8 / 2] = s0;
                    p[NP / 2][2 * t + i / 8][i % 8 / 2] = s1;
                    p[NP - 1][2 * t + i / 8][i % 8 / 2] = s2;
                }
            }
        bool clean = true;
        if (!whole) {
            // an infinity or NaN among the values would reach rows that do not see it: 0 * NaN
            constexpr uint32_t EXP = __is_same(E, _Float16) ? 0x7C007C00u : 0x7F807F80u, ONE = __is_same(E, _Float16) ? 0x04000400u : 0x00800080u;
            uint32_t bad = 0;
            for (uint32_t e = lane; e < PB / 16; e += 64) {
                const u32x4v x4 = *(const u32x4v *)(V + e * 16);
#pragma unroll
                for (int i = 0; i < 4; i++) bad |= (x4[i] & EXP) + ONE;
            }
            clean = !__ballot((bad & 0x80008000u) != 0);
        }
        if (clean) {
#pragma unroll
            for (int kk = 0; kk < 2 * TT; kk++)
#pragma unroll
                for (int dt = 0; dt < DT; dt++) {
                    if (!FULL && 32 * dt >= (int)D) break;
                    const u32x4v v0 = read_v(V, kk, dt);
                    if constexpr (NP == 1) {
                        o[dt] = at_mfma<E>(v0, p[0][kk], o[dt]);
                    } else {
                        const u32x4v v1 = read_v(V + PB, kk, dt), v2 = read_v(V + 2 * PB, kk, dt);
                        o[dt] = at_mfma<E>(v2, p[0][kk], o[dt]);
                        o[dt] = at_mfma<E>(v0, p[NP - 1][kk], o[dt]);
                        o[dt] = at_mfma<E>(v1, p[NP / 2][kk], o[dt]);
                        o[dt] = at_mfma<E>(v1, p[0][kk], o[dt]);
                        o[dt] = at_mfma<E>(v0, p[NP / 2][kk], o[dt]);
                        o[dt] = at_mfma<E>(v0, p[0][kk], o[dt]);
                    }
                }
        } else {
            // key by key: its products alone, taken by the rows that see it
#pragma unroll 1
            for (int key = 0; key < BN; key++) {
                const int kk = key / 16, e = key % 16;   // e = 4 (half) + (e & 3) + 8 (second four)
                const bool mine = (e / 4 & 1) == (int)h;
                const int el = (e & 3) + (e >= 8 ? 4 : 0);
                const bool seen = j + key < hi && j + key >= lo;
                u32x4v y[NP];
#pragma unroll
                for (int pp = 0; pp < NP; pp++) {
                    y[pp] = u32x4v{0, 0, 0, 0};
#pragma unroll
                    for (int kq = 0; kq < 2 * TT; kq++)
                        if (kq == kk) y[pp] = p[pp][kq];
                }
                u32x4v mask;
#pragma unroll
                for (int i = 0; i < 4; i++) mask[i] = mine && el / 2 == i ? (el & 1 ? 0xFFFF0000u : 0x0000FFFFu) : 0;
#pragma unroll
                for (int dt = 0; dt < DT; dt++) {
                    if (!FULL && 32 * dt >= (int)D) break;
                    floatx16 one = {};
#pragma unroll
                    for (int vv = 0; vv < NP; vv++) {
                        const u32x4v x = read_v(V + vv * PB, kk, dt) & mask;
#pragma unroll
                        for (int pp = 0; pp < NP - vv; pp++) one = at_mfma<E>(x, y[pp] & mask, one);
                    }
#pragma unroll
                    for (int i = 0; i < 16; i++) o[dt][i] += seen ? one[i] : 0.0f;
                }
            }
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
            if (!FULL && d >= D) break;
            if constexpr (NP == 1) {
                u32x2v r = {at_pack<E>(o[dt][i] * inv, o[dt][i + 1] * inv), at_pack<E>(o[dt][i + 2] * inv, o[dt][i + 3] * inv)};
                if (l == 0) r = {0, 0};
                *(u32x2v *)(out + d) = r;
            } else {
                *(floatx4 *)(out + d) = l != 0 ? floatx4{o[dt][i] * inv, o[dt][i + 1] * inv, o[dt][i + 2] * inv, o[dt][i + 3] * inv}
                                               : floatx4{0, 0, 0, 0};
            }
        }
}

}  // namespace okf
