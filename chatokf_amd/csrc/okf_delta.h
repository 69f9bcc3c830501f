// okf_delta.h -- the gated delta rule token by token (okf_delta_step), and what both of
// its forms share.
//
// Per value head a state S [k_dim][v_dim] takes each token as S <- e^g S, S += k u^T with
// u = beta (v - S^T k), o = scale S^T q.  With r = S^T k and p = S^T q of the state before the
// token that is u = beta (v - e^g r), S <- e^g S + k u^T and o = scale (e^g p + (q.k) u), so that
// one pass over the state reads it for both.
#pragma once
#include "okf_conv.h"

namespace okf {

struct DeltaArgs {
    const void *q, *k, *v;
    const float *g, *beta;
    void *o;
    uint64_t qs, ks, vs, os, gs, bs;
    uint32_t k_heads, v_heads, k_dim, v_dim;
    float scale;
    const float *si;
    float *so;
    StateSeqs s;
};

template <int CTRL>
__device__ __forceinline__ float dl_lane(float x) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), CTRL, 0xF, 0xF, true));
}
// Sum over the 4 lanes of the same l % 16, in every one of them.
__device__ __forceinline__ float dl_sum_rows(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
// Sum over the lanes of the same l % CQ, in every one of them.
template <int CQ>
__device__ __forceinline__ float dl_sum_groups(float x) {
    x += dl_lane<0x128>(x);  // (rows of 16 lanes turned by 8, by 4)
    if constexpr (CQ == 4) x += dl_lane<0x124>(x);
    return dl_sum_rows(x);
}

constexpr int DS_NT = 256;

// A wavefront holds 4 CQ columns of one head's state, four a lane, over its 64 / CQ lanes of
// RK = k_dim CQ / 64 rows each.  Bound by the state's bytes, 64 KB in and 64 KB out for a head of 128 x 128: 32 sequences of 48
// such heads 43 us, 4.7 TB/s.  One sequence 5 us, a chain of loads; a token more 1.1 us (fp32), its two sums over the
// lanes behind each other (its loads made a token ahead: 0.9, and slower where 256 rows then fill the registers).
template <class T, int CQ, int RK>
__global__ __launch_bounds__(DS_NT) void delta_step_kernel(const DeltaArgs a) {
    const uint32_t lane = threadIdx.x & 63, rg = lane / CQ, tiles = (a.v_dim + 4 * CQ - 1) / (4 * CQ);
    const uint32_t w = blockIdx.x * (DS_NT / 64) + (threadIdx.x >> 6);
    const uint32_t tile = w % tiles, h = w / tiles % a.v_heads, s = w / tiles / a.v_heads;
    if (s >= a.s.count) return;
    // (columns past the last: the last's again, not written)
    const uint32_t place = (tile * CQ + lane % CQ) * 4, col = min(place, a.v_dim - 4), kh = h / (a.v_heads / a.k_heads), row0 = rg * RK;
    const bool on = place < a.v_dim;
    const uint2 r = kv_rows(a.s.start, s, a.s.n);
    const int64_t slot = a.s.state(s);
    floatx4 S[RK];
    const uint64_t at = (((uint64_t)(slot < 0 ? 0 : slot) * a.v_heads + h) * a.k_dim + row0) * a.v_dim + col;
    if (a.si && slot >= 0) {
#pragma unroll
        for (int i = 0; i < RK; i++) S[i] = *(const floatx4 *)(a.si + at + (uint64_t)i * a.v_dim);
    } else {
#pragma unroll
        for (int i = 0; i < RK; i++) S[i] = floatx4{0, 0, 0, 0};
    }
    const T *q = (const T *)a.q + kh * a.k_dim + row0, *k = (const T *)a.k + kh * a.k_dim + row0;
    const T *v = (const T *)a.v + h * a.v_dim + col;
    T *o = (T *)a.o + h * a.v_dim + col;
    for (uint32_t t = r.x; t < r.y; t++) {
        float kt[RK], qt[RK], kq = 0;
        floatx4 vt, kr{0, 0, 0, 0}, qr{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < RK; i++) kt[i] = to_f32(k[t * a.ks + i]), qt[i] = to_f32(q[t * a.qs + i]);
#pragma unroll
        for (int j = 0; j < 4; j++) vt[j] = to_f32(v[t * a.vs + j]);
        const float e = expf(a.g[t * a.gs + h]), beta = a.beta[t * a.bs + h];
#pragma unroll
        for (int i = 0; i < RK; i++) {
            kq = fmaf(kt[i], qt[i], kq);
#pragma unroll
            for (int j = 0; j < 4; j++) kr[j] = fmaf(kt[i], S[i][j], kr[j]), qr[j] = fmaf(qt[i], S[i][j], qr[j]);
        }
        kq = dl_sum_groups<CQ>(kq);
        floatx4 u;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            kr[j] = dl_sum_groups<CQ>(kr[j]), qr[j] = dl_sum_groups<CQ>(qr[j]);
            u[j] = beta * (vt[j] - (e == 0 ? 0.0f : e * kr[j]));
            qr[j] = ((e == 0 ? 0.0f : e * qr[j]) + kq * u[j]) * a.scale;
        }
#pragma unroll
        for (int i = 0; i < RK; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) S[i][j] = fmaf(kt[i], u[j], e == 0 ? 0.0f : e * S[i][j]);
        if (rg == 0 && on) {
            typedef T vec __attribute__((ext_vector_type(4)));
            vec x;
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] = (T)qr[j];
            *(vec *)(o + t * a.os) = x;
        }
    }
    if (a.so && slot >= 0 && on) {
#pragma unroll
        for (int i = 0; i < RK; i++) *(floatx4 *)(a.so + at + (uint64_t)i * a.v_dim) = S[i];
    }
}

}  // namespace okf
