// okf_attn.h -- causal attention over packed prompts (okf_attn_prompt).
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
};

constexpr int AT_NT = 256;

template <int NT>
__device__ __forceinline__ float at_max(float v, float *red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float r = red[0];
#pragma unroll
    for (int w = 1; w < NT / 64; w++) r = fmaxf(r, red[w]);
    return r;
}

// One row of attention by a workgroup, chunk by chunk of AT_NT keys with the
// running maximum and sum: key(j) the scaled score of key j, value(j, d).
// Returns dimension threadIdx.x of the result; m and l are the maximum and sum.
template <class S, class V>
__device__ __forceinline__ float at_row(uint32_t lo, uint32_t hi, uint32_t D, float *p, float *red, S key, V value,
                                        float &m, float &l) {
    const uint32_t tid = threadIdx.x;
    float acc = 0;
    m = -__builtin_inff();
    l = 0;
    for (uint32_t b = lo; b < hi; b += AT_NT) {
        const uint32_t n = min(hi - b, (uint32_t)AT_NT);
        const float s = tid < n ? key(b + tid) : -__builtin_inff();
        const float nm = fmaxf(m, at_max<AT_NT>(s, red)), ref = nm == -__builtin_inff() ? 0.0f : nm;
        const float f = expf(m - ref), e = expf(s - ref);
        p[tid] = e;
        __syncthreads();
        acc *= f;
        l *= f;
        if (tid < D)
            for (uint32_t j = 0; j < n; j++) acc += p[j] * value(b + j, tid);
        for (uint32_t j = 0; j < n; j++) l += p[j];
        m = nm;
        __syncthreads();
    }
    return l != 0 ? acc / l : 0.0f;
}

template <class T>
__global__ __launch_bounds__(AT_NT) void attn_prompt_kernel(AttnArgs a) {
    __shared__ float q[256], p[AT_NT], red[AT_NT / 64];
    const uint32_t row = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, D = a.dim;
    const SeqItem it = kv_find(row, a.seqs, [&](uint32_t s) {
        const uint2 r = kv_rows(a.q_start, s, a.nq);
        return r.y - r.x;
    });
    if (it.seq >= a.seqs) return;
    const uint2 rq = kv_rows(a.q_start, it.seq, a.nq), rk = kv_rows(a.k_start, it.seq, a.nk);
    const uint32_t nk = rk.y - rk.x;
    const int64_t at = (int64_t)nk - (rq.y - rq.x) + it.at;  // the query's position
    const uint32_t hi = (uint32_t)max(at + 1, (int64_t)0);
    const uint32_t lo = a.window && hi > a.window ? hi - a.window : 0;
    const uint64_t r = rq.x + it.at;
    if (tid < D) q[tid] = to_f32(((const T *)a.q)[r * a.qs + h * a.qh + tid]);
    __syncthreads();
    const uint32_t kh = h / (a.heads / a.kv_heads);
    const T *k = (const T *)a.k + rk.x * a.ks + kh * a.kh, *v = (const T *)a.v + rk.x * a.vs + kh * a.vh;
    float m, l;
    const float o = at_row(
        lo, hi, D, p, red,
        [&](uint32_t j) {
            float s = 0;
            for (uint32_t d = 0; d < D; d++) s += q[d] * to_f32(k[j * a.ks + d]);
            return s * a.scale;
        },
        [&](uint32_t j, uint32_t d) { return to_f32(v[j * a.vs + d]); }, m, l);
    if (tid < D) ((T *)a.o)[r * a.os + h * a.oh + tid] = (T)o;
}

}  // namespace okf
