// okf_rope.h -- norms of queries and keys for each head with the rotation by positions in
// the same pass (okf_norm_rope_rows).
//
// y = R(pos) (x w / sqrt(mean(x^2) + eps)): the norm's sum goes over a head, R turns the
// pairs of its first rot dimensions.  Bound by memory: every value is read once and
// written once, some 8 operations for each.  8192 rows of 40 + 8 bf16 heads of 128 with norms: 43 us, 4.7 TB/s in
// and out (a large copy 5.15); one row of 16 + 8 fp32 heads 3.5 us, the launch and a chain of two loads.
#pragma once
#include "okf_kv_seqs.h"

namespace okf {

constexpr int RP_NT = 256;

struct RopeArgs {
    const void *q, *k;
    void *qo, *ko;
    uint64_t qs, ks, qos, kos, qh, kh, qoh, koh;
    const float *qn, *kn, *div;
    const int32_t *pos;
    uint32_t heads, kv, dim, n, rot;
    int32_t pairs;
    uint32_t tq, tk;   // tasks of queries and of keys: as many heads as a wavefront takes at once
    uint32_t per, wpr; // tasks a wavefront, wavefronts a row
    float eps, mag;
    double f[128];     // turns a position of each pair
};

// cos and sin of 2 pi t: t less the nearest quarter is at most 1/8, where the series of
// both in x = 2 pi t, |x| <= pi / 4, are left off below 1.2e-10; the quarter swaps and signs them.
__device__ __forceinline__ float2 rp_turn(double t) {
    t -= rint(t);
    const double q = rint(4 * t);
    const float x = (float)(fma(q, -0.25, t) * 6.283185307179586), z = x * x;
    const float s = fmaf(x * z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1.0f / 39916800, 1.0f / 362880), -1.0f / 5040), 1.0f / 120), -1.0f / 6), x);
    const float c = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1.0f / 3628800, 1.0f / 40320), -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
    const int n = (int)q;  // -2 .. 2
    const float a = n & 1 ? s : c, b = n & 1 ? c : s;
    return {n == 1 || n == 2 || n == -2 ? -a : a, n == 2 || n == -1 || n == -2 ? -b : b};
}

// Sum over the L lanes of a group; every lane gets it.
template <int L>
__device__ __forceinline__ float rp_sum(float x) {
    auto dpp = [](float v, auto ctrl) {  // (ctrl: a constant)
        return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), decltype(ctrl)::value, 0xF, 0xF, true));
    };
    if constexpr (L > 1) x += dpp(x, std::integral_constant<int, 0xB1>{});   // quads: neighbours
    if constexpr (L > 2) x += dpp(x, std::integral_constant<int, 0x4E>{});   // ... pairs
    if constexpr (L > 4) x += dpp(x, std::integral_constant<int, 0x141>{});  // mirrored halves of a row
    if constexpr (L > 8) x += dpp(x, std::integral_constant<int, 0x140>{});  // the row mirrored
    if constexpr (L > 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return x;
}

// 16 bytes of T as floats, and back.
template <class T>
__device__ __forceinline__ void rp_load(const T *p, float *x) {
    typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
    const vec v = *(const vec *)p;
#pragma unroll
    for (uint32_t j = 0; j < 16 / sizeof(T); j++) x[j] = to_f32(v[j]);
}
template <class T>
__device__ __forceinline__ void rp_store(T *p, const float *x) {
    typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
    vec v;
#pragma unroll
    for (uint32_t j = 0; j < 16 / sizeof(T); j++) v[j] = (T)x[j];
    *(vec *)p = v;
}

// A wavefront takes rows, and of each `per` tasks of G = 64 / L heads; L lanes hold a head,
// 32 bytes each: where the pairs are neighbours, contiguous ones; where they are a head's
// halves, 16 of each half, so that a lane holds both of a pair.  Halves that do not
// break at 16 bytes (CROSS) are exchanged through LDS.  The row's angles are computed
// once, one or two a lane, and handed round through LDS.
template <class T, int L, bool CROSS>
__global__ __launch_bounds__(RP_NT) void norm_rope_kernel(const RopeArgs a) {
    constexpr uint32_t V = 16 / sizeof(T), G = 64 / L;
    __shared__ float2 turns[RP_NT / 64][128];
    __shared__ __align__(16) float norms[2][256];
    __shared__ float cross[CROSS ? RP_NT / 64 : 1][CROSS ? 64 * 2 * V : 1];
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63, u = lane % L;
    const uint32_t w = blockIdx.x * (RP_NT / 64) + wave, half = a.rot / 2;
    const uint32_t first = w % a.wpr * a.per, last = min(first + a.per, a.tq + a.tk), step = gridDim.x * (RP_NT / 64) / a.wpr;
    const bool mine = u < a.dim / (2 * V);
    // the lane's two pieces of a head: their first dimensions, and how many of their pairs turn
    uint32_t d0 = 2 * u * V, d1 = d0 + V;
    if (!CROSS && !a.pairs && a.rot) {
        const uint32_t hc = half / V;  // (whole pieces of a half)
        d0 = u < hc ? u * V : 2 * u * V;
        d1 = u < hc ? d0 + half : d0 + V;
    }
    // the norms' weights, once for the workgroup's rows
    for (uint32_t i = threadIdx.x; i < 2 * a.dim; i += RP_NT) {
        const float *nw = i < a.dim ? a.qn : a.kn;
        if (nw) norms[i >= a.dim][i < a.dim ? i : i - a.dim] = nw[i < a.dim ? i : i - a.dim];
    }
    __syncthreads();
    const float per_dim = 1.0f / (float)a.dim;
    const uint32_t turning = half > u * V ? min(half - u * V, V) : 0;
    for (uint32_t row = w / a.wpr; row < a.n; row += step) {
        if (a.rot) {
            const double p = a.pos[row];
#pragma unroll
            for (uint32_t i = lane; i < 128; i += 64)
                if (i < half) {
                    const double f = a.div ? a.f[i] / (double)a.div[i] : a.f[i], t = p * f;
                    const float2 cs = rp_turn(fma(p, f, -rint(t)));
                    turns[wave][i] = {cs.x * a.mag, cs.y * a.mag};
                }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        float2 cs[V];
#pragma unroll
        for (uint32_t j = 0; j < V; j++) cs[j] = !CROSS && j < turning ? turns[wave][u * V + j] : float2{1.0f, 0.0f};
        for (uint32_t t = first; t < last; t++) {
            const bool key = t >= a.tq;
            const uint32_t head = (key ? t - a.tq : t) * G + lane / L;
            const bool on = mine && head < (key ? a.kv : a.heads);
            const T *x = key ? (const T *)a.k + row * a.ks + head * a.kh : (const T *)a.q + row * a.qs + head * a.qh;
            T *y = key ? (T *)a.ko + row * a.kos + head * a.koh : (T *)a.qo + row * a.qos + head * a.qoh;
            float v[2 * V], g[2 * V];
#pragma unroll
            for (uint32_t j = 0; j < 2 * V; j++) v[j] = 0.0f;
            if (on) rp_load(x + d0, v), rp_load(x + d1, v + V);
            if (key ? a.kn : a.qn) {
                const float *nw = norms[key];
#pragma unroll
                for (uint32_t j = 0; j < V; j += 4) {
                    const floatx4 x0 = *(const floatx4 *)(nw + (mine ? d0 : 0) + j), x1 = *(const floatx4 *)(nw + (mine ? d1 : 0) + j);
#pragma unroll
                    for (uint32_t i = 0; i < 4; i++) g[j + i] = x0[i], g[V + j + i] = x1[i];
                }
                float ss = 0;
#pragma unroll
                for (uint32_t j = 0; j < 2 * V; j++) ss = fmaf(v[j], v[j], ss);
                const float r = __builtin_amdgcn_rsqf(fmaf(rp_sum<L>(ss), per_dim, a.eps));  // (right to one step)
#pragma unroll
                for (uint32_t j = 0; j < 2 * V; j++) v[j] = v[j] * r * g[j];
            }
            if constexpr (CROSS) {
                float *all = cross[wave] + lane / L * (L * 2 * V);
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
                for (uint32_t j = 0; j < 2 * V; j++) all[2 * u * V + j] = v[j];
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
                for (uint32_t j = 0; j < 2 * V; j++) {
                    const uint32_t d = 2 * u * V + j;
                    if (d < a.rot) {
                        const bool low = d < half;
                        const float2 c = turns[wave][low ? d : d - half];
                        const float o = all[low ? d + half : d - half];
                        v[j] = low ? v[j] * c.x - o * c.y : o * c.y + v[j] * c.x;
                    }
                }
            } else if (turning) {  // (a lane's pairs turn, but for those that the end of rot cuts off)
                auto turn = [&](float &x0, float &x1, uint32_t j) {
                    const float y0 = x0 * cs[j].x - x1 * cs[j].y, y1 = x0 * cs[j].y + x1 * cs[j].x;
                    if (j < turning) x0 = y0, x1 = y1;
                };
                if (a.pairs) {
#pragma unroll
                    for (uint32_t j = 0; j < V; j++) turn(v[2 * j], v[2 * j + 1], j);
                } else {
#pragma unroll
                    for (uint32_t j = 0; j < V; j++) turn(v[j], v[V + j], j);
                }
            }
            if (on) rp_store(y + d0, v), rp_store(y + d1, v + V);
        }
    }
}

}  // namespace okf
