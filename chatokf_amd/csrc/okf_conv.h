// okf_conv.h -- the short causal convolution of each channel over packed sequences with
// their states (okf_conv_rows): y[t] = act(b + sum_j w[j] x[t - W + 1 + j]).
//
// Bound by memory: a value is read once (the W - 1 rows in front of a thread's first once
// more) and written once, 2 W + 4 operations for each.  7036 rows of 10240 channels, width 4, SiLU: fp32 123 us, 4.7 TB/s in and
// out; bf16 77 us, 3.8 TB/s: the vector units are busy for half of that, with conversions, products and SiLU, and wavefronts
// wait for a third of it, since a group's loads begin only when the one before is used up, behind its stores.
// 32 sequences of one fp32 row: 5.4 us, the search for the sequence and two loads behind each other.
#pragma once
#include "okf_kv_seqs.h"

namespace okf {

// Packed sequences and their states, as kernels take them.
struct StateSeqs {
    const int32_t *start, *slot;
    uint32_t count, n, slots;
    // the state of sequence s, -1: it begins from zeros and is not kept
    __device__ __forceinline__ int64_t state(uint32_t s) const {
        const int64_t i = slot ? slot[s] : (int64_t)s;
        return i < (int64_t)slots ? i : -1;
    }
};

struct ConvArgs {
    const void *x, *si;
    void *y, *so;
    const float *w, *b;
    uint64_t xs, ys;
    uint32_t channels, silu, rows;  // rows: that a thread goes through
    StateSeqs s;
};

// x / (1 + e^-x).  The reciprocal and the power of two are right to one step of the last place, and the
// power's argument -x log2 e to half a step, which moves the result by less than 0.6 2^-24.  (A true
// division and expf: a third more time for 16-bit rows.)
__device__ __forceinline__ float cv_silu(float x) {
    return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.4426950408889634f));
}

// A thread takes V channels (a 16-byte piece, or one) through up to `rows` rows of a sequence with the
// last W - 1 rows in registers.  The thread of a sequence's first rows has read its
// state before it writes what the sequence leaves, so that it may go to the same
// place.
// (Two wavefronts a SIMD at least: bf16 at width 8 has one without that, 512 rows 18.5 us for 15.6; with it a lane spills 20 bytes.)
template <class T, int W, int V>
__global__ __launch_bounds__(256, 2) void conv_kernel(const ConvArgs a) {
    typedef T vec __attribute__((ext_vector_type(V)));
    const SeqItem it = kv_find(blockIdx.x, a.s.count, [&](uint32_t s) {
        const uint2 r = kv_rows(a.s.start, s, a.s.n);
        return max((r.y - r.x + a.rows - 1) / a.rows, 1u);
    });
    const uint32_t c = (blockIdx.y * 256 + threadIdx.x) * V;
    if (it.seq >= a.s.count || c >= a.channels) return;
    const uint2 r = kv_rows(a.s.start, it.seq, a.s.n);
    const uint32_t first = r.x + it.at * a.rows, last = min(first + a.rows, r.y);
    if (it.at && first >= r.y) return;  // (not with starts that rise)
    const int64_t slot = a.s.state(it.seq);
    const T *x = (const T *)a.x + c;
    T *y = (T *)a.y + c;
    const bool held = a.si && slot >= 0;
    const T *si = (const T *)a.si + (held ? (uint64_t)slot * (W - 1) * a.channels + c : 0);
    vec h[W];  // the last W - 1 rows, and the next
#pragma unroll
    for (int j = 0; j < W - 1; j++) {
        vec v;
#pragma unroll
        for (int k = 0; k < V; k++) v[k] = (T)0.0f;
        const int64_t t = (int64_t)first + j - (W - 1);
        if (t >= (int64_t)r.x) v = *(const vec *)(x + t * a.xs);
        else if (held) v = *(const vec *)(si + (t - (int64_t)r.x + (W - 1)) * a.channels);
        h[j] = v;
    }
    float w[V][W], b[V];
#pragma unroll
    for (int k = 0; k < V; k++) {
        b[k] = a.b ? a.b[c + k] : 0.0f;
#pragma unroll
        for (int j = 0; j < W; j++) w[k][j] = a.w[(uint64_t)(c + k) * W + j];
    }
    if (it.at == 0 && a.so && slot >= 0) {
        // the rows len - W + 1 .. len - 1, those before the first from the state: they stand
        // behind the place that they go to, so that writing from the oldest on overwrites none of them
        T *so = (T *)a.so + (uint64_t)slot * (W - 1) * a.channels + c;
#pragma unroll
        for (int j = 0; j < W - 1; j++) {
            const int64_t t = (int64_t)r.y + j - (W - 1);
            vec v;
#pragma unroll
            for (int k = 0; k < V; k++) v[k] = (T)0.0f;
            if (t >= (int64_t)r.x) v = *(const vec *)(x + t * a.xs);
            else if (held) v = *(const vec *)(si + (t - (int64_t)r.x + (W - 1)) * a.channels);
            *(vec *)(so + (uint64_t)j * a.channels) = v;
        }
    }
    // (rows on their way at a time: 8 for 4 took 7036 bf16 rows of 10240 channels from 80 us to 77)
    constexpr uint32_t AHEAD = W * V <= 32 ? 8 : 4;
    for (uint32_t t = first; t < last; t += AHEAD) {
        vec in[AHEAD];
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; i++) in[i] = *(const vec *)(x + (uint64_t)min(t + i, last - 1) * a.xs);
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; i++) {
            if (t + i >= last) break;
            h[W - 1] = in[i];
            vec o;
#pragma unroll
            for (int k = 0; k < V; k++) {
                float s = b[k];
#pragma unroll
                for (int j = 0; j < W; j++) s = fmaf(w[k][j], to_f32(h[j][k]), s);
                o[k] = (T)(a.silu ? cv_silu(s) : s);
            }
            *(vec *)(y + (uint64_t)(t + i) * a.ys) = o;
#pragma unroll
            for (int j = 0; j < W - 1; j++) h[j] = h[j + 1];
        }
    }
}

}  // namespace okf
