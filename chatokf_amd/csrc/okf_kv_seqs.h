// okf_kv_seqs.h -- the paged KV cache and packed sequences as kernels take them.
#pragma once
#include "okf_common.h"

namespace okf {

constexpr uint32_t KV_B = 64;  // tokens a page

struct KvCache {
    int8_t *k, *v;
    float *ks, *vs;
    uint32_t pages, heads, dim;
};

struct KvSeqs {
    const int32_t *pages;
    int32_t *len;
    uint32_t count, stride;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(_Float16 x) { return (float)x; }
__device__ __forceinline__ float to_f32(__bf16 x) { return (float)x; }

// x of the lane CTRL says, 0 where there is none (a lane of the row of 16, or the last
// one of the rows before, for the rows of RM).
template <int CTRL, int RM>
__device__ __forceinline__ uint32_t lane_of(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, RM, 0xF, false);
}
// Sums of the lanes up to this one; the largest of all lanes.  (Shuffles by way of LDS took
// half a microsecond for the six steps.)
__device__ __forceinline__ uint32_t lanes_sum(uint32_t x) {
    x += lane_of<0x111, 0xF>(x);
    x += lane_of<0x112, 0xF>(x);
    x += lane_of<0x114, 0xF>(x);
    x += lane_of<0x118, 0xF>(x);
    x += lane_of<0x142, 0xA>(x);
    x += lane_of<0x143, 0xC>(x);
    return x;
}
__device__ __forceinline__ uint32_t lanes_max(uint32_t x) {
    x = max(x, lane_of<0x111, 0xF>(x));
    x = max(x, lane_of<0x112, 0xF>(x));
    x = max(x, lane_of<0x114, 0xF>(x));
    x = max(x, lane_of<0x118, 0xF>(x));
    x = max(x, lane_of<0x142, 0xA>(x));
    x = max(x, lane_of<0x143, 0xC>(x));
    return (uint32_t)__builtin_amdgcn_readlane(x, 63);
}

// The sequence that item idx belongs to when sequence s has items(s) of them,
// and the item's place in it; seq = count past the last.  Every lane of the
// wavefront calls this with the same idx and gets the same answer.
struct SeqItem {
    uint32_t seq, at;
};
template <class F>
__device__ __forceinline__ SeqItem kv_find(uint32_t idx, uint32_t count, F items) {
    const uint32_t lane = threadIdx.x & 63;
    uint64_t before = 0;
    for (uint32_t b = 0; b < count; b += 64) {  // (64 sequences' items stay below 2^32: rows do)
        const uint32_t n = b + lane < count ? items(b + lane) : 0, sum = lanes_sum(n);
        const uint64_t here = __ballot(before + sum > idx);
        if (here) {
            const int l = __ffsll((unsigned long long)here) - 1;
            return {b + l, (uint32_t)__builtin_amdgcn_readlane(idx - (uint32_t)before - (sum - n), l)};
        }
        before += (uint32_t)__builtin_amdgcn_readlane(sum, 63);
    }
    return {count, 0};
}

// The rows [a, b) that packed starts give a sequence, inside [0, n].
__device__ __forceinline__ uint2 kv_rows(const int32_t *start, uint32_t s, uint32_t n) {
    const uint32_t a = (uint32_t)min(max(start[s], 0), (int)n);
    return {a, (uint32_t)min(max(start[s + 1], (int)a), (int)n)};
}

}  // namespace okf
