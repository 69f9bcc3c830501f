// okf_attn_run.h -- the launches of attn_prompt_kernel, one instance of launch_prompt
// per type in okf_attn_<type>.hip, so that they compile in parallel.
#pragma once
#include "okf_impl.h"
#include "okf_attn.h"

namespace okf_impl {

template <class T, class S>
int launch_prompt_s(okf_ctx *c, okf::AttnArgs a) {
    using namespace okf;
    // (sequences' tiles: at most n_q / rows and one each; never more than the rows)
    const uint64_t tiles = std::min<uint64_t>((uint64_t)a.nq / S::BM + a.seqs, a.nq);
    uint64_t grid = tiles * a.heads;
    if (8 % a.kv_heads == 0) {  // (as the kernel deals them to the XCDs)
        const uint64_t each = 8 / a.kv_heads;
        grid = (tiles * (a.heads / a.kv_heads) + each - 1) / each * 8;
    }
    if (grid * S::NT > 0xFFFFFFFFull) return OKF_E_SHAPE;  // (a grid has less than 2^32 threads)
    a.tiles = (uint32_t)tiles;
    static std::atomic<uint64_t> attr{0};
    set_lds_attr(c, (const void *)attn_prompt_kernel<T, S>, attr);
    hipLaunchKernelGGL((attn_prompt_kernel<T, S>), dim3((uint32_t)grid), dim3(S::NT), (at_lds<S>()), c->stream, a);
    return OKF_OK;
}

// Which workgroups: 4 x 32 rows; 2 x 32 rows with the keys dealt to 2 groups of
// wavefronts, where 128 rows each would not fill the CUs (up to two 64-row tiles a CU); with
// 4 groups (8 wavefronts, one workgroup a CU), where there is one tile a CU at most and
// their keys are many.  Measured, us, for 4 x 1 / 2 x 2 / 2 x 4 (32 heads of 128, bf16; 64-row
// tiles x heads): 256 rows 11.8 / 9.2 / 10.5 (128 tiles), 1000 rows 26.3 / 21.7 / 26.0
// (512), behind 2000 keys 64 rows 43.4 / 34.0 / 29.0 (32), 500 rows 52.7 / 42.0 / 34.8 (256),
// 1000 rows 61.6 / 56.7 / 69.1 (512), 1300 rows 78.2 / 91.5 / 103.3 (672).  Shapes whose tiles
// do not fit LDS fall to the next.
template <class T, int DP, int DH>
int launch_prompt_d(okf_ctx *c, const okf::AttnArgs &a) {
    using namespace okf;
    const uint64_t tiles = std::min<uint64_t>(a.nq / 64 + a.seqs, a.nq) * a.heads;
    uint64_t keys = a.nk / a.seqs;  // a tile's
    if (a.window) keys = std::min<uint64_t>(keys, (uint64_t)a.window + 64);
    if constexpr (DH && at_fits<AtShape<T, DP, DH, 2, 4>>())
        if (tiles <= c->cus && keys >= 768) return launch_prompt_s<T, AtShape<T, DP, DH, 2, 4>>(c, a);
    if constexpr (at_fits<AtShape<T, DP, DH, 2, 2>>())
        if (tiles <= 2 * (uint64_t)c->cus) return launch_prompt_s<T, AtShape<T, DP, DH, 2, 2>>(c, a);
    return launch_prompt_s<T, AtShape<T, DP, DH, 4, 1>>(c, a);
}

template <class T>
int launch_prompt(okf_ctx *c, const okf::AttnArgs &a) {
    switch (a.dim) {
    case 64: return launch_prompt_d<T, 64, 64>(c, a);
    case 80: return launch_prompt_d<T, 128, 80>(c, a);
    case 96: return launch_prompt_d<T, 128, 96>(c, a);
    case 128: return launch_prompt_d<T, 128, 128>(c, a);
    case 256: return launch_prompt_d<T, 256, 256>(c, a);
    default:
        if (a.dim < 64) return launch_prompt_d<T, 64, 0>(c, a);
        if (a.dim < 128) return launch_prompt_d<T, 128, 0>(c, a);
        return launch_prompt_d<T, 256, 0>(c, a);
    }
}

#ifndef OKF_ATTN_TYPE
extern template int launch_prompt<float>(okf_ctx *, const okf::AttnArgs &);
extern template int launch_prompt<_Float16>(okf_ctx *, const okf::AttnArgs &);
extern template int launch_prompt<__bf16>(okf_ctx *, const okf::AttnArgs &);
#else
template int launch_prompt<OKF_ATTN_TYPE>(okf_ctx *, const okf::AttnArgs &);
#endif

}  // namespace okf_impl
