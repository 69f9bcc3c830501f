// okf_delta_run.h -- the launches of the gated delta rule, one instance of each per type in
// okf_delta_<type>.hip, so that they compile in parallel.
#pragma once
#include "okf_impl.h"
#include "okf_delta_scan.h"

namespace okf_impl {

// 16 columns a wavefront, or 32, whose rows are whole lines of 128 bytes, where those still leave
// DS_WAVES wavefronts a CU (32 sequences of 48 heads of 128 x 128: 43 us for 50; one sequence, spread
// over half the CUs: 5.2 for 4.8).
constexpr uint32_t DS_WAVES = 8;
template <class T, int RK = 1>
void launch_delta_step(okf_ctx *c, const okf::DeltaArgs &a) {
    if constexpr (RK < 16)
        if (a.k_dim != 16 * RK) return launch_delta_step<T, RK + 1>(c, a);
    const uint64_t heads = (uint64_t)a.s.count * a.v_heads, wide = heads * ((a.v_dim + 31) / 32), narrow = heads * (a.v_dim / 16);
    if (wide >= (uint64_t)DS_WAVES * c->cus)
        hipLaunchKernelGGL((okf::delta_step_kernel<T, 8, 2 * RK>), dim3((uint32_t)((wide + 3) / 4)), dim3(okf::DS_NT), 0, c->stream, a);
    else
        hipLaunchKernelGGL((okf::delta_step_kernel<T, 4, RK>), dim3((uint32_t)((narrow + 3) / 4)), dim3(okf::DS_NT), 0, c->stream, a);
}

// The chunks p.c0 .. p.c1 - 1: what each of them needs, then one behind the other.
template <class T, int KS = 1>
void launch_delta_chunks(okf_ctx *c, const okf::ScanArgs &p) {
    using namespace okf;
    if constexpr (KS < 8)
        if (p.a.k_dim > 32 * KS) return launch_delta_chunks<T, KS + 1>(c, p);
    constexpr uint32_t waves = DP_NT / 64;
    const uint32_t tasks = (p.c1 - p.c0) * p.a.k_heads * p.passes;
    hipLaunchKernelGGL((delta_prepare_kernel<T, KS>), dim3((tasks + waves - 1) / waves), dim3(DP_NT), 0, c->stream, p);
    static std::atomic<uint64_t> attr{0};
    set_lds_attr(c, (const void *)delta_scan_kernel<T, KS>, attr);
    const uint32_t grid = p.a.s.count * p.a.v_heads * ((p.a.v_dim / 16 + 1) / 2);
    hipLaunchKernelGGL((delta_scan_kernel<T, KS>), dim3(grid), dim3(DN_NT), dl_scan_lds<KS>(), c->stream, p);
}

#ifndef OKF_DELTA_TYPE
extern template void launch_delta_step<float>(okf_ctx *, const okf::DeltaArgs &);
extern template void launch_delta_step<_Float16>(okf_ctx *, const okf::DeltaArgs &);
extern template void launch_delta_step<__bf16>(okf_ctx *, const okf::DeltaArgs &);
extern template void launch_delta_chunks<float>(okf_ctx *, const okf::ScanArgs &);
extern template void launch_delta_chunks<_Float16>(okf_ctx *, const okf::ScanArgs &);
extern template void launch_delta_chunks<__bf16>(okf_ctx *, const okf::ScanArgs &);
#else
template void launch_delta_step<OKF_DELTA_TYPE>(okf_ctx *, const okf::DeltaArgs &);
template void launch_delta_chunks<OKF_DELTA_TYPE>(okf_ctx *, const okf::ScanArgs &);
#endif

}  // namespace okf_impl
