// okf_delta_run.h -- the launches of the gated delta rule, one instance of each per type in
// okf_delta_<type>.hip, so that they compile in parallel.
#pragma once
#include "okf_impl.h"
#include "okf_delta.h"

namespace okf_impl {

template <class T, int RK = 1>
void launch_delta_step(okf_ctx *c, const okf::DeltaArgs &a) {
    if constexpr (RK < 16)
        if (a.k_dim != 16 * RK) return launch_delta_step<T, RK + 1>(c, a);
    const uint64_t waves = (uint64_t)a.s.count * a.v_heads * (a.v_dim / 16);
    hipLaunchKernelGGL((okf::delta_step_kernel<T, RK>), dim3((uint32_t)((waves + 3) / 4)), dim3(okf::DS_NT), 0, c->stream, a);
}

#ifndef OKF_DELTA_TYPE
extern template void launch_delta_step<float>(okf_ctx *, const okf::DeltaArgs &);
extern template void launch_delta_step<_Float16>(okf_ctx *, const okf::DeltaArgs &);
extern template void launch_delta_step<__bf16>(okf_ctx *, const okf::DeltaArgs &);
#else
template void launch_delta_step<OKF_DELTA_TYPE>(okf_ctx *, const okf::DeltaArgs &);
#endif

}  // namespace okf_impl
