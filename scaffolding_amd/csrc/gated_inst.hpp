// gated_inst.hpp — instantiations and launch table of the gated feed-forward
// products for one input type (included by gated_bf16.hip and gated_f16.hip).
#pragma once

#include "gemm16mid.hpp"
#include "gemm16nt_pp.hpp"
#include "sf_internal.hpp"
#include "skinny16.hpp"

namespace sf {

template <typename T>
static int launch_gated_t(int cfg, const GatedParams& p, unsigned gx, hipStream_t st) {
  const dim3 g(gx);
  switch (cfg) {
    case TILE_NT_BIG:
      if (p.K % 128 != 0) return fail(SF_ERR_INVALID_ARG, "the gated 256x256 kernel needs K %% 128 == 0");
      if (p.persist > 0) {
        if (p.persist % kNumXcd != 0) return fail(SF_ERR_INVALID_ARG, "the gated persistent kernel needs a grid %% 8");
        hipLaunchKernelGGL((gemm16nt_pp_kernel<T, T, 2, true, true, true, false, GatedParams>), g, dim3(512), 0, st, p);
      } else {
        hipLaunchKernelGGL((gemm16nt_pp_kernel<T, T, 2, true, true, false, false, GatedParams>), g, dim3(512), 0, st, p);
      }
      break;
    case TILE_MID_128:
      hipLaunchKernelGGL((gemm16mid_kernel<T, T, 128, 128, 2, 4, 2, true, true, true, 4, GatedParams>), g, dim3(512), 0,
                         st, p);
      break;
    case TILE_MID_64:
      hipLaunchKernelGGL((gemm16mid_kernel<T, T, 64, 64, 2, 2, 3, true, true, true, 3, GatedParams>), g, dim3(256), 0,
                         st, p);
      break;
    case TILE_MID_32:
      hipLaunchKernelGGL((gemm16mid_kernel<T, T, 32, 64, 2, 2, 4, true, true, true, 3, GatedParams>), g, dim3(256), 0,
                         st, p);
      break;
    case TILE_RAG_128:
      hipLaunchKernelGGL((gemm16mid_kernel<T, T, 128, 128, 2, 4, 2, true, true, false, 4, GatedParams>), g, dim3(512),
                         0, st, p);
      break;
    case TILE_RAG_64:
      hipLaunchKernelGGL((gemm16mid_kernel<T, T, 64, 64, 2, 2, 2, true, true, false, 4, GatedParams>), g, dim3(256), 0,
                         st, p);
      break;
    case TILE_SKINNY:
      hipLaunchKernelGGL((skinny16_kernel<T, T, 4, 2, 8, GatedParams>), g, dim3(256), 0, st, p);
      break;
    default:
      return fail(SF_ERR_INVALID_ARG, "tile config %d has no gated variant", cfg);
  }
  return check_launch("gated product");
}

}  // namespace sf
