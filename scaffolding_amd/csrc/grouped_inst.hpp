// grouped_inst.hpp — instantiations and launch table of the 16-bit grouped
// products for one input type (included by grouped_bf16.hip and
// grouped_f16.hip).
#pragma once

#include "gemm16mid.hpp"
#include "gemm16nt_pp.hpp"
#include "sf_internal.hpp"

namespace sf {

// KM: B K-contiguous (y = W x) or N-contiguous (dx = W^T g).
template <typename T, bool KM>
static int launch_grouped_rows_t(int cfg, const GroupedRows& p, unsigned gx, hipStream_t st) {
  const dim3 g(gx);
  switch (cfg) {
    case TILE_NT_BIG:
      if (p.K % 128 != 0) return fail(SF_ERR_INVALID_ARG, "the grouped 256x256 kernel needs K %% 128 == 0");
      hipLaunchKernelGGL((gemm16nt_pp_kernel<T, T, 2, true, KM, false, false, GroupedRows>), g, dim3(512), 0, st, p);
      break;
    case TILE_MID_128:
      hipLaunchKernelGGL((gemm16mid_kernel<T, T, 128, 128, 2, 4, 2, true, KM, true, 4, GroupedRows>), g, dim3(512), 0,
                         st, p);
      break;
    case TILE_MID_64:
      hipLaunchKernelGGL((gemm16mid_kernel<T, T, 64, 64, 2, 2, 3, true, KM, true, 3, GroupedRows>), g, dim3(256), 0, st,
                         p);
      break;
    case TILE_MID_32:
      if constexpr (KM) {
        hipLaunchKernelGGL((gemm16mid_kernel<T, T, 32, 64, 2, 2, 4, true, true, true, 3, GroupedRows>), g, dim3(256), 0,
                           st, p);
        break;
      }
      return fail(SF_ERR_UNSUPPORTED, "the 32x64 tile needs K-contiguous A and B");
    case TILE_RAG_128:
      hipLaunchKernelGGL((gemm16mid_kernel<T, T, 128, 128, 2, 4, 2, true, KM, false, 4, GroupedRows>), g, dim3(512), 0,
                         st, p);
      break;
    case TILE_RAG_64:
      hipLaunchKernelGGL((gemm16mid_kernel<T, T, 64, 64, 2, 2, 2, true, KM, false, 4, GroupedRows>), g, dim3(256), 0,
                         st, p);
      break;
    default:
      return fail(SF_ERR_INVALID_ARG, "tile config %d has no grouped variant", cfg);
  }
  return check_launch("grouped product");
}

template <typename T>
static int launch_grouped_sums_t(int cfg, const GroupedSums& p, unsigned gx, unsigned gy, hipStream_t st) {
  const dim3 g(gx, gy);
  switch (cfg) {
    case TILE_NT_BIG:
      hipLaunchKernelGGL((gemm16nt_pp_kernel<T, T, 2, false, false, false, false, GroupedSums>), g, dim3(512), 0, st, p);
      break;
    case TILE_MID_128:
      hipLaunchKernelGGL((gemm16mid_kernel<T, T, 128, 128, 2, 4, 2, false, false, true, 4, GroupedSums>), g, dim3(512),
                         0, st, p);
      break;
    case TILE_MID_64:
      hipLaunchKernelGGL((gemm16mid_kernel<T, T, 64, 64, 2, 2, 3, false, false, true, 3, GroupedSums>), g, dim3(256), 0,
                         st, p);
      break;
    case TILE_RAG_128:
      hipLaunchKernelGGL((gemm16mid_kernel<T, T, 128, 128, 2, 4, 2, false, false, false, 4, GroupedSums>), g, dim3(512),
                         0, st, p);
      break;
    case TILE_RAG_64:
      hipLaunchKernelGGL((gemm16mid_kernel<T, T, 64, 64, 2, 2, 2, false, false, false, 4, GroupedSums>), g, dim3(256),
                         0, st, p);
      break;
    default:
      return fail(SF_ERR_INVALID_ARG, "tile config %d has no grouped variant", cfg);
  }
  return check_launch("grouped sums");
}

}  // namespace sf
