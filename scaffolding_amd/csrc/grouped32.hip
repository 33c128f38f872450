// grouped32.hip — fp32 grouped products: the direct-to-LDS tiles and, for few
// rows in groups, the small blocks; register-staged tiles past the direct
// loads' 2 GiB.
#include "gemm32.hpp"
#include "gemm32dma.hpp"
#include "gemm32small.hpp"
#include "sf_internal.hpp"

namespace sf {

template <bool KM>
static int launch_rows_t(int cfg, const GroupedRows& p, const dim3& g, hipStream_t st) {
  switch (cfg) {
    case TILE32_SMALL2:
      hipLaunchKernelGGL((gemm32small_kernel<2, KM, 8, GroupedRows>), g, dim3(512), 0, st, p);
      break;
    case TILE32_SMALL2_ANY:
      hipLaunchKernelGGL((gemm32small_kernel<2, KM, 8, GroupedRows, true>), g, dim3(512), 0, st, p);
      break;
    case TILE32_DMA:
      hipLaunchKernelGGL((gemm32dma_kernel<64, 64, true, KM, 2, 2, 4, true, GroupedRows>), g, dim3(512), 0, st, p);
      break;
    case TILE32_RAG:
      hipLaunchKernelGGL((gemm32dma_kernel<64, 64, true, KM, 2, 2, 1, true, GroupedRows>), g, dim3(512), 0, st, p);
      break;
    case TILE_GENERIC:
      hipLaunchKernelGGL((gemm32_kernel<64, 64, 2, 2, KM, false, true, GroupedRows>), g, dim3(256), 0, st, p);
      break;
    default:
      return fail(SF_ERR_INVALID_ARG, "tile config %d has no grouped fp32 variant", cfg);
  }
  return check_launch("grouped fp32 product");
}

int launch_grouped_rows_f32(bool b_kmajor, int cfg, const GroupedRows& p, unsigned gx, hipStream_t st) {
  return b_kmajor ? launch_rows_t<true>(cfg, p, dim3(gx), st) : launch_rows_t<false>(cfg, p, dim3(gx), st);
}

int launch_grouped_sums_f32(int cfg, const GroupedSums& p, unsigned gx, unsigned gy, hipStream_t st) {
  const dim3 g(gx, gy);
  switch (cfg) {
    case TILE32_DMA:
      hipLaunchKernelGGL((gemm32dma_kernel<64, 64, false, false, 2, 2, 4, true, GroupedSums>), g, dim3(512), 0, st, p);
      break;
    case TILE32_RAG:
      hipLaunchKernelGGL((gemm32dma_kernel<64, 64, false, false, 2, 2, 1, true, GroupedSums>), g, dim3(512), 0, st, p);
      break;
    case TILE_GENERIC:
      hipLaunchKernelGGL((gemm32_kernel<64, 64, 2, 2, false, false, false, GroupedSums>), g, dim3(256), 0, st, p);
      break;
    default:
      return fail(SF_ERR_INVALID_ARG, "tile config %d has no grouped fp32 variant", cfg);
  }
  return check_launch("grouped fp32 sums");
}

}  // namespace sf
