// grouped32.hip — fp32 grouped products on gemm32_kernel's register-staged
// tiles.
#include "gemm32.hpp"
#include "sf_internal.hpp"

namespace sf {

template <bool KM, bool AKM, typename P>
static int launch_grouped32_t(int cfg, const P& p, const dim3& g, hipStream_t st) {
  switch (cfg) {
    case TILE_128x128:
      hipLaunchKernelGGL((gemm32_kernel<128, 128, 2, 2, KM, true, AKM, P>), g, dim3(256), 0, st, p);
      break;
    case TILE_64x64:
      hipLaunchKernelGGL((gemm32_kernel<64, 64, 2, 2, KM, true, AKM, P>), g, dim3(256), 0, st, p);
      break;
    case TILE_GENERIC:
      hipLaunchKernelGGL((gemm32_kernel<64, 64, 2, 2, KM, false, AKM, P>), g, dim3(256), 0, st, p);
      break;
    default:
      return fail(SF_ERR_INVALID_ARG, "tile config %d has no grouped fp32 variant", cfg);
  }
  return check_launch("grouped fp32 product");
}

int launch_grouped_rows_f32(bool b_kmajor, int cfg, const GroupedRows& p, unsigned gx, hipStream_t st) {
  return b_kmajor ? launch_grouped32_t<true, true>(cfg, p, dim3(gx), st)
                  : launch_grouped32_t<false, true>(cfg, p, dim3(gx), st);
}
int launch_grouped_sums_f32(int cfg, const GroupedSums& p, unsigned gx, unsigned gy, hipStream_t st) {
  return launch_grouped32_t<false, false>(cfg, p, dim3(gx, gy), st);
}

}  // namespace sf
