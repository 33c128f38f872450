// grouped_bf16.hip — grouped products for bf16 operands.
#include "grouped_inst.hpp"

namespace sf {
int launch_grouped_rows_bf16(bool b_kmajor, int cfg, const GroupedRows& p, unsigned gx, hipStream_t st) {
  return b_kmajor ? launch_grouped_rows_t<BF16, true>(cfg, p, gx, st) : launch_grouped_rows_t<BF16, false>(cfg, p, gx, st);
}
int launch_grouped_sums_bf16(int cfg, const GroupedSums& p, unsigned gx, unsigned gy, hipStream_t st) {
  return launch_grouped_sums_t<BF16>(cfg, p, gx, gy, st);
}
}  // namespace sf
