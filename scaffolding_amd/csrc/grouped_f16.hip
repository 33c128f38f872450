// grouped_f16.hip — grouped products for f16 operands.
#include "grouped_inst.hpp"

namespace sf {
int launch_grouped_rows_f16(bool b_kmajor, int cfg, const GroupedRows& p, unsigned gx, hipStream_t st) {
  return b_kmajor ? launch_grouped_rows_t<F16, true>(cfg, p, gx, st) : launch_grouped_rows_t<F16, false>(cfg, p, gx, st);
}
int launch_grouped_sums_f16(int cfg, const GroupedSums& p, unsigned gx, unsigned gy, hipStream_t st) {
  return launch_grouped_sums_t<F16>(cfg, p, gx, gy, st);
}
}  // namespace sf
