// gated_f16.hip — gated feed-forward products of f16 operands.
#include "gated_inst.hpp"

namespace sf {

int launch_gated_f16(int cfg, const GatedParams& p, unsigned gx, hipStream_t st) {
  return launch_gated_t<F16>(cfg, p, gx, st);
}

}  // namespace sf
