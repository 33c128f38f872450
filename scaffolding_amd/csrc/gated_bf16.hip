// gated_bf16.hip — gated feed-forward products of bf16 operands.
#include "gated_inst.hpp"

namespace sf {

int launch_gated_bf16(int cfg, const GatedParams& p, unsigned gx, hipStream_t st) {
  return launch_gated_t<BF16>(cfg, p, gx, st);
}

}  // namespace sf
