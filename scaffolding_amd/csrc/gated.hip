// gated.hip — the elementwise parts of a gated feed-forward layer over its two
// projections pre [M, 2 F] (gate, then up):
//
//   forward   y = act(gate) up                       (fp32, whose products have
//                                                     no fused epilogue)
//   backward  dgate = g up act'(gate), dup = g act(gate), as one [M, 2 F]
//
// One read of each operand, one write: bound by HBM.  A thread takes eight
// columns of a row, in 16-byte pieces at any alignment.
#include "rowio.hpp"
#include "sf_internal.hpp"

namespace sf {

template <typename T, int ACT, bool BACK>
__global__ __launch_bounds__(256) void gate_kernel(const void* g, const void* pre, void* out, int64_t M, int F) {
  const int per = (F + 7) / 8;  // pieces of a row
  const int64_t total = M * per;
  for (int64_t w = (int64_t)blockIdx.x * 256 + threadIdx.x; w < total; w += (int64_t)gridDim.x * 256) {
    int64_t m;
    if (total <= UINT32_MAX) m = (uint32_t)w / (uint32_t)per;
    else m = w / per;
    const int f = (int)(w - m * per) * 8, left = F - f < 8 ? F - f : 8;
    float gate[8], up[8];
    load_cols<T>(pre, m * 2 * F + f, left, gate);
    load_cols<T>(pre, m * 2 * F + F + f, left, up);
    if constexpr (BACK) {
      float d[8];
      load_cols<T>(g, m * F + f, left, d);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = gate[e];
        gate[e] = ACT == ACT_NONE ? d[e] * up[e] : d[e] * up[e] * act_slope<ACT>(v);
        up[e] = d[e] * act_t<ACT>(v);
      }
      store_cols<T>(out, m * 2 * F + f, left, gate);
      store_cols<T>(out, m * 2 * F + F + f, left, up);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) gate[e] = act_t<ACT>(gate[e]) * up[e];
      store_cols<T>(out, m * F + f, left, gate);
    }
  }
}

template <typename T>
static int launch_gate_t(int act, bool back, const void* g, const void* pre, void* out, int64_t M, int64_t F,
                         hipStream_t st) {
  int64_t nb = (M * ((F + 7) / 8) + 255) / 256;
  if (nb > (1 << 20)) nb = 1 << 20;
  const dim3 grid(static_cast<unsigned>(nb)), block(256);
  const int f = static_cast<int>(F);
#define SF_GATE(A)                                                                                    \
  do {                                                                                                \
    if (back) hipLaunchKernelGGL((gate_kernel<T, A, true>), grid, block, 0, st, g, pre, out, M, f);   \
    else hipLaunchKernelGGL((gate_kernel<T, A, false>), grid, block, 0, st, g, pre, out, M, f);       \
  } while (0)
  if (act == ACT_SILU) SF_GATE(ACT_SILU);
  else if (act == ACT_GELU) SF_GATE(ACT_GELU);
  else SF_GATE(ACT_NONE);
#undef SF_GATE
  return check_launch("gate");
}

int launch_gate(int act, bool back, const void* g, const void* pre, void* out, int64_t M, int64_t F, sf_dtype dt,
                hipStream_t st) {
  switch (dt) {
    case SF_F16: return launch_gate_t<F16>(act, back, g, pre, out, M, F, st);
    case SF_BF16: return launch_gate_t<BF16>(act, back, g, pre, out, M, F, st);
    default: return launch_gate_t<float>(act, back, g, pre, out, M, F, st);
  }
}

}  // namespace sf
