// gated.hpp — a gated feed-forward layer's up side on the tiled 16-bit
// kernels: with W [2 F, K] holding the gate's rows, then the up-projection's,
//
//   y[m, f] = act(x[m] . W[f] + b[f]) * (x[m] . W[F + f] + b[F + f])
//
// The kernels' B tile is BN lines of W; here half of them are gate rows and
// half the up rows of the same columns f, laid out so that a wave's own WN
// lines are WN / 2 of each: its accumulator blocks i and i + FN / 2 then hold
// gate and up of the same outputs in the same lane, and the product needs no
// exchange.  A tile gives BN / 2 columns of y.
//
// `pre` (or NULL) takes the two projections themselves, [M, 2 F] rounded to
// the operands' type, for the backward pass; y is formed from the unrounded
// ones.
#pragma once

#include "gemm16.hpp"
#include "rowio.hpp"

namespace sf {

// M, K, A, B, C (y, ldc = F), bias [2 F] and epi as GemmParams says; N = 2 F.
//
// A launch may leave the last, part round of 256 x 256 tiles to a second one:
// the first runs tiles 0 .. head - 1, the second, of 128 x 128 tiles with big_n >
// 0, the quarters of the tiles from `head` on of big_m x big_n.
struct GatedParams : GemmParams {
  void* pre;
  int F;
  int head, big_m, big_n;
};

// The product's columns (0: not a gated launch).
__device__ __forceinline__ int gated_columns(const GemmParams&) { return 0; }
__device__ __forceinline__ int gated_columns(const GatedParams& p) { return p.F; }

// The row of W on line r of a tile whose waves own WN lines and whose first
// column is f0; `in` false where its column is past F (row: of column F - 1).
template <int WN>
__device__ __forceinline__ int gated_row(int r, int f0, int F, bool& in) {
  constexpr int HW = WN / 2;
  int f = f0 + (r / WN) * HW + (r % HW);
  in = f < F;
  f = in ? f : F - 1;
  return f + ((r % WN) / HW) * F;
}

// Stores a wave's FM x 16 rows (from row m0) of WN / 2 columns (from f0): bias,
// activation and product in registers, then 16 rows at a time through `stage`
// (gated_stage_bytes<WN> of the wave's own) in 16-byte pieces.
template <int WN>
constexpr int gated_pitch() { return 3 * WN + 16; }  // gate | up | product, WN / 2 each
template <int WN>
constexpr int gated_stage_bytes() { return 16 * gated_pitch<WN>(); }

template <typename T, bool NT>
__device__ __forceinline__ void gated_put(uint16_t* row, int f, int F, bool vec, u32x4 v) {
  if (f + 8 <= F) {
    if (NT && vec) __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(row + f));
    else reinterpret_cast<H8u*>(row + f)->v = v;
  } else {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (f + e < F) row[f + e] = static_cast<uint16_t>(v[e >> 1] >> ((e & 1) * 16));
  }
}

template <typename T, int FM, int FN, int WN, bool NT>
__device__ __forceinline__ void gated_store(const GatedParams& p, const f32x4 (&acc)[FN][FM], int m0, int f0, int M,
                                            int lane, uint8_t* stage) {
  constexpr int FH = FN / 2, HW = WN / 2, PITCH = gated_pitch<WN>();
  static_assert(FN % 2 == 0 && WN == FN * 16, "half of a wave's lines are gate rows");
  const int F = p.F;
  const bool has_bias = epi_has_bias(p.epi);
  float bg[FH][4], bu[FH][4];
#pragma unroll
  for (int i = 0; i < FH; ++i) {
#pragma unroll
    for (int q = 0; q < 4; ++q) bg[i][q] = bu[i][q] = 0.f;
    if (has_bias) {
      const int f = f0 + i * 16 + 4 * (lane >> 4);
      const uint16_t* b = static_cast<const uint16_t*>(p.bias);
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (f + q < F) {
          bg[i][q] = Elem<T>::to_f32(b[f + q]);
          bu[i][q] = Elem<T>::to_f32(b[F + f + q]);
        }
    }
  }
  uint16_t* C = static_cast<uint16_t*>(p.C);
  uint16_t* P = static_cast<uint16_t*>(p.pre);
  const bool vec = (F & 7) == 0 && ((reinterpret_cast<uintptr_t>(C) | reinterpret_cast<uintptr_t>(P)) & 15) == 0;
  constexpr int PIECES = HW / 8;  // 16-byte pieces of a row, per array
  with_act(epi_act(p.epi), [&](auto act_c) {
    constexpr int ACT = decltype(act_c)::value;
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      wave_lds_sync();
      uint8_t* row = stage + (lane & 15) * PITCH + 8 * (lane >> 4);
#pragma unroll
      for (int i = 0; i < FH; ++i) {
        float g[4], u[4], y[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          g[q] = acc[i][j][q] + bg[i][q];
          u[q] = acc[i + FH][j][q] + bu[i][q];
          y[q] = act_t<ACT>(g[q]) * u[q];
        }
        if (P != nullptr) {
          *reinterpret_cast<u32x2*>(row + i * 32) = u32x2{pack2<T>(g[0], g[1]), pack2<T>(g[2], g[3])};
          *reinterpret_cast<u32x2*>(row + 2 * HW + i * 32) = u32x2{pack2<T>(u[0], u[1]), pack2<T>(u[2], u[3])};
        }
        *reinterpret_cast<u32x2*>(row + 4 * HW + i * 32) = u32x2{pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3])};
      }
      wave_lds_sync();
      const int r = (lane / PIECES) & 15, c = lane % PIECES;
      const int m = m0 + j * 16 + r, f = f0 + c * 8;
      if (m < M && f < F && (PIECES == 4 || lane < 16 * PIECES)) {
        const uint8_t* at = stage + r * PITCH + c * 16;
        gated_put<T, NT>(C + (int64_t)m * F, f, F, vec, *reinterpret_cast<const u32x4*>(at + 4 * HW));
        if (P != nullptr) {
          uint16_t* pr = P + (int64_t)m * 2 * F;
          gated_put<T, NT>(pr, f, F, vec, *reinterpret_cast<const u32x4*>(at));
          gated_put<T, NT>(pr + F, f, F, vec, *reinterpret_cast<const u32x4*>(at + 2 * HW));
        }
      }
    }
  });
}

}  // namespace sf
