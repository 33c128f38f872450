// q4.hip — a linear layer whose weight is held in 4 bits with group scales:
//
//   y[m, n] = act(sum_k x[m, k] (q[n, k] - z[k / G, n]) s[k / G, n] (+ b[n]))
//
// for 16-bit x, either one weight for all rows or one per group of rows
// (grouped.hpp).  Decoding with few rows is bound by reading the weight, a
// quarter of its 16-bit size; the arithmetic that unpacks it must stay below
// that.
//
// Unpacking.  A 16-byte load gives a lane 32 weights of one row.  For the
// pair (k, k + 4) of a dword, two nibbles 16 bits apart, a shift and one
// and-or put them into the mantissas of two 16-bit numbers whose exponent is
// that of 16:  0x4180 | q << 3 (bf16) or 0x4c00 | q << 6 (fp16) is 16 + q
// exactly, no conversion and no rounding.  The MFMA multiplies x by these
// integers with fp32 sums; per scale group
//   sum += s (acc - (16 + z) X),  X = the group's sum of x,
// in fp32 brings in the scale and takes the offset out.  X comes from one
// more MFMA with a matrix of ones (exact products, the same fp32 sums), shared
// by all row blocks of the weight.  The sums run over terms of up to 31 |x|
// where the result's are up to 15 |x|, in fp32: a few of its steps.  The order (0, 4, 1, 5, 2, 6, 3, 7) of the eight weights
// of a dword is met by giving x the same order (v_perm).
//
// k order.  v_mfma_f32_16x16x32 takes 8 consecutive k from each of four lane
// groups.  Loaded as it lies, lane group h's 16 bytes are k = 32 h .. 32 h + 31
// of a block of 128, and dword d of all groups covers k = 32 h + 8 d + 0..7:
// a sum over the whole block, right for G % 128 == 0.  For G = 32 and 64 a
// 4 x 4 transpose of dwords between the lane groups (four lane swaps) first
// makes dword d cover k = 32 d .. 32 d + 31.
//
// A workgroup of NW waves takes 16 NB weight rows and up to 16 MB rows of x;
// the waves take the blocks of 128 k in turn, and their sums are joined
// through LDS in wave order.
#include "grouped.hpp"
#include "rowio.hpp"
#include "sf_internal.hpp"

namespace sf {

struct Q4Params {
  const uint16_t* x;
  const uint8_t* q;
  const uint16_t* s;
  const uint8_t* z;  // NULL: 8
  const void* bias;
  uint16_t* y;
  const int* offsets;  // NULL: one weight for all rows
  int groups, rows, N, K, G;
  int tiles_n;
  int epi;
};

template <typename T> struct Q4Bits;
template <> struct Q4Bits<BF16> {
  static constexpr uint32_t kExp = 0x41804180u, kMask = 0x00780078u, kOnes = 0x3f803f80u;
  static constexpr int kShift = 3;
};
template <> struct Q4Bits<F16> {
  static constexpr uint32_t kExp = 0x4c004c00u, kMask = 0x03c003c0u, kOnes = 0x3c003c00u;
  static constexpr int kShift = 6;
};

// The eight weights of a dword as 16 + q, in the order 0 4 1 5 2 6 3 7.
template <typename T>
__device__ __forceinline__ u32x4 q4_unpack(uint32_t w) {
  typedef Q4Bits<T> B;
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int sh = B::kShift - 4 * i;
    const uint32_t t = sh >= 0 ? w << (sh & 31) : w >> (-sh & 31);
    r[i] = (t & B::kMask) | B::kExp;
  }
  return r;
}
// Eight 16-bit x of consecutive k in that order.
__device__ __forceinline__ u32x4 q4_order(u32x4 v) {
  u32x4 r;
  r[0] = __builtin_amdgcn_perm(v[2], v[0], 0x05040100u);
  r[1] = __builtin_amdgcn_perm(v[2], v[0], 0x07060302u);
  r[2] = __builtin_amdgcn_perm(v[3], v[1], 0x05040100u);
  r[3] = __builtin_amdgcn_perm(v[3], v[1], 0x07060302u);
  return r;
}

// v[d] of lane group h becomes v[h] of lane group d (groups of 16 lanes).
__device__ __forceinline__ u32x4 lane_groups_transpose(u32x4 v) {
  typedef uint32_t u2 __attribute__((ext_vector_type(2)));
  const u2 a = __builtin_amdgcn_permlane32_swap(v[0], v[2], false, false);
  const u2 b = __builtin_amdgcn_permlane32_swap(v[1], v[3], false, false);
  const u2 c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  const u2 d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  return u32x4{c[0], c[1], d[0], d[1]};
}

// GB: scale groups per block of 128 k (1: G % 128 == 0; 2; 4).
template <typename T, int NB, int MB, int NW, int GB, bool ZEROS, bool GROUPED>
__global__ __launch_bounds__(NW * 64) void q4_kernel(Q4Params p) {
  constexpr int BM = 16 * MB;
  __shared__ f32x4 part[NW > 1 ? NW : 1][NB * MB][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, h = lane >> 4;
  const int K = p.K, N = p.N;
  int row0, rows, tn;
  int64_t e = 0;
  int epi = p.epi;
  bool none = false;  // rows of no group
  if constexpr (GROUPED) {
    GroupTile g;
    if (!group_find<BM>(p, g)) return;  // workgroup-uniform
    row0 = g.row;
    rows = g.rows;
    tn = g.tn;
    e = g.e;
    none = g.e == p.groups;
  } else {
    tn = blockIdx.x;
    row0 = blockIdx.y * BM;
    rows = p.rows - row0 < BM ? p.rows - row0 : BM;
  }
  if (none) epi = SF_EPI_NONE;
  const int n0 = tn * 16 * NB;
  const int KG = K / p.G;  // scale rows
  const uint8_t* __restrict__ Q = p.q + e * (int64_t)N * (K / 2);
  const uint16_t* __restrict__ S = p.s + e * (int64_t)N * KG;
  const uint8_t* __restrict__ Z = ZEROS ? p.z + e * (int64_t)N * KG : nullptr;
  const uint16_t* __restrict__ X = p.x + (int64_t)row0 * K;

  f32x4 sum[NB][MB];
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < MB; ++j) sum[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int nblk = none ? 0 : (K + 127) / 128;
  const int gstep = GB == 1 ? p.G / 128 : 1;  // blocks per scale group
  const u32x4 ones = {Q4Bits<T>::kOnes, Q4Bits<T>::kOnes, Q4Bits<T>::kOnes, Q4Bits<T>::kOnes};
  // this lane's weight rows and x rows; rows past the edge read the last one
  // (weights: their outputs are not stored) or zeros (x)
  int64_t qrow[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const int n = n0 + 16 * i + r16;
    qrow[i] = (int64_t)(n < N ? n : N - 1) * (K / 2);
  }
  for (int blk = wave; blk < nblk; blk += NW) {
    const int k0 = blk * 128;
    u32x4 w[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int k = k0 + 32 * h;
      w[i] = k < K ? *reinterpret_cast<const u32x4*>(Q + qrow[i] + k / 2) : u32x4{0u, 0u, 0u, 0u};
      if constexpr (GB > 1) w[i] = lane_groups_transpose(w[i]);
    }
    // the k of lane group h in dword d
    auto k_of = [&](int d) { return GB == 1 ? k0 + 32 * h + 8 * d : k0 + 32 * d + 8 * h; };
    u32x4 xs[MB][4];
#pragma unroll
    for (int j = 0; j < MB; ++j) {
      const int m = 16 * j + r16;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const int k = k_of(d);
        u32x4 v = {0u, 0u, 0u, 0u};
        if (m < rows && k < K) v = *reinterpret_cast<const u32x4*>(X + (int64_t)m * K + k);
        xs[j][d] = q4_order(v);
      }
    }
#pragma unroll
    for (int gi = 0; gi < GB; ++gi) {
      constexpr int DG = 4 / GB;  // dwords per scale group
      const int kg = GB == 1 ? blk / gstep : blk * GB + gi;
      if (GB > 1 && kg >= KG) break;
      f32x4 xsum[MB];
#pragma unroll
      for (int j = 0; j < MB; ++j) {
        xsum[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = gi * DG; d < gi * DG + DG; ++d) xsum[j] = Mfma16<T>::run(ones, xs[j][d], xsum[j]);
      }
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        f32x4 acc[MB];
#pragma unroll
        for (int j = 0; j < MB; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = gi * DG; d < gi * DG + DG; ++d) {
          const u32x4 wf = q4_unpack<T>(w[i][d]);
#pragma unroll
          for (int j = 0; j < MB; ++j) acc[j] = Mfma16<T>::run(wf, xs[j][d], acc[j]);
        }
        // this lane's outputs are n0 + 16 i + 4 h + 0..3 of x row r16
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int n = n0 + 16 * i + 4 * h + c;
          const int64_t at = (int64_t)kg * N + (n < N ? n : N - 1);
          const float sc = Elem<T>::to_f32(S[at]);
          const float off = ZEROS ? 16.0f + (float)Z[at] : 24.0f;
#pragma unroll
          for (int j = 0; j < MB; ++j) sum[i][j][c] += sc * __builtin_fmaf(-off, xsum[j][c], acc[j][c]);
        }
      }
    }
  }
  if constexpr (NW > 1) {
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int j = 0; j < MB; ++j) part[wave][i * MB + j][lane] = sum[i][j];
    __syncthreads();
  }
  // fragment f (of NB MB) is finished by wave f % NW
  const bool has_bias = epi_has_bias(epi);
  const uint16_t* bias = has_bias ? static_cast<const uint16_t*>(p.bias) + e * N : nullptr;
  with_act(epi_act(epi), [&](auto act_c) {
    constexpr int ACT = decltype(act_c)::value;
#pragma unroll
    for (int f = 0; f < NB * MB; ++f) {
      if (f % NW != wave) continue;
      const int i = f / MB, j = f % MB;
      f32x4 v = sum[i][j];
      if constexpr (NW > 1) {
        v = part[0][f][lane];
#pragma unroll
        for (int w = 1; w < NW; ++w) v += part[w][f][lane];
      }
      const int m = 16 * j + r16, n = n0 + 16 * i + 4 * h;
      if (m >= rows) continue;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (n + c >= N) continue;
        float o = v[c];
        if (has_bias) o += Elem<T>::to_f32(bias[n + c]);
        p.y[(int64_t)(row0 + m) * N + n + c] = Elem<T>::from_f32(act_t<ACT>(o));
      }
    }
  });
}

template <typename T, int NB, int MB, int NW, int GB>
static void launch_q4_gz(const Q4Params& p, const dim3& g, hipStream_t st) {
  if (p.offsets != nullptr) {
    if (p.z != nullptr) hipLaunchKernelGGL((q4_kernel<T, NB, MB, NW, GB, true, true>), g, dim3(NW * 64), 0, st, p);
    else hipLaunchKernelGGL((q4_kernel<T, NB, MB, NW, GB, false, true>), g, dim3(NW * 64), 0, st, p);
  } else {
    if (p.z != nullptr) hipLaunchKernelGGL((q4_kernel<T, NB, MB, NW, GB, true, false>), g, dim3(NW * 64), 0, st, p);
    else hipLaunchKernelGGL((q4_kernel<T, NB, MB, NW, GB, false, false>), g, dim3(NW * 64), 0, st, p);
  }
}

template <typename T, int NB, int MB, int NW>
static int launch_q4_g(Q4Params p, hipStream_t st) {
  p.tiles_n = (p.N + 16 * NB - 1) / (16 * NB);
  int64_t gx = p.tiles_n, gy = 1;
  if (p.offsets != nullptr) gx *= grouped_max_tiles(p.rows, p.groups, 16 * MB);
  else gy = (p.rows + 16 * MB - 1) / (16 * MB);
  if (gx > (int64_t(1) << 22) || gy > 65535) return fail(SF_ERR_UNSUPPORTED, "sf_linear_q4: too many tiles");
  const dim3 g(static_cast<unsigned>(gx), static_cast<unsigned>(gy));
  if (p.G % 128 == 0) launch_q4_gz<T, NB, MB, NW, 1>(p, g, st);
  else if (p.G == 64) launch_q4_gz<T, NB, MB, NW, 2>(p, g, st);
  else launch_q4_gz<T, NB, MB, NW, 4>(p, g, st);
  return check_launch("4-bit linear");
}

template <typename T>
static int launch_q4_t(const Q4Params& p, hipStream_t st) {
  const int per = p.offsets != nullptr ? (int)(p.rows / (p.groups < p.rows ? p.groups : p.rows)) : p.rows;
  if (per <= 16) return launch_q4_g<T, 2, 1, 4>(p, st);
  if (per <= 32) return launch_q4_g<T, 2, 2, 4>(p, st);
  return launch_q4_g<T, 2, 4, 4>(p, st);
}

int launch_q4(const void* x, const void* q, const void* s, const void* z, const void* bias, void* y,
              const int* offsets, int64_t groups, int64_t rows, int64_t N, int64_t K, int64_t G, sf_dtype dt,
              sf_epilogue epi, hipStream_t st) {
  Q4Params p;
  p.x = static_cast<const uint16_t*>(x);
  p.q = static_cast<const uint8_t*>(q);
  p.s = static_cast<const uint16_t*>(s);
  p.z = static_cast<const uint8_t*>(z);
  p.bias = bias;
  p.y = static_cast<uint16_t*>(y);
  p.offsets = offsets;
  p.groups = static_cast<int>(groups);
  p.rows = static_cast<int>(rows);
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.G = static_cast<int>(G);
  p.tiles_n = 0;
  p.epi = epi;
  return dt == SF_BF16 ? launch_q4_t<BF16>(p, st) : launch_q4_t<F16>(p, st);
}

// The weight in 16 bits, w = (q - z) s rounded once: for products with many
// rows, which read it so often that unpacking once is cheaper.  A thread takes
// 32 k of one row (a scale group or part of one).
template <typename T>
__global__ __launch_bounds__(256) void q4_expand_kernel(const uint8_t* __restrict__ q, const uint16_t* __restrict__ s,
                                                        const uint8_t* __restrict__ z, uint16_t* __restrict__ w,
                                                        int64_t total, int64_t N, int K, int G) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;  // 32 k each
  if (i >= total) return;
  const int per = K / 32;
  const int64_t row = i / per;  // e * N + n
  const int k = (int)(i - row * per) * 32;
  const int64_t e = row / N, n = row - e * N;
  const int64_t at = (e * (K / G) + k / G) * N + n;
  const float sc = Elem<T>::to_f32(s[at]);
  const float zero = z != nullptr ? (float)z[at] : 8.0f;
  const u32x4 v = *reinterpret_cast<const u32x4*>(q + row * (K / 2) + k / 2);
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    float o[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) o[c] = ((float)((v[d] >> (4 * c)) & 15u) - zero) * sc;
    store8u<T>(w, row * K + k + 8 * d, o);
  }
}

int launch_q4_expand(const void* q, const void* s, const void* z, void* w, int64_t groups, int64_t N, int64_t K,
                     int64_t G, sf_dtype dt, hipStream_t st) {
  const int64_t total = groups * N * (K / 32);
  const int64_t nb = (total + 255) / 256;
  if (nb > (int64_t(1) << 23)) return fail(SF_ERR_UNSUPPORTED, "sf_q4_expand: weight too large");
  const dim3 g(static_cast<unsigned>(nb));
  const uint8_t* qq = static_cast<const uint8_t*>(q);
  const uint8_t* zz = static_cast<const uint8_t*>(z);
  const uint16_t* ss = static_cast<const uint16_t*>(s);
  uint16_t* ww = static_cast<uint16_t*>(w);
  if (dt == SF_BF16)
    hipLaunchKernelGGL((q4_expand_kernel<BF16>), g, dim3(256), 0, st, qq, ss, zz, ww, total, N, (int)K, (int)G);
  else
    hipLaunchKernelGGL((q4_expand_kernel<F16>), g, dim3(256), 0, st, qq, ss, zz, ww, total, N, (int)K, (int)G);
  return check_launch("4-bit expansion");
}

}  // namespace sf
