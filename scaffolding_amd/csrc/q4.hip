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
// where the result's are up to 15 |x|, in fp32: a few of its steps.  The order
// (0, 4, 1, 5, 2, 6, 3, 7) of the eight weights of a dword is met by giving x
// the same order (v_perm).
//
// k order.  v_mfma_f32_16x16x32 takes 8 consecutive k from each of four lane
// groups.  Loaded as it lies, lane group h's 16 bytes are k = 32 h .. 32 h + 31
// of a block of 128, and dword d of all groups covers k = 32 h + 8 d + 0..7:
// a sum over the whole block, right for G % 128 == 0.  For G = 32 and 64 a
// 4 x 4 transpose of dwords between the lane groups (four lane swaps) first
// makes dword d cover k = 32 d .. 32 d + 31.
//
// A workgroup of NW waves takes 16 NB weight rows and up to 16 rows of x (more
// rows read the weight again, from the caches); the waves take the blocks of
// 128 k in turn, and their sums are joined through LDS in wave order.
//
// What bounds it.  With few rows the weight's bytes come in at 4.0 TB/s (28672
// x 8192, past the 256 MB cache: a copy that only loads the weight reaches
// 5.2); small weights run at the launch and one memory latency (11008 x 4096,
// 1 row: 7.8 us, of them 3.4 the launch).  With more rows it is the unpacking's
// VALU work.
#include "gemm16nt_pp.hpp"
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
  int sg;  // scale rows of a tile that are in LDS at a time (a multiple of 4, or all)
};

constexpr int kQ4ScaleBytes = 32768;  // most LDS for the scales of a tile

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
// `mask` and `exp` are Q4Bits' constants in registers, which one v_and_or_b32
// takes (as literals they would need two instructions).
template <typename T>
__device__ __forceinline__ u32x4 q4_unpack(uint32_t w, uint32_t mask, uint32_t exp) {
  typedef Q4Bits<T> B;
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int sh = B::kShift - 4 * i;
    const uint32_t t = sh >= 0 ? w << (sh & 31) : w >> (-sh & 31);
    r[i] = (t & mask) | exp;
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
template <typename T, int NB, int NW, int GB, bool ZEROS, bool GROUPED>
__global__ __launch_bounds__(NW * 64) void q4_kernel(Q4Params p) {
  constexpr int BM = 16, BN = 16 * NB;
  constexpr int XP = 272;                        // bytes of a staged x row of 128 k: 16 rows on 16 bank groups
  constexpr int XB = NW * 16 * XP;               // staged x, one area per wave
  constexpr int PB = NW * NB * 1024;             // the waves' partial sums
  __shared__ __attribute__((aligned(16))) uint8_t area[XB > PB ? XB : PB];
  extern __shared__ __attribute__((aligned(16))) uint8_t dyn[];  // scales, then zero points
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
  const int n0 = tn * BN;
  const int KG = K / p.G;  // scale rows
  const uint8_t* __restrict__ Q = p.q + e * (int64_t)N * (K / 2);
  const uint16_t* __restrict__ S = p.s + e * (int64_t)N * KG;
  const uint8_t* __restrict__ Z = ZEROS ? p.z + e * (int64_t)N * KG : nullptr;
  const uint16_t* __restrict__ X = p.x + (int64_t)row0 * K;

  f32x4 sum[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) sum[i] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int nblk = none ? 0 : (K + 127) / 128;
  const int gstep = GB == 1 ? p.G / 128 : 1;  // blocks per scale group
  uint32_t mask = Q4Bits<T>::kMask, exp = Q4Bits<T>::kExp;
  asm("" : "+v"(mask));
  asm("" : "+v"(exp));
  mask = __builtin_amdgcn_readfirstlane(mask);
  const u32x4 ones = {Q4Bits<T>::kOnes, Q4Bits<T>::kOnes, Q4Bits<T>::kOnes, Q4Bits<T>::kOnes};

  // The tile's scales and zero points go through LDS as [scale row][column], as
  // many scale rows at a time as the launch gives room for (all of them but for
  // very long K): read per block they would take as many load instructions as
  // the weight, with 32 useful bytes each (28672 x 8192, 4 rows: 34 us against
  // 29).
  uint16_t* const sS = reinterpret_cast<uint16_t*>(dyn);
  uint8_t* const sZ = dyn + p.sg * BN * 2;
  const bool vec = (N & 3) == 0 && (reinterpret_cast<uintptr_t>(p.s) & 7) == 0 &&
                   (!ZEROS || (reinterpret_cast<uintptr_t>(p.z) & 3) == 0);
  auto stage_scales = [&](int kg0) {
    const int cnt = KG - kg0 < p.sg ? KG - kg0 : p.sg;
    for (int c = threadIdx.x; c < cnt * (BN / 4); c += NW * 64) {
      const int kg = c / (BN / 4), n = c % (BN / 4) * 4;  // four columns, past N the last
      const int64_t at = (int64_t)(kg0 + kg) * N;
      u32x2 sc;
      uint32_t zp = 0;
      if (vec) {
        const int g = n0 + n < N ? n0 + n : N - 4;
        sc = *reinterpret_cast<const u32x2*>(S + at + g);
        if constexpr (ZEROS) zp = *reinterpret_cast<const uint32_t*>(Z + at + g);
      } else {
        uint32_t v[4], z[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int g = n0 + n + q < N ? n0 + n + q : N - 1;
          v[q] = S[at + g];
          z[q] = ZEROS ? Z[at + g] : 0;
        }
        sc = u32x2{v[0] | v[1] << 16, v[2] | v[3] << 16};
        if constexpr (ZEROS) zp = z[0] | z[1] << 8 | z[2] << 16 | z[3] << 24;
      }
      *reinterpret_cast<u32x2*>(sS + kg * BN + n) = sc;
      if constexpr (ZEROS) *reinterpret_cast<uint32_t*>(sZ + kg * BN + n) = zp;
    }
  };

  // Loads go through buffer resources whose ranges are this tile's weight rows
  // and x rows: lanes past either read zeros without a branch (a weight row
  // past N only reaches outputs that are not stored).  The range check leaves
  // out the scalar offset, which moves along k within a row.
  const int tile_rows = N - n0 < BN ? N - n0 : BN;
  const __amdgpu_buffer_rsrc_t rq = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(Q + (int64_t)n0 * (K / 2)), (short)0, none ? 0 : tile_rows * (K / 2), 0x00020000);
  const __amdgpu_buffer_rsrc_t rx =
      __builtin_amdgcn_make_buffer_rsrc((void*)X, (short)0, none ? 0 : rows * K * 2, 0x00020000);
  constexpr uint32_t OOB = 0x80000000u;  // past every range
  uint32_t vq[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) vq[i] = (uint32_t)(16 * i + r16) * (uint32_t)(K / 2) + 16u * h;
  // x is loaded 16 bytes a lane, four rows of 128 k at a time, and put into MFMA
  // order through the wave's LDS area: up to four rows take one load
  // instruction a block (QX = 1), which is what a launch with few rows is bound
  // by next to the weight's own (11008 x 4096, 1 row: 9.0 us with four, 7.8).
  const uint32_t vx = (uint32_t)h * (uint32_t)K * 2u + 16u * r16;
  uint8_t* const xw = area + wave * 16 * XP;

  auto run = [&](auto qx_c) {
    constexpr int QX = decltype(qx_c)::value;
    u32x4 w[NB], xs[4];
    auto load = [&](int blk, int last) {
      const int k0 = blk * 128;
      const bool gone = blk >= last;             // uniform
      const bool tail = GB > 1 && k0 + 128 > K;  // uniform: a last block of 32, 64 or 96 k
      const int ks = gone ? 0 : k0;
#pragma unroll
      for (int d = 0; d < QX; ++d) {
        const uint32_t o = gone || (tail && k0 + 8 * r16 >= K) ? OOB : vx + (uint32_t)(4 * d * K) * 2u;
        xs[d] = __builtin_amdgcn_raw_buffer_load_b128(rx, o, ks * 2, 0);
      }
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const uint32_t o = gone || (tail && k0 + 32 * h >= K) ? OOB : vq[i];
        w[i] = __builtin_amdgcn_raw_buffer_load_b128(rq, o, ks / 2, 0);
      }
    };
    auto compute = [&](int blk, int kg0) {
      // row 4 d + h, chunk r16 (8 k)
#pragma unroll
      for (int d = 0; d < QX; ++d) *reinterpret_cast<u32x4*>(xw + (4 * d + h) * XP + r16 * 16) = q4_order(xs[d]);
      wave_lds_sync();
      // rows past the last: any staged bytes (their outputs are not stored)
      const int m = QX == 4 ? r16 : r16 & 3;
      // the k of lane group h in dword d: 32 h + 8 d, or 32 d + 8 h
#pragma unroll
      for (int d = 0; d < 4; ++d)
        xs[d] = *reinterpret_cast<const u32x4*>(xw + m * XP + (GB == 1 ? 4 * h + d : 4 * d + h) * 16);
      wave_lds_sync();
      if constexpr (GB > 1)
#pragma unroll
        for (int i = 0; i < NB; ++i) w[i] = lane_groups_transpose(w[i]);
#pragma unroll
      for (int gi = 0; gi < GB; ++gi) {
        constexpr int DG = 4 / GB;  // dwords per scale group
        const int kg = GB == 1 ? blk / gstep : blk * GB + gi;
        if (GB > 1 && kg >= KG) break;  // past K
        f32x4 xsum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = gi * DG; d < gi * DG + DG; ++d) xsum = Mfma16<T>::run(ones, xs[d], xsum);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          const u32x2 sc = *reinterpret_cast<const u32x2*>(sS + (kg - kg0) * BN + 16 * i + 4 * h);
          uint32_t zp = 0;
          if constexpr (ZEROS) zp = *reinterpret_cast<const uint32_t*>(sZ + (kg - kg0) * BN + 16 * i + 4 * h);
          f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int d = gi * DG; d < gi * DG + DG; ++d)
            acc = Mfma16<T>::run(q4_unpack<T>(w[i][d], mask, exp), xs[d], acc);
          // this lane's outputs are four columns of x row r16
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float s = Elem<T>::to_f32(static_cast<uint16_t>(sc[c >> 1] >> ((c & 1) * 16)));
            const float off = ZEROS ? 16.0f + (float)((zp >> (8 * c)) & 255u) : 24.0f;
            sum[i][c] += s * __builtin_fmaf(-off, xsum[c], acc[c]);
          }
        }
      }
    };
    // blocks whose scale rows are staged together
    const int seg = GB == 1 ? p.sg * gstep : (p.sg + GB - 1) / GB;
    for (int s0 = 0; s0 < nblk; s0 += seg) {
      const int last = s0 + seg < nblk ? s0 + seg : nblk;
      const int kg0 = GB == 1 ? s0 / gstep : s0 * GB;
      int b0 = s0 + wave;
      load(b0, last);  // in flight while the scales are staged
      if (s0 > 0) __syncthreads();
      stage_scales(kg0);
      __syncthreads();
      while (b0 < last) {
        compute(b0, kg0);
        b0 += NW;
        if (b0 < last) load(b0, last);
      }
    }
  };
  if (rows <= 4)
    run(std::integral_constant<int, 1>{});
  else
    run(std::integral_constant<int, 4>{});

  // The waves' sums through LDS, column block i finished by wave i % NW.
  const bool has_bias = epi_has_bias(epi);
  const uint16_t* bias = has_bias ? static_cast<const uint16_t*>(p.bias) + e * N : nullptr;
  const bool yvec = (N & 3) == 0 && (reinterpret_cast<uintptr_t>(p.y) & 7) == 0;
  f32x4* const part = reinterpret_cast<f32x4*>(area);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NB; ++i) part[(wave * NB + i) * 64 + lane] = sum[i];
  __syncthreads();
  with_act(epi_act(epi), [&](auto act_c) {
    constexpr int ACT = decltype(act_c)::value;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      if (i % NW != wave) continue;
      f32x4 v = part[i * 64 + lane];
#pragma unroll
      for (int q = 1; q < NW; ++q) v += part[(q * NB + i) * 64 + lane];
      const int n = n0 + 16 * i + 4 * h;
      if (r16 >= rows || n >= N) continue;
      float o[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        o[c] = v[c];
        if (has_bias && n + c < N) o[c] += Elem<T>::to_f32(bias[n + c]);
        o[c] = act_t<ACT>(o[c]);
      }
      uint16_t* y = p.y + (int64_t)(row0 + r16) * N + n;
      if (yvec) {
        *reinterpret_cast<u32x2*>(y) = u32x2{pack2<T>(o[0], o[1]), pack2<T>(o[2], o[3])};
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (n + c < N) y[c] = Elem<T>::from_f32(o[c]);
      }
    }
  });
}

template <typename T, int NB, int NW, int GB>
static void launch_q4_gz(const Q4Params& p, const dim3& g, unsigned lds, hipStream_t st) {
  if (p.offsets != nullptr) {
    if (p.z != nullptr) hipLaunchKernelGGL((q4_kernel<T, NB, NW, GB, true, true>), g, dim3(NW * 64), lds, st, p);
    else hipLaunchKernelGGL((q4_kernel<T, NB, NW, GB, false, true>), g, dim3(NW * 64), lds, st, p);
  } else {
    if (p.z != nullptr) hipLaunchKernelGGL((q4_kernel<T, NB, NW, GB, true, false>), g, dim3(NW * 64), lds, st, p);
    else hipLaunchKernelGGL((q4_kernel<T, NB, NW, GB, false, false>), g, dim3(NW * 64), lds, st, p);
  }
}

// Scale rows that a tile of `columns` holds in LDS at a time.
static int q4_staged(int columns, int64_t scale_rows, bool zeros) {
  const int fit = kQ4ScaleBytes / (columns * (zeros ? 3 : 2)) / 4 * 4;
  return scale_rows >= fit ? fit : (scale_rows > 1 ? static_cast<int>(scale_rows) : 1);
}

template <typename T, int NB, int NW>
static int launch_q4_g(Q4Params p, hipStream_t st) {
  p.tiles_n = (p.N + 16 * NB - 1) / (16 * NB);
  int64_t gx = p.tiles_n, gy = 1;
  if (p.offsets != nullptr) gx *= grouped_max_tiles(p.rows, p.groups, 16);
  else gy = (p.rows + 15) / 16;
  if (gx > (int64_t(1) << 22) || gy > 65535) return fail(SF_ERR_UNSUPPORTED, "sf_linear_q4: too many tiles");
  p.sg = q4_staged(16 * NB, p.K / p.G, p.z != nullptr);
  const unsigned lds = static_cast<unsigned>((p.sg + 3) / 4 * 4 * 16 * NB * (p.z != nullptr ? 3 : 2));
  const dim3 g(static_cast<unsigned>(gx), static_cast<unsigned>(gy));
  if (p.G % 128 == 0) launch_q4_gz<T, NB, NW, 1>(p, g, lds, st);
  else if (p.G == 64) launch_q4_gz<T, NB, NW, 2>(p, g, lds, st);
  else launch_q4_gz<T, NB, NW, 4>(p, g, lds, st);
  return check_launch("4-bit linear");
}

// Variants by how many tiles of 16 rows and 32 columns there are to share out
// (rows per weight: their mean where the sizes are on the device), and 64
// columns a tile once the rows of a weight fill more than two.  Measured in us,
// bf16, groups of 128 (28672 x 8192 x 4 rows, 11008 x 4096 x 1, 4096 x 11008 x
// 1, 4096 x 4096 x 1, 8 experts 11008 x 4096 x 16 rows, 11008 x 4096 x 32, x
// 64, x 256, 4096 x 11008 x 48, x 128):
//   16 columns, 8 waves     33.1   7.7   8.6  4.1  52.0  15.5  26.9
//   16 columns, 16 waves    33.5   8.9   7.3  4.4  79.6  17.7  30.0
//   32 columns, 4 waves     29.1   8.1  15.0  6.8  37.0  12.0  20.3
//   32 columns, 8 waves     29.7   7.8  10.4  5.6  40.6  12.2  20.8  74.5  24.9  45.7
//   64 columns, 4 waves     30.0   9.6  20.2  9.0  38.8  13.5  19.1  60.7  38.9  49.3
//   64 columns, 8 waves     29.5   8.1  14.8  7.6  39.6  13.5  19.3  65.8  26.1  39.2
// (32 and 64 rows a tile, the weight unpacked once for them, were slower at
// every size: 11008 x 4096 x 64 23.9 us at best, x 256 62.5.)
Q4Variant q4_variant(int64_t rows, int64_t groups, bool grouped, int64_t N, int64_t K, int64_t G, bool zeros) {
  const int64_t some = groups < rows ? groups : rows;
  const int64_t reached = !grouped || some < 1 ? 1 : some;  // no groups: all rows are set to 0
  const int64_t per = rows / reached, blocks = reached * ((per + 15) / 16);
  const int64_t cus = cu_count_current(), tiles = blocks * ((N + 31) / 32);
  Q4Variant v;
  if (per > 32 && 2 * blocks * ((N + 63) / 64) >= 3 * cus) v = {64, K >= 8192 ? 8 : 4, 1};
  else if (tiles >= cus) v = {32, tiles >= 2 * cus ? 4 : 8, 1};
  else v = {16, K >= 8192 ? 16 : 8, 1};
  // as q4_kernel counts them: segments of whole blocks of 128 k
  const int64_t staged = q4_staged(v.columns, K / G, zeros), per_block = G < 128 ? 128 / G : 1;
  const int64_t seg = G < 128 ? (staged + per_block - 1) / per_block : staged * (G / 128);
  v.segments = static_cast<int>(((K + 127) / 128 + seg - 1) / seg);
  return v;
}

template <typename T>
static int launch_q4_t(const Q4Params& p, hipStream_t st) {
  const Q4Variant v = q4_variant(p.rows, p.groups, p.offsets != nullptr, p.N, p.K, p.G, p.z != nullptr);
  if (v.columns == 64) return v.waves == 8 ? launch_q4_g<T, 4, 8>(p, st) : launch_q4_g<T, 4, 4>(p, st);
  if (v.columns == 32) return v.waves == 8 ? launch_q4_g<T, 2, 8>(p, st) : launch_q4_g<T, 2, 4>(p, st);
  return v.waves == 16 ? launch_q4_g<T, 1, 16>(p, st) : launch_q4_g<T, 1, 8>(p, st);
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
  p.sg = 0;
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
