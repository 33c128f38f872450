// gated.hip — the elementwise parts of a gated feed-forward layer over its two
// projections pre [M, 2 F] (gate, then up):
//
//   forward   y = act(gate) up                       (fp32 of many rows, whose
//                                                     products have no fused
//                                                     epilogue)
//   backward  dgate = g up act'(gate), dup = g act(gate), as one [M, 2 F], and
//             their sums over the rows, a bias's gradient
//
// One read of each operand, one write: bound by HBM.  A thread takes eight
// columns of a row, in 16-byte pieces at any alignment.
//
// And the fp32 layer for few rows, whole: gated_skinny32_kernel.
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

// The backward pass with the sums over the rows: block (strip, chunk) takes TC *
// 8 columns and p.rows rows, its 256 / TC thread rows every 256 / TC-th of them;
// each thread row leaves its sums (fp32, of the gradients ahead of their
// rounding) in a row of part [chunks * 256 / TC, 2 F].  The columns' threads
// stay with their columns, so the sums need no reading of what was written:
// 4096 rows, F 7680, bf16 in 73 us (315 MB, 4.3 TB/s) and 5 for the parts' sums,
// where the gate alone takes 63 and summing its result 25.
struct GateSums {
  const void *g, *pre;
  void *out, *db;
  float* part;
  int64_t M, rows;  // of a chunk
  int F, strips, lg;  // TC = 2^lg threads for the columns
  unsigned parts;
};

template <typename T, int ACT>
__global__ __launch_bounds__(256) void gate_sums_kernel(GateSums p) {
  const int tc = threadIdx.x & ((1 << p.lg) - 1), tr = threadIdx.x >> p.lg, step = 256 >> p.lg;
  const int strip = blockIdx.x % (unsigned)p.strips, F = p.F;
  const int64_t chunk = blockIdx.x / (unsigned)p.strips;
  const int f = (strip << p.lg | tc) * 8, left = F - f < 8 ? F - f : 8;
  if (left <= 0) return;
  const int64_t end = (chunk + 1) * p.rows < p.M ? (chunk + 1) * p.rows : p.M;
  float sg[8] = {}, su[8] = {};
  for (int64_t m = chunk * p.rows + tr; m < end; m += step) {
    float gate[8], up[8], d[8];
    load_cols<T>(p.pre, m * 2 * F + f, left, gate);
    load_cols<T>(p.pre, m * 2 * F + F + f, left, up);
    load_cols<T>(p.g, m * F + f, left, d);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = gate[e];
      gate[e] = ACT == ACT_NONE ? d[e] * up[e] : d[e] * up[e] * act_slope<ACT>(v);
      up[e] = d[e] * act_t<ACT>(v);
      sg[e] += gate[e];
      su[e] += up[e];
    }
    store_cols<T>(p.out, m * 2 * F + f, left, gate);
    store_cols<T>(p.out, m * 2 * F + F + f, left, up);
  }
  float* row = p.part + (chunk * step + tr) * 2 * F + f;
  for (int e = 0; e < left; ++e) {
    row[e] = sg[e];
    row[F + e] = su[e];
  }
}

// db [2 F] from the parts: one block per 32 columns, 32 threads of each.
template <typename T>
__global__ __launch_bounds__(1024) void gate_bias_kernel(GateSums p) {
  const int x = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int64_t N = 2 * (int64_t)p.F;
  __shared__ float red[32][33];
  for (int64_t c0 = (int64_t)blockIdx.x * 32; c0 < N; c0 += (int64_t)gridDim.x * 32) {
    const int64_t c = c0 + x;
    float v = 0.f;
    if (c < N) {
#pragma unroll 4
      for (unsigned j = row; j < p.parts; j += 32) v += p.part[(int64_t)j * N + c];
    }
    red[row][x] = v;
    __syncthreads();
    if (threadIdx.x < 32 && c < N) {
      float s = 0.f;
      for (int j = 0; j < 32; ++j) s += red[j][x];
      static_cast<typename Elem<T>::storage*>(p.db)[c] = Elem<T>::from_f32(s);
    }
    __syncthreads();
  }
}

// Chunks of at least 16 rows a thread, in at most 8 workgroups a CU (32 rows,
// half as many workgroups at 4096 rows: 103 us instead of 73).
static void gate_sums_split(int64_t M, int64_t F, GateSums& p) {
  const int64_t pieces = (F + 7) / 8;
  p.lg = 0;
  while (p.lg < 8 && (int64_t(1) << p.lg) < pieces) ++p.lg;
  const int64_t step = 256 >> p.lg, strips = (pieces + (1 << p.lg) - 1) >> p.lg;
  int64_t chunks = (M + 16 * step - 1) / (16 * step);
  const int64_t most = (8 * (int64_t)cu_count_current() + strips - 1) / strips;
  if (chunks > most) chunks = most;
  p.strips = (int)strips;
  p.rows = (M + chunks - 1) / chunks;
  chunks = (M + p.rows - 1) / p.rows;
  p.parts = (unsigned)(chunks * step);
}

int64_t gate_sums_work(int64_t M, int64_t F) {
  GateSums p;
  gate_sums_split(M, F, p);
  return (int64_t)p.parts * 2 * F * 4;
}

template <typename T>
static int launch_gate_sums_t(int act, const GateSums& p, hipStream_t st) {
  const dim3 grid(p.parts / (256u >> p.lg) * (unsigned)p.strips);
  if (act == ACT_SILU) hipLaunchKernelGGL((gate_sums_kernel<T, ACT_SILU>), grid, dim3(256), 0, st, p);
  else if (act == ACT_GELU) hipLaunchKernelGGL((gate_sums_kernel<T, ACT_GELU>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((gate_sums_kernel<T, ACT_NONE>), grid, dim3(256), 0, st, p);
  const int rc = check_launch("gate gradient");
  if (rc != SF_OK) return rc;
  int64_t blocks = (2 * (int64_t)p.F + 31) / 32;
  if (blocks > (1 << 20)) blocks = 1 << 20;
  hipLaunchKernelGGL((gate_bias_kernel<T>), dim3((unsigned)blocks), dim3(1024), 0, st, p);
  return check_launch("gate gradient (sums)");
}

int launch_gate_sums(int act, const void* g, const void* pre, void* out, void* db, float* part, int64_t M, int64_t F,
                     sf_dtype dt, hipStream_t st) {
  GateSums p;
  gate_sums_split(M, F, p);
  p.g = g, p.pre = pre, p.out = out, p.db = db, p.part = part;
  p.M = M;
  p.F = (int)F;
  switch (dt) {
    case SF_F16: return launch_gate_sums_t<F16>(act, p, st);
    case SF_BF16: return launch_gate_sums_t<BF16>(act, p, st);
    default: return launch_gate_sums_t<float>(act, p, st);
  }
}

// y = act(x Wg^T + bg) * (x Wu^T + bu), and the two projections, fp32, M <= 16:
// bound by reading the weight once.  A workgroup takes 8 gate rows and their 8
// up rows, the 16 rows of one MFMA operand; its eight waves share K, each step
// of a wave 16 k: a lane loads four of its row of W (and of x), and the k-th
// MFMA of 16 x 16 x 4 takes the k-th of each, UNROLL steps asked for ahead of
// their products (8 steps: 10 % slower; 16 gate rows a workgroup: 33 us for 25 at
// F 5312, whose 332 workgroups fill 256 CUs badly).  The waves' sums are added in
// order through LDS.  One row, F 11008, K 4096: 81 us, 361 MB, 4.5 TB/s; 16 rows
// 122 us, with x read from L2 by every workgroup.
template <int UNROLL>
__global__ __launch_bounds__(512) void gated_skinny32_kernel(const float* X, const float* W, const float* bias, float* Y,
                                                             float* pre, int M, int F, int K, int act) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, kc = (lane >> 4) * 4;
  const int n0 = blockIdx.x * 8, n = n0 + (r & 7);
  const int steps = (K + 15) / 16, per = (steps + 7) / 8, begin = wave * per;
  const int end = begin + per < steps ? begin + per : steps;
  const bool wok = n < F, xok = r < M;
  const float* wr = W + ((wok ? n : 0) + (r < 8 ? 0 : (int64_t)F)) * K + kc;
  const float* xr = X + (int64_t)(xok ? r : 0) * K + kc;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = begin; s0 < end; s0 += UNROLL) {
    f32x4 w[UNROLL], x[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int s = s0 + u;
      const bool in = s < end && s * 16 + kc < K;  // K % 4 == 0: all four or none
      const f32x4 z = {0.f, 0.f, 0.f, 0.f};
      w[u] = in && wok ? __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(wr + s * 16)) : z;
      x[u] = in && xok ? *reinterpret_cast<const f32x4*>(xr + s * 16) : z;
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(w[u][e], x[u][e], acc, 0, 0, 0);
  }
  // Lane (g, m) holds rows 4 g .. 4 g + 3 of token m: rows 0 .. 7 gates, 8 .. 15
  // the up rows.
  __shared__ float red[8][4][64];
#pragma unroll
  for (int q = 0; q < 4; ++q) red[wave][q][lane] = acc[q];
  __syncthreads();
  const int m = threadIdx.x >> 3, c = threadIdx.x & 7, f = n0 + c;
  if (m >= M || f >= F) return;
  float g = 0.f, u = 0.f;
  for (int v = 0; v < 8; ++v) {
    g += red[v][c & 3][(c >> 2) * 16 + m];
    u += red[v][c & 3][(c >> 2) * 16 + 32 + m];
  }
  if (bias != nullptr) {
    g += bias[f];
    u += bias[F + f];
  }
  Y[(int64_t)m * F + f] = (act == ACT_SILU ? act_t<ACT_SILU>(g) : act == ACT_GELU ? act_t<ACT_GELU>(g) : g) * u;
  pre[(int64_t)m * 2 * F + f] = g;
  pre[(int64_t)m * 2 * F + F + f] = u;
}

int launch_gated_skinny32(const void* x, const void* W, const void* bias, void* y, void* pre, int64_t M, int64_t F,
                          int64_t K, int act, hipStream_t st) {
  hipLaunchKernelGGL((gated_skinny32_kernel<4>), dim3((unsigned)((F + 7) / 8)), dim3(512), 0, st,
                     static_cast<const float*>(x), static_cast<const float*>(W), static_cast<const float*>(bias),
                     static_cast<float*>(y), static_cast<float*>(pre), (int)M, (int)F, (int)K, act);
  return check_launch("gated product (fp32, few rows)");
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
