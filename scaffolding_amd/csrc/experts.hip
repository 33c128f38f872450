// experts.hip — the row kernels around the grouped products: top-k routing
// and its gradient, the exchange between token order and expert order, the
// gradient of a fused activation and the bias gradient per group.
#include "grouped.hpp"
#include "rowio.hpp"
#include "sf_internal.hpp"

namespace sf {

// ---------------------------------------------------------------------
// Routing.  One wave per token: lane l holds logits l, l + 64, ... as integers
// in the numbers' order (a NaN above every number).  The k largest are found
// one after the other: the largest integer by a wave maximum in the lane
// network, then the first lane that holds it, so ties go to the lowest index.
// (With the index in the low half of a 64-bit key and the maximum by lane
// permutes, 16384 x 64 bf16 with k = 8 took 24.5 us instead of 13.)
//
// Places.  The assignments (t, j) are ordered by expert, within an expert by
// t k + j.  A block covers kRouteTokens consecutive tokens: it counts its
// assignments per expert, and an assignment's place is
//   first place of its expert  +  that expert's assignments in earlier blocks
//   +  those in earlier waves of its block  +  those in earlier lanes,
// all integer counts, so the places do not depend on which block or wave ran
// first.  With several blocks the counts of each go to `counts` and a second
// launch forms the sums; one block needs neither.  Past kRouteDirect blocks,
// where every block summing all counts would cost the square of the tokens, a
// launch in between turns the counts into sums over the earlier blocks.
// ---------------------------------------------------------------------
constexpr int kRouteTokens = 64;   // tokens per block
constexpr int kRouteThreads = 1024;
constexpr int kRouteMaxK = 16;
constexpr int kRouteDirect = 512;  // blocks

__device__ __forceinline__ uint32_t order_key(float f) {
  if (f != f) return 0xffffffffu;
  const uint32_t u = __float_as_uint(f + 0.0f);  // -0 and +0 are equal
  return (u >> 31) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float order_value(uint32_t k) {
  if (k == 0xffffffffu) return __uint_as_float(0x7fc00000u);
  return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k);
}

// Largest value of the 64 lanes, by the lane network (row shifts, then row
// broadcasts; the last lane ends with it).
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
  auto step = [&](uint32_t o) { v = o > v ? o : v; };
  step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false));
  step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false));
  step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false));
  step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false));
  step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false));
  step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false));
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// Places of the block's `n` <= 1024 assignments ex[] (experts, in order):
// base[e] is the first place of this block's assignments of expert e.
__device__ __forceinline__ void route_place(const int* ex, int n, int E, int (*hist)[kMaxGroups], const int* base,
                                            int* __restrict__ slots) {
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  constexpr int NW = kRouteThreads / 64;
  for (int i = tid; i < NW * E; i += kRouteThreads) hist[i / E][i % E] = 0;
  __syncthreads();
  const int e = tid < n ? ex[tid] : -1;
  // the lanes of this wave with the same expert: those that agree in every bit
  uint64_t same = __ballot(e >= 0);
  for (int bit = 1; bit < E; bit <<= 1) {
    const uint64_t has = __ballot((e & bit) != 0);
    same &= (e & bit) != 0 ? has : ~has;
  }
  const int rank = __popcll(same & ((1ull << lane) - 1));  // earlier ones
  if (e >= 0 && rank == 0) hist[wave][e] = __popcll(same);
  __syncthreads();
  if (e >= 0) {
    int at = base[e] + rank;
    for (int w = 0; w < wave; ++w) at += hist[w][e];
    slots[tid] = at;
  }
}

// Exclusive sums over experts of tot[0 .. E) into first[0 .. E], by one wave.
__device__ __forceinline__ void route_scan(const int* tot, int E, int* first) {
  const int lane = threadIdx.x & 63;
  int run = 0;
  for (int e0 = 0; e0 < E; e0 += 64) {
    const int v = e0 + lane < E ? tot[e0 + lane] : 0;
    const int s = wave_scan_sum(v);
    if (e0 + lane < E) first[e0 + lane] = run + s - v;
    run += __builtin_amdgcn_readlane(s, 63);
  }
  if (lane == 0) first[E] = run;
}

template <typename T, int CH>
__global__ __launch_bounds__(kRouteThreads) void route_kernel(const void* __restrict__ logits, int rows, int E, int k,
                                                              int renorm, float* __restrict__ weights,
                                                              int* __restrict__ experts, int* __restrict__ offsets,
                                                              int* __restrict__ slots, int* __restrict__ counts) {
  __shared__ int ex[kRouteTokens * kRouteMaxK];
  __shared__ int cnt[kMaxGroups];
  __shared__ int first[kMaxGroups + 1];
  __shared__ int hist[kRouteThreads / 64][kMaxGroups];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int t0 = blockIdx.x * kRouteTokens;
  const int nt = rows - t0 < kRouteTokens ? rows - t0 : kRouteTokens;
  for (int e = tid; e < E; e += kRouteThreads) cnt[e] = 0;
  __syncthreads();
  // all of this wave's tokens' logits are loaded ahead of the first one's work
  constexpr int PER = kRouteTokens * 64 / kRouteThreads;
  float all[PER][CH];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int t = wave + i * (kRouteThreads / 64);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int e = c * 64 + lane;
      all[i][c] = t < nt && e < E ? Chunk8<T>::get(logits, (int64_t)(t0 + t) * E + e) : -INFINITY;
    }
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int t = wave + i * (kRouteThreads / 64);
    if (t >= nt) break;
    const int64_t row = t0 + t;
    const float(&v)[CH] = all[i];
    uint32_t key[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) key[c] = c * 64 + lane < E ? order_key(v[c]) : 0;  // 0 is below the key of every number
    uint32_t top = 0, val = 0;  // the largest key, and lane j's: the j-th
    int mine = 0;
    for (int j = 0; j < k; ++j) {
      uint32_t best = key[0];
#pragma unroll
      for (int c = 1; c < CH; ++c) best = key[c] > best ? key[c] : best;
      best = wave_max_u32(best);
      int e = 0;
      bool found = false;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const uint64_t has = __ballot(key[c] == best);
        if (!found && has != 0) {  // uniform
          const int src = __builtin_ctzll(has);
          e = c * 64 + src;
          if (lane == src) key[c] = 0;
          found = true;
        }
      }
      if (j == 0) top = best;
      if (lane == j) {
        val = best;
        mine = e;
      }
    }
    // softmax numerators; a token with no expert allowed (all -inf) has none
    const float most = order_value(top);
    const float w = lane < k && most != -INFINITY ? expf(order_value(val) - most) : 0.f;
    float sum = wave_sum(w);
    if (!renorm) {  // over every expert instead of the chosen ones
      float s = 0.f;
#pragma unroll
      for (int c = 0; c < CH; ++c)
        if (c * 64 + lane < E) s += most == -INFINITY ? 0.f : expf(v[c] - most);
      sum = wave_sum(s);
    }
    if (lane < k) {
      weights[row * k + lane] = most == -INFINITY ? 0.f : w / sum;
      experts[row * k + lane] = mine;
      ex[t * k + lane] = mine;
      atomicAdd(&cnt[mine], 1);
    }
  }
  __syncthreads();
  if (counts != nullptr) {
    for (int e = tid; e < E; e += kRouteThreads) counts[(int64_t)blockIdx.x * E + e] = cnt[e];
    return;
  }
  if (wave == 0) route_scan(cnt, E, first);
  __syncthreads();
  for (int e = tid; e <= E; e += kRouteThreads) offsets[e] = first[e];
  route_place(ex, nt * k, E, hist, first, slots);
}

// counts[b][e] -> assignments of e in blocks before b, for the nb blocks, and
// counts[nb][e] -> all of them.  A block takes 16 experts: 64 threads each, a
// contiguous share of the blocks per thread, the shares' sums scanned by lane.
__global__ __launch_bounds__(1024) void route_scan_kernel(int* __restrict__ counts, int nb, int E) {
  __shared__ int sums[16][65];
  const int q = threadIdx.x & 15, share = threadIdx.x >> 4;
  const int e = blockIdx.x * 16 + q;
  const int b0 = (int)((int64_t)nb * share / 64), b1 = (int)((int64_t)nb * (share + 1) / 64);
  int sum = 0;
  if (e < E)
#pragma unroll 8
    for (int b = b0; b < b1; ++b) sum += counts[(int64_t)b * E + e];
  sums[q][share] = sum;
  __syncthreads();
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int v = sums[wave][lane];
  const int upto = wave_scan_sum(v);
  sums[wave][lane] = upto - v;
  if (lane == 63) sums[wave][64] = upto;
  __syncthreads();
  if (e >= E) return;
  int run = sums[q][share];
  for (int b = b0; b < b1; ++b) {
    const int c = counts[(int64_t)b * E + e];
    counts[(int64_t)b * E + e] = run;
    run += c;
  }
  if (share == 0) counts[(int64_t)nb * E + e] = sums[q][64];
}

// Last launch of several blocks: block b places its own assignments, after
// summing the blocks' counts if they are not sums already; block 0 writes the
// offsets.
__global__ __launch_bounds__(kRouteThreads) void route_place_kernel(const int* __restrict__ experts, int rows, int E,
                                                                    int k, const int* __restrict__ counts, int summed,
                                                                    int* __restrict__ offsets,
                                                                    int* __restrict__ slots) {
  __shared__ int ex[kRouteTokens * kRouteMaxK];
  __shared__ int before[kMaxGroups];
  __shared__ int total[kMaxGroups];
  __shared__ int first[kMaxGroups + 1];
  __shared__ int hist[kRouteThreads / 64][kMaxGroups];
  const int tid = threadIdx.x, wave = tid >> 6;
  const int t0 = blockIdx.x * kRouteTokens;
  const int nt = rows - t0 < kRouteTokens ? rows - t0 : kRouteTokens;
  const int64_t a0 = (int64_t)t0 * k;
  const int n = nt * k;
  const int nb = gridDim.x;
  if (tid < n) ex[tid] = experts[a0 + tid];
  if (summed) {
    for (int e = tid; e < E; e += kRouteThreads) {
      before[e] = counts[(int64_t)blockIdx.x * E + e];
      total[e] = counts[(int64_t)nb * E + e];
    }
  } else {
    for (int e = tid; e < E; e += kRouteThreads) before[e] = total[e] = 0;
    __syncthreads();
    // every thread sums a share of the blocks for one expert
    const int lanes = E < kRouteThreads ? E : kRouteThreads;
    const int shares = kRouteThreads / lanes;
    const int share = tid / lanes;
    if (share < shares) {
      for (int e = tid % lanes; e < E; e += lanes) {
        int sum = 0, pre = 0;
#pragma unroll 8
        for (int b = share; b < nb; b += shares) {
          const int c = counts[(int64_t)b * E + e];
          sum += c;
          pre += b < (int)blockIdx.x ? c : 0;
        }
        atomicAdd(&total[e], sum);
        atomicAdd(&before[e], pre);
      }
    }
  }
  __syncthreads();
  if (wave == 0) route_scan(total, E, first);
  __syncthreads();
  if (blockIdx.x == 0)
    for (int e = tid; e <= E; e += kRouteThreads) offsets[e] = first[e];
  __syncthreads();
  for (int e = tid; e < E; e += kRouteThreads) first[e] += before[e];
  route_place(ex, n, E, hist, first, slots + a0);
}

// Gradient of the logits, one wave per token.  Renormalised weights are a
// softmax over the chosen logits: dl = w (g - <g, w>) there, 0 elsewhere;
// otherwise over all: dl = p ([chosen] g - <g, p>).  p is formed again from
// the logits.  A token without an allowed expert has zero gradient.
template <typename T, int CH>
__global__ __launch_bounds__(256) void route_backward_kernel(const float* __restrict__ gw,
                                                             const void* __restrict__ logits,
                                                             const float* __restrict__ weights,
                                                             const int* __restrict__ experts, int rows, int E, int k,
                                                             int renorm, void* __restrict__ dl) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  float g = 0.f, w = 0.f;
  int e = -1;
  if (lane < k) {
    g = gw[row * k + lane];
    w = weights[row * k + lane];
    e = experts[row * k + lane];
  }
  const float dot = wave_sum(g * w);
  float p[CH], out[CH];
  if (renorm) {
#pragma unroll
    for (int c = 0; c < CH; ++c) out[c] = 0.f;
  } else {
    float most = -INFINITY;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      p[c] = c * 64 + lane < E ? Chunk8<T>::get(logits, row * E + c * 64 + lane) : -INFINITY;
      most = fmaxf(most, p[c]);
    }
    most = wave_max(most);
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      p[c] = most == -INFINITY ? 0.f : expf(p[c] - most);
      s += p[c];
    }
    s = wave_sum(s);
    const float inv = most == -INFINITY ? 0.f : 1.0f / s;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      p[c] *= inv;
      out[c] = -p[c] * dot;
    }
  }
  for (int j = 0; j < k; ++j) {  // the chosen experts, one lane each
    const int ej = __builtin_amdgcn_readlane(e, j);
    const float gj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(g), j));
    const float wj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), j));
#pragma unroll
    for (int c = 0; c < CH; ++c)
      if (c * 64 + lane == ej) out[c] = wj * (gj - dot);
  }
#pragma unroll
  for (int c = 0; c < CH; ++c)
    if (c * 64 + lane < E) Chunk8<T>::put(dl, row * E + c * 64 + lane, out[c]);
}

int64_t route_blocks(int64_t rows) { return (rows + kRouteTokens - 1) / kRouteTokens; }
int route_max_k() { return kRouteMaxK; }

template <typename T>
static int launch_route_t(const void* logits, int64_t rows, int64_t E, int k, bool renorm, float* weights,
                          int* experts, int* offsets, int* slots, int* work, hipStream_t st) {
  const unsigned nb = static_cast<unsigned>(route_blocks(rows));
  int* counts = nb > 1 ? work : nullptr;
  const int r = static_cast<int>(rows), e = static_cast<int>(E);
#define SF_ROUTE(CH)                                                                                              \
  hipLaunchKernelGGL((route_kernel<T, CH>), dim3(nb), dim3(kRouteThreads), 0, st, logits, r, e, k, renorm ? 1 : 0, \
                     weights, experts, offsets, slots, counts)
  if (E <= 64) SF_ROUTE(1);
  else if (E <= 128) SF_ROUTE(2);
  else if (E <= 256) SF_ROUTE(4);
  else SF_ROUTE(16);
#undef SF_ROUTE
  int rc = check_launch("routing");
  if (rc != SF_OK || nb == 1) return rc;
  const int summed = nb > kRouteDirect ? 1 : 0;
  if (summed) {
    hipLaunchKernelGGL(route_scan_kernel, dim3((e + 15) / 16), dim3(1024), 0, st, work, static_cast<int>(nb), e);
    rc = check_launch("routing sums");
    if (rc != SF_OK) return rc;
  }
  hipLaunchKernelGGL(route_place_kernel, dim3(nb), dim3(kRouteThreads), 0, st, experts, r, e, k, work, summed, offsets,
                     slots);
  return check_launch("routing places");
}

int launch_route(const void* logits, int64_t rows, int64_t E, int k, sf_dtype dt, bool renorm, float* weights,
                 int* experts, int* offsets, int* slots, int* work, hipStream_t st) {
  switch (dt) {
    case SF_F16: return launch_route_t<F16>(logits, rows, E, k, renorm, weights, experts, offsets, slots, work, st);
    case SF_BF16: return launch_route_t<BF16>(logits, rows, E, k, renorm, weights, experts, offsets, slots, work, st);
    default: return launch_route_t<float>(logits, rows, E, k, renorm, weights, experts, offsets, slots, work, st);
  }
}

template <typename T>
static int launch_route_backward_t(const float* gw, const void* logits, const float* weights, const int* experts,
                                   int64_t rows, int64_t E, int k, bool renorm, void* dl, hipStream_t st) {
  const dim3 g(static_cast<unsigned>((rows + 3) / 4));
  const int r = static_cast<int>(rows), e = static_cast<int>(E);
#define SF_ROUTE(CH)                                                                                              \
  hipLaunchKernelGGL((route_backward_kernel<T, CH>), g, dim3(256), 0, st, gw, logits, weights, experts, r, e, k,   \
                     renorm ? 1 : 0, dl)
  if (E <= 64) SF_ROUTE(1);
  else if (E <= 128) SF_ROUTE(2);
  else if (E <= 256) SF_ROUTE(4);
  else SF_ROUTE(16);
#undef SF_ROUTE
  return check_launch("routing gradient");
}

int launch_route_backward(const float* gw, const void* logits, const float* weights, const int* experts, int64_t rows,
                          int64_t E, int k, sf_dtype dt, bool renorm, void* dl, hipStream_t st) {
  switch (dt) {
    case SF_F16: return launch_route_backward_t<F16>(gw, logits, weights, experts, rows, E, k, renorm, dl, st);
    case SF_BF16: return launch_route_backward_t<BF16>(gw, logits, weights, experts, rows, E, k, renorm, dl, st);
    default: return launch_route_backward_t<float>(gw, logits, weights, experts, rows, E, k, renorm, dl, st);
  }
}

// ---------------------------------------------------------------------
// Rows between token order and expert order: bound by memory, one pass.  A
// token's row is shared by 2^lg consecutive threads of a block of 256, eight
// columns each at a time; rows may start at any element (16-byte accesses at
// element alignment).  Slots outside [0, n) are skipped.
// ---------------------------------------------------------------------
struct RowsParams {
  const void* x;  // dispatch: tokens; combine: rows; its gradient: token gradients
  const void* y;  // combine's gradient: rows
  const int* slots;
  const float* w;  // NULL: 1
  void* out;
  float* dw;
  int64_t tokens, n;  // n = tokens * k rows
  int k, D, lg;
};

template <typename T>
__global__ __launch_bounds__(256) void dispatch_kernel(RowsParams p) {
  const int64_t t = (int64_t)blockIdx.x * (256 >> p.lg) + (threadIdx.x >> p.lg);
  if (t >= p.tokens) return;
  const int step = 8 << p.lg;
  for (int c = (threadIdx.x & ((1 << p.lg) - 1)) * 8; c < p.D; c += step) {
    float v[8];
    load_cols<T>(p.x, t * p.D + c, p.D - c, v);
    for (int j = 0; j < p.k; ++j) {
      const int s = p.slots[t * p.k + j];
      if ((uint64_t)(int64_t)s < (uint64_t)p.n) store_cols<T>(p.out, (int64_t)s * p.D + c, p.D - c, v);
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void combine_kernel(RowsParams p) {
  const int64_t t = (int64_t)blockIdx.x * (256 >> p.lg) + (threadIdx.x >> p.lg);
  if (t >= p.tokens) return;
  const int step = 8 << p.lg;
  for (int c = (threadIdx.x & ((1 << p.lg) - 1)) * 8; c < p.D; c += step) {
    float a[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int j = 0; j < p.k; ++j) {
      const int s = p.slots[t * p.k + j];
      if ((uint64_t)(int64_t)s < (uint64_t)p.n) {
        float v[8];
        load_cols<T>(p.x, (int64_t)s * p.D + c, p.D - c, v);
        const float w = p.w != nullptr ? p.w[t * p.k + j] : 1.0f;
#pragma unroll
        for (int q = 0; q < 8; ++q) a[q] = __builtin_fmaf(w, v[q], a[q]);
      }
    }
    store_cols<T>(p.out, t * p.D + c, p.D - c, a);
  }
}

// drows[s] = w g[t], dw = <g[t], rows[s]>.  A wave at most takes a token and
// its slots one after the other, so its sums are formed per thread and then
// over the lanes, without a barrier (4096 x 2 rows of 1283 fp16: 16.8 us with a
// block of four waves a token, 14.0).  Where the tokens are too few for that to
// fill the GPU (PAIR: below 16 a CU), a block takes one slot of one token and
// the waves' sums are joined in their order.  bf16, us, PAIR / a wave a token:
// 512 x 8 rows of 4096 columns 19 / 52, 1024 x 2 of 1283 5.6 / 7.5, 2048 x 8 of
// 512 7.9 / 13.2, of 1283 35.1 / 35.8; 4095 x 2 of 1283 19.3 / 13.3, of 4096
// 31.3 / 30.5; 8192 x 8 of 1283 181 / 139, of 4096 253 / 296.
template <typename T, bool PAIR>
__global__ __launch_bounds__(256) void combine_backward_kernel(RowsParams p) {
  __shared__ float part[4];
  const int64_t item = (int64_t)blockIdx.x * (256 >> p.lg) + (threadIdx.x >> p.lg);
  const int64_t t = PAIR ? item / p.k : item;
  const bool live = t < p.tokens;
  const int in = threadIdx.x & ((1 << p.lg) - 1);
  const int step = 8 << p.lg;
  const int j0 = PAIR ? (int)(item % p.k) : 0, j1 = PAIR ? j0 + 1 : p.k;
  for (int j = j0; j < j1; ++j) {
    const int s = live ? p.slots[t * p.k + j] : -1;
    float dot = 0.f;
    if ((uint64_t)(int64_t)s < (uint64_t)p.n) {
      const float w = p.w[t * p.k + j];
#pragma unroll 2
      for (int c = in * 8; c < p.D; c += step) {
        float g[8], v[8], o[8];
        load_cols<T>(p.x, t * p.D + c, p.D - c, g);
        load_cols<T>(p.y, (int64_t)s * p.D + c, p.D - c, v);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          dot = __builtin_fmaf(g[q], v[q], dot);
          o[q] = w * g[q];
        }
        store_cols<T>(p.out, (int64_t)s * p.D + c, p.D - c, o);
      }
    }
    for (int off = p.lg < 6 ? 1 << p.lg >> 1 : 32; off > 0; off >>= 1) dot += __shfl_xor(dot, off, 64);
    if (PAIR && p.lg > 6) {  // uniform: the slot's columns are over several waves
      if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = dot;
      __syncthreads();
      const int w0 = (threadIdx.x >> p.lg) << (p.lg - 6);
      dot = 0.f;
      for (int i = 0; i < 1 << (p.lg - 6); ++i) dot += part[w0 + i];
    }
    if (live && in == 0) p.dw[t * p.k + j] = dot;
  }
}

template <typename T>
static int launch_rows_t(int op, RowsParams p, hipStream_t st) {
  // threads per token: enough for its columns, at most the block (the gradient:
  // a wave, or the block for each of its slots)
  const bool pair = op == 2 && p.tokens < 16 * static_cast<int64_t>(cu_count_current());
  int lg = 0;
  while (lg < (op == 2 && !pair ? 6 : 8) && (8 << lg) < p.D) ++lg;
  p.lg = lg;
  const int64_t per = 256 >> lg;
  const int64_t items = pair ? p.n : p.tokens;
  const int64_t nb = (items + per - 1) / per;
  if (nb >= int64_t(1) << 24) return fail(SF_ERR_UNSUPPORTED, "row exchange: too many tokens of this width");
  const dim3 g(static_cast<unsigned>(nb));
  if (op == 0) hipLaunchKernelGGL((dispatch_kernel<T>), g, dim3(256), 0, st, p);
  else if (op == 1) hipLaunchKernelGGL((combine_kernel<T>), g, dim3(256), 0, st, p);
  else if (pair) hipLaunchKernelGGL((combine_backward_kernel<T, true>), g, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((combine_backward_kernel<T, false>), g, dim3(256), 0, st, p);
  return check_launch("row exchange");
}

int launch_rows(int op, const void* x, const void* y, const int* slots, const float* w, void* out, float* dw,
                int64_t tokens, int k, int64_t D, sf_dtype dt, hipStream_t st) {
  RowsParams p;
  p.x = x; p.y = y; p.slots = slots; p.w = w; p.out = out; p.dw = dw;
  p.tokens = tokens; p.n = tokens * k; p.k = k; p.D = static_cast<int>(D); p.lg = 0;
  switch (dt) {
    case SF_F16: return launch_rows_t<F16>(op, p, st);
    case SF_BF16: return launch_rows_t<BF16>(op, p, st);
    default: return launch_rows_t<float>(op, p, st);
  }
}

// ---------------------------------------------------------------------
// out = g act'(pre), elementwise (act_slope).
// ---------------------------------------------------------------------
// (out may be g or pre, so no pointer is marked as the only one to its memory.)
template <typename T, int ACT>
__global__ __launch_bounds__(256) void act_backward_kernel(const void* g, const void* pre, void* out, int64_t n) {
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8; i < n; i += (int64_t)gridDim.x * 2048) {
    const int left = n - i < 8 ? (int)(n - i) : 8;
    float a[8], b[8];
    load_cols<T>(g, i, left, a);
    load_cols<T>(pre, i, left, b);
#pragma unroll
    for (int q = 0; q < 8; ++q) a[q] *= act_slope<ACT>(b[q]);
    store_cols<T>(out, i, left, a);
  }
}

template <typename T>
static int launch_act_backward_t(int act, const void* g, const void* pre, void* out, int64_t n, hipStream_t st) {
  int64_t nb = (n + 2047) / 2048;
  if (nb > (1 << 20)) nb = 1 << 20;
  const dim3 grid(static_cast<unsigned>(nb));
  if (act == ACT_SILU)
    hipLaunchKernelGGL((act_backward_kernel<T, ACT_SILU>), grid, dim3(256), 0, st, g, pre, out, n);
  else
    hipLaunchKernelGGL((act_backward_kernel<T, ACT_GELU>), grid, dim3(256), 0, st, g, pre, out, n);
  return check_launch("activation gradient");
}

int launch_act_backward(int act, const void* g, const void* pre, void* out, int64_t n, sf_dtype dt, hipStream_t st) {
  switch (dt) {
    case SF_F16: return launch_act_backward_t<F16>(act, g, pre, out, n, st);
    case SF_BF16: return launch_act_backward_t<BF16>(act, g, pre, out, n, st);
    default: return launch_act_backward_t<float>(act, g, pre, out, n, st);
  }
}

// ---------------------------------------------------------------------
// Column sums of each group's rows (the bias gradients): out[e, n] = sum over
// the rows r of group e of g[r, n].  A block takes 128 columns of one group:
// 16 lanes eight columns each, the 64 quarter-waves of the block every 64th
// row, fp32 partial sums joined through LDS in a fixed order.  Bound by
// memory; narrow blocks give every CU some (4096 rows, 8 groups, 7680 columns
// bf16: 24 us in 120 blocks of 512 columns, 480 of 128 take 12).
// ---------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(1024) void group_colsum_kernel(const void* __restrict__ g, const int* __restrict__ offsets,
                                                            int rows, int64_t N, void* __restrict__ out) {
  __shared__ float part[64][132];
  int first, cnt;
  group_bounds(offsets, (int)blockIdx.y, rows, first, cnt);
  const int q = threadIdx.x >> 4, l = threadIdx.x & 15;
  const int64_t c = (int64_t)blockIdx.x * 128 + l * 8;
  const int left = N - c >= 8 ? 8 : (int)(N - c);
  float a[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (left > 0) {
#pragma unroll 4
    for (int r = q; r < cnt; r += 64) {
      float v[8];
      load_cols<T>(g, (int64_t)(first + r) * N + c, left, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] += v[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) part[q][l * 8 + i] = a[i];
  __syncthreads();
  // eight threads a column, eight partial sums each, then a fixed tree
  const int col = threadIdx.x >> 3, o = threadIdx.x & 7;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s += part[o * 8 + i][col];
#pragma unroll
  for (int off = 4; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  const int64_t n = (int64_t)blockIdx.x * 128 + col;
  if (o == 0 && n < N) Chunk8<T>::put(out, (int64_t)blockIdx.y * N + n, s);
}

int launch_group_colsum(const void* g, const int* offsets, int64_t rows, int64_t groups, int64_t N, void* out,
                        sf_dtype dt, hipStream_t st) {
  if (N > int64_t(1) << 28) return fail(SF_ERR_UNSUPPORTED, "group column sums: more than 2^28 columns");
  const dim3 grid(static_cast<unsigned>((N + 127) / 128), static_cast<unsigned>(groups));
  const int r = static_cast<int>(rows);
  switch (dt) {
    case SF_F16: hipLaunchKernelGGL((group_colsum_kernel<F16>), grid, dim3(1024), 0, st, g, offsets, r, N, out); break;
    case SF_BF16: hipLaunchKernelGGL((group_colsum_kernel<BF16>), grid, dim3(1024), 0, st, g, offsets, r, N, out); break;
    default: hipLaunchKernelGGL((group_colsum_kernel<float>), grid, dim3(1024), 0, st, g, offsets, r, N, out); break;
  }
  return check_launch("group column sums");
}

}  // namespace sf
