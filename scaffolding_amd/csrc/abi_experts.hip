// abi_experts.hip — C entry points of the expert operators and the 4-bit
// linear layer: argument checks
// (before any HIP call) and the choice of tiles.
#include "sf_internal.hpp"

namespace sf {

static bool known(sf_dtype d) { return d == SF_F32 || d == SF_F16 || d == SF_BF16; }
static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

static void tile_size(int cfg, int& bm, int& bn) {
  switch (cfg) {
    case TILE_NT_BIG: bm = bn = 256; return;
    case TILE_MID_128:
    case TILE_RAG_128: bm = bn = 128; return;
    case TILE_MID_32: bm = 32; bn = 64; return;
    case TILE32_SMALL2:
    case TILE32_SMALL2_ANY: bm = 16; bn = 32; return;
    default: bm = bn = 64; return;
  }
}

// Estimated us of a grouped product.  The sizes of the groups are on the
// device: `rows` rows in `reached` groups, each leaving half a tile.
//   256 x 256 tiles, one a CU and round: 12.4 us and 0.0227 us per k
//   smaller ones: tau[r - 1] us per 64 k when r workgroups share each CU
// Fitted to sweeps (bf16, us, 256 / 128 / 64 / 32 x 64 measured): 8192 rows, 8
// groups, K 1920 -> N 7680 282 / 298 / 467 / 632; 4096 rows 164 / 176 / 252 /
// 339; 1024 rows 67 / 85 / 89 / 110; dx of 2048 rows, 7680 -> 1920 201 / 125 /
// 153; 16384 rows, 8 groups, 4096 -> 4096 520 / 625 / 967; 256 rows 99 / 71 / 61
// / 59; 8192 rows, 64 groups, 2048 -> 1408 129 / 111 / 129 / 163.
struct TileCost {
  int cfg, bm, bn, occ;
  float tau[4];
};
static constexpr TileCost kDirect[] = {
    {TILE_MID_128, 128, 128, 2, {0.72f, 1.15f}},
    {TILE_MID_64, 64, 64, 3, {0.32f, 0.44f, 0.74f}},
    {TILE_MID_32, 32, 64, 3, {0.22f, 0.30f, 0.48f}},
};
// Register-staged loads (unaligned rows).
static constexpr TileCost kStaged[] = {
    {TILE_RAG_128, 128, 128, 2, {0.90f, 1.50f}},
    {TILE_RAG_64, 64, 64, 4, {0.45f, 0.85f, 1.10f, 1.75f}},
};

static int64_t row_tiles(int64_t rows, int64_t reached, int64_t bm) {
  const int64_t t = (2 * rows + bm * reached) / (2 * bm);
  return t > reached ? t : reached;
}

static float tile_us(const TileCost& c, int64_t rows, int64_t reached, int64_t N, int64_t K, int64_t cus) {
  const int64_t tiles = row_tiles(rows, reached, c.bm) * cdiv(N, c.bn), slots = c.occ * cus;
  float t = static_cast<float>(tiles / slots) * c.tau[c.occ - 1];
  const int64_t rem = tiles % slots;
  if (rem > 0) t += c.tau[cdiv(rem, cus) - 1];
  return t * static_cast<float>(cdiv(K, 64));
}

// Tile of a grouped product.  `vec`: operands for the 16-byte direct loads;
// `dma`: for 4-byte ones (fp32); `big`: a bias for the 256 x 256 tiles.
static int rows_tile(int64_t rows, int64_t reached, int64_t N, int64_t K, bool vec, bool dma, bool big, bool f32,
                     bool b_kmajor) {
  const int64_t cus = cu_count_current();
  if (f32) {
    // 64 x 64 tiles, a round of one a CU: 0.0178 us per k (0.023 by 4-byte
    // loads); 16 x 32 blocks, n a CU: 0.0065 n us per k, 0.008 n by shorter
    // loads, 0.9 of one at least.  Fitted to sweeps (us, tiles / blocks):
    // 3 rows, 5632 -> 195 100 / 29; 64 rows, 8 groups, 2048 -> 2048 42 / 31; 128
    // rows 42 / 44; 512 rows 71 / 113; 64 groups, 1024 -> 1024, 256 rows 81 / 68;
    // 1024 rows 83 / 97; 4-byte loads, 8 rows, 8 groups, 4095 -> 4095 171 / 102;
    // 512 rows, 1 group, 1023 -> 1021 29 / 34.  (n < 4096 keeps the grid small.)
    const float cu = static_cast<float>(cus);
    const int64_t t64 = row_tiles(rows, reached, 64) * cdiv(N, 64);
    const float n = static_cast<float>(row_tiles(rows, reached, 16) * cdiv(N, 32)) / cu;
    const float big = (vec ? 0.0178f : 0.023f) * static_cast<float>(cdiv(t64, cus));
    if ((vec && b_kmajor ? 0.0065f : 0.008f) * (n > 0.9f ? n : 0.9f) < big && n < 4096.0f)
      return vec ? TILE32_SMALL2 : TILE32_SMALL2_ANY;
    return vec ? TILE32_DMA : dma ? TILE32_RAG : TILE_GENERIC;
  }
  float best = 3.0e38f;
  int cfg = -1;
  if (vec && big && N > 128 && K % 128 == 0 && K >= 128) {
    const int64_t tiles = row_tiles(rows, reached, 256) * cdiv(N, 256), rem = tiles % cus;
    // a short last round runs as quarters (grouped_rows)
    const float last = rem == 0 ? 0.0f : (tiles > cus && 2 * rem <= cus ? 0.7f : 1.0f);
    best = (static_cast<float>(tiles / cus) + last) * (12.4f + 0.0227f * static_cast<float>(K));
    cfg = TILE_NT_BIG;
  }
  for (int i = 0; i < (vec ? 3 : 2); ++i) {
    const TileCost& c = vec ? kDirect[i] : kStaged[i];
    if (c.cfg == TILE_MID_32 && !b_kmajor) continue;
    const float us = tile_us(c, rows, reached, N, K, cus) + 5.0f;  // launch, first loads, epilogue
    if (us < best) {
      best = us;
      cfg = c.cfg;
    }
  }
  return cfg;
}

template <typename P>
static void fill(P& p, const void* A, const void* B, void* C, const void* bias, int64_t M, int64_t N, int64_t K,
                 const int32_t* offsets, int64_t groups, int64_t rows, sf_epilogue epi) {
  p = P{};
  p.A = A;
  p.B = B;
  p.C = C;
  p.bias = bias;
  p.M = static_cast<int>(M);
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.alpha = 1.0f;
  p.epi = epi;
  p.offsets = offsets;
  p.groups = static_cast<int>(groups);
  p.rows = static_cast<int>(rows);
}

// The sizes that all entries of the grouped products share.
static int grouped_check(const char* name, int64_t rows, int64_t groups, int64_t N, int64_t K, sf_dtype dtype) {
  if (!known(dtype)) return fail(SF_ERR_INVALID_ARG, "%s: unknown dtype %d", name, (int)dtype);
  if (rows < 0 || groups < 0 || N < 0 || K < 0) return fail(SF_ERR_INVALID_ARG, "%s: negative size", name);
  if (groups > kMaxGroups) return fail(SF_ERR_UNSUPPORTED, "%s: %lld groups (at most %d)", name, (long long)groups, kMaxGroups);
  constexpr int64_t most = int64_t(1) << 30;
  if (rows > most || N > most || K > most)
    return fail(SF_ERR_UNSUPPORTED, "%s: sizes must be at most 2^30 (tiles past them stay below 2^31)", name);
  return SF_OK;
}

// C rows = op(B[e]) A rows: M = rows, `N` columns out, `K` summed.
static int grouped_rows(const char* name, const void* A, const void* B, const void* bias, void* C,
                        const int32_t* offsets, int64_t rows, int64_t groups, int64_t N, int64_t K, bool b_kmajor,
                        sf_dtype dtype, sf_epilogue epi, hipStream_t st) {
  GroupedRows p;
  fill(p, A, B, C, bias, rows, N, K, offsets, groups, rows, epi);
  p.lda = K;
  p.ldb = b_kmajor ? K : N;
  p.ldc = N;
  p.sB = N * K;
  const bool f32 = dtype == SF_F32;
  // 16-byte rows; one weight and one tile of A below the direct loads' 2 GiB
  // (fp32, an N-contiguous weight: and the 64 rows past its K that the last
  // step's offsets reach, which would wrap at 4 GiB and read it again)
  const bool dma = f32 && N * K < (int64_t(1) << 28) && K < (int64_t(1) << 20) &&
                   (b_kmajor || N * (K + 64) < (int64_t(1) << 29));
  const bool vec = f32 ? dma && K % 4 == 0 && (b_kmajor || N % 4 == 0) && aligned16(A) && aligned16(B)
                       : K % 8 == 0 && (b_kmajor || N % 8 == 0) && aligned16(A) && aligned16(B) &&
                             N * K < (int64_t(1) << 30) && K < (int64_t(1) << 22);
  const int64_t reached = groups < rows ? (groups > 0 ? groups : 1) : rows;
  // the 256 x 256 tiles load an even group's bias by dwords, straight into LDS
  const bool big = !epi_has_bias(epi) || (reinterpret_cast<uintptr_t>(bias) & 3) == 0;
  const int cfg = rows_tile(rows, reached, N, K, vec, dma, big, f32, b_kmajor);
  int bm, bn;
  tile_size(cfg, bm, bn);
  p.tiles_n = static_cast<int>(cdiv(N, bn));
  const int64_t gx = grouped_max_tiles(rows, groups, bm) * p.tiles_n;
  if (gx > (int64_t(1) << 22)) return fail(SF_ERR_UNSUPPORTED, "%s: more than 2^22 tiles", name);
  // 256 x 256 tiles run in rounds of one a CU.  What the last round holds, if
  // it is half a round at most, runs as 128 x 128 tiles in a second launch
  // (8192 rows, 8 groups, 1920 -> 7680 bf16: 282 -> 271 us; 16384 rows, 4096 ->
  // 4096: 520 -> 497).
  const int64_t cus = cu_count_current();
  const bool pair = cfg == TILE_NT_BIG && gx > cus;
  if (pair) p.cus = static_cast<int>(cus);
  auto launch = [&](int c, int64_t grid) {
    const unsigned g = static_cast<unsigned>(grid);
    switch (dtype) {
      case SF_F16: return launch_grouped_rows_f16(b_kmajor, c, p, g, st);
      case SF_BF16: return launch_grouped_rows_bf16(b_kmajor, c, p, g, st);
      default: return launch_grouped_rows_f32(b_kmajor, c, p, g, st);
    }
  };
  const int rc = launch(cfg, gx);
  if (rc != SF_OK || !pair) return rc;
  return launch(TILE_MID_128, 2 * cus);  // four quarters of at most half the CUs' tiles
}

}  // namespace sf

using namespace sf;

extern "C" {

int64_t sf_route_topk_work(int64_t tokens, int64_t experts) {
  const int64_t nb = tokens > 0 ? route_blocks(tokens) : 0;
  return nb > 1 && experts > 0 ? (nb + 1) * experts * 4 : 0;
}

static int route_check(const char* name, int64_t tokens, int64_t experts, int64_t k, sf_dtype dtype) {
  if (!known(dtype)) return fail(SF_ERR_INVALID_ARG, "%s: unknown dtype %d", name, (int)dtype);
  if (tokens < 0 || experts < 1 || k < 1 || k > experts)
    return fail(SF_ERR_INVALID_ARG, "%s: needs tokens >= 0 and 1 <= k <= experts (tokens=%lld experts=%lld k=%lld)",
                name, (long long)tokens, (long long)experts, (long long)k);
  if (experts > kMaxGroups || k > route_max_k())
    return fail(SF_ERR_UNSUPPORTED, "%s: at most %d experts and k <= %d (experts=%lld k=%lld)", name, kMaxGroups,
                route_max_k(), (long long)experts, (long long)k);
  if (tokens * k >= INT32_MAX || tokens >= INT32_MAX)
    return fail(SF_ERR_UNSUPPORTED, "%s: tokens * k must be < 2^31 - 1", name);
  // the gradient takes four tokens a block of 256 threads, in a grid of fewer than 2^32
  if (tokens > (int64_t(1) << 26) - 4) return fail(SF_ERR_UNSUPPORTED, "%s: tokens must be at most 2^26 - 4", name);
  return SF_OK;
}

int sf_route_topk(const void* logits, int64_t tokens, int64_t experts, int64_t k, sf_dtype dtype, int renormalize,
                  float* weights, int32_t* expert, int32_t* offsets, int32_t* slots, void* work, void* stream) {
  clear_error();
  const int rc = route_check("sf_route_topk", tokens, experts, k, dtype);
  if (rc != SF_OK) return rc;
  if (offsets == nullptr) return fail(SF_ERR_INVALID_ARG, "sf_route_topk: null pointer");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (tokens == 0) return launch_zero(offsets, static_cast<size_t>(experts + 1) * 4, st);
  if (logits == nullptr || weights == nullptr || expert == nullptr || slots == nullptr ||
      (work == nullptr && sf_route_topk_work(tokens, experts) > 0))
    return fail(SF_ERR_INVALID_ARG, "sf_route_topk: null pointer");
  return launch_route(logits, tokens, experts, static_cast<int>(k), dtype, renormalize != 0, weights, expert, offsets,
                      slots, static_cast<int*>(work), st);
}

int sf_route_topk_backward(const float* grad_weights, const void* logits, const float* weights,
                           const int32_t* expert, int64_t tokens, int64_t experts, int64_t k, sf_dtype dtype,
                           int renormalize, void* grad_logits, void* stream) {
  clear_error();
  const int rc = route_check("sf_route_topk_backward", tokens, experts, k, dtype);
  if (rc != SF_OK) return rc;
  if (tokens == 0) return SF_OK;
  if (grad_weights == nullptr || logits == nullptr || weights == nullptr || expert == nullptr ||
      grad_logits == nullptr)
    return fail(SF_ERR_INVALID_ARG, "sf_route_topk_backward: null pointer");
  return launch_route_backward(grad_weights, logits, weights, expert, tokens, experts, static_cast<int>(k), dtype,
                               renormalize != 0, grad_logits, static_cast<hipStream_t>(stream));
}

static int rows_check(const char* name, int64_t tokens, int64_t k, int64_t cols, sf_dtype dtype) {
  if (!known(dtype)) return fail(SF_ERR_INVALID_ARG, "%s: unknown dtype %d", name, (int)dtype);
  if (tokens < 0 || k < 1 || cols < 0)
    return fail(SF_ERR_INVALID_ARG, "%s: needs tokens >= 0, k >= 1 and cols >= 0 (tokens=%lld k=%lld cols=%lld)", name,
                (long long)tokens, (long long)k, (long long)cols);
  if (tokens >= INT32_MAX || k >= INT32_MAX || cols >= INT32_MAX || tokens * k >= INT32_MAX)
    return fail(SF_ERR_UNSUPPORTED, "%s: tokens * k and cols must be < 2^31 - 1", name);
  if (cols > int64_t(1) << 30) return fail(SF_ERR_UNSUPPORTED, "%s: cols must be at most 2^30", name);
  return SF_OK;
}

int sf_dispatch_rows(const void* x, const int32_t* slots, void* rows, int64_t tokens, int64_t k, int64_t cols,
                     sf_dtype dtype, void* stream) {
  clear_error();
  const int rc = rows_check("sf_dispatch_rows", tokens, k, cols, dtype);
  if (rc != SF_OK || tokens == 0 || cols == 0) return rc;
  if (x == nullptr || slots == nullptr || rows == nullptr)
    return fail(SF_ERR_INVALID_ARG, "sf_dispatch_rows: null pointer");
  return launch_rows(0, x, nullptr, slots, nullptr, rows, nullptr, tokens, static_cast<int>(k), cols, dtype,
                     static_cast<hipStream_t>(stream));
}

int sf_combine_rows(const void* rows, const int32_t* slots, const float* weights, void* y, int64_t tokens, int64_t k,
                    int64_t cols, sf_dtype dtype, void* stream) {
  clear_error();
  const int rc = rows_check("sf_combine_rows", tokens, k, cols, dtype);
  if (rc != SF_OK || tokens == 0 || cols == 0) return rc;
  if (rows == nullptr || slots == nullptr || y == nullptr)
    return fail(SF_ERR_INVALID_ARG, "sf_combine_rows: null pointer");
  return launch_rows(1, rows, nullptr, slots, weights, y, nullptr, tokens, static_cast<int>(k), cols, dtype,
                     static_cast<hipStream_t>(stream));
}

int sf_combine_rows_backward(const void* grad, const void* rows, const int32_t* slots, const float* weights,
                             void* grad_rows, float* grad_weights, int64_t tokens, int64_t k, int64_t cols,
                             sf_dtype dtype, void* stream) {
  clear_error();
  const int rc = rows_check("sf_combine_rows_backward", tokens, k, cols, dtype);
  if (rc != SF_OK || tokens == 0) return rc;
  if (slots == nullptr || weights == nullptr || grad_weights == nullptr ||
      (cols > 0 && (grad == nullptr || rows == nullptr || grad_rows == nullptr)))
    return fail(SF_ERR_INVALID_ARG, "sf_combine_rows_backward: null pointer");
  return launch_rows(2, grad, rows, slots, weights, grad_rows, grad_weights, tokens, static_cast<int>(k), cols, dtype,
                     static_cast<hipStream_t>(stream));
}

int sf_grouped_linear(const void* x, const void* W, const int32_t* offsets, const void* bias, void* y, int64_t rows,
                      int64_t groups, int64_t N, int64_t K, sf_dtype dtype, sf_epilogue epi, void* stream) {
  clear_error();
  const int rc = grouped_check("sf_grouped_linear", rows, groups, N, K, dtype);
  if (rc != SF_OK) return rc;
  if (epi < SF_EPI_NONE || epi > SF_EPI_GELU_TANH)
    return fail(SF_ERR_INVALID_ARG, "sf_grouped_linear: unknown epilogue %d", (int)epi);
  if (epi_has_bias(epi) && bias == nullptr && groups > 0 && N > 0)
    return fail(SF_ERR_INVALID_ARG, "sf_grouped_linear: the epilogue needs a bias");
  if (rows == 0 || N == 0) return SF_OK;
  if (y == nullptr || offsets == nullptr || (K > 0 && (x == nullptr || (groups > 0 && W == nullptr))))
    return fail(SF_ERR_INVALID_ARG, "sf_grouped_linear: null pointer");
  return grouped_rows("sf_grouped_linear", x, W, bias, y, offsets, rows, groups, N, K, true, dtype, epi,
                      static_cast<hipStream_t>(stream));
}

int sf_grouped_linear_dx(const void* grad, const void* W, const int32_t* offsets, void* grad_x, int64_t rows,
                         int64_t groups, int64_t N, int64_t K, sf_dtype dtype, void* stream) {
  clear_error();
  const int rc = grouped_check("sf_grouped_linear_dx", rows, groups, N, K, dtype);
  if (rc != SF_OK || rows == 0 || K == 0) return rc;
  if (grad_x == nullptr || offsets == nullptr || (N > 0 && (grad == nullptr || (groups > 0 && W == nullptr))))
    return fail(SF_ERR_INVALID_ARG, "sf_grouped_linear_dx: null pointer");
  return grouped_rows("sf_grouped_linear_dx", grad, W, nullptr, grad_x, offsets, rows, groups, K, N, false, dtype,
                      SF_EPI_NONE, static_cast<hipStream_t>(stream));
}

int sf_grouped_linear_dw(const void* grad, const void* x, const int32_t* offsets, void* grad_W, void* grad_bias,
                         int64_t rows, int64_t groups, int64_t N, int64_t K, sf_dtype dtype, void* stream) {
  clear_error();
  int rc = grouped_check("sf_grouped_linear_dw", rows, groups, N, K, dtype);
  if (rc != SF_OK || groups == 0 || N == 0) return rc;
  if (offsets == nullptr || (K > 0 && grad_W == nullptr) || (rows > 0 && grad == nullptr) ||
      (rows > 0 && K > 0 && x == nullptr))
    return fail(SF_ERR_INVALID_ARG, "sf_grouped_linear_dw: null pointer");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (K > 0) {
    GroupedSums p;
    fill(p, grad, x, grad_W, nullptr, N, K, rows, offsets, groups, rows, SF_EPI_NONE);
    p.lda = N;
    p.ldb = K;
    p.ldc = K;
    p.sC = N * K;
    const bool f32 = dtype == SF_F32;
    // 16-byte rows; a group's rows, all rows at most, below the direct loads' 2 GiB
    const int64_t wide = N > K ? N : K;
    const bool small = (rows + 64) * wide < (int64_t(1) << (f32 ? 29 : 30));
    const int64_t step = f32 ? 4 : 8;
    const bool vec = small && N % step == 0 && K % step == 0 && aligned16(grad) && aligned16(x);
    // 256 x 256 tiles lead from the first row (bf16, us, 256 / 128: 8192 rows,
    // 8 groups, 1920 x 7680 253 / 302; 512 rows, 64 groups, 1024 x 1024 40 / 43)
    int cfg;
    if (f32)
      cfg = vec ? TILE32_DMA : (small ? TILE32_RAG : TILE_GENERIC);
    else if (N > 64 && K > 64)
      cfg = vec ? (N > 128 && K > 128 ? TILE_NT_BIG : TILE_MID_128) : TILE_RAG_128;
    else
      cfg = vec ? TILE_MID_64 : TILE_RAG_64;
    int bm, bn;
    tile_size(cfg, bm, bn);
    p.tiles_m = static_cast<int>(cdiv(N, bm));
    p.tiles_n = static_cast<int>(cdiv(K, bn));
    const int64_t gx = int64_t(p.tiles_m) * p.tiles_n;
    if (gx * groups > (int64_t(1) << 22)) return fail(SF_ERR_UNSUPPORTED, "sf_grouped_linear_dw: more than 2^22 tiles");
    const unsigned g = static_cast<unsigned>(gx), gy = static_cast<unsigned>(groups);
    switch (dtype) {
      case SF_F16: rc = launch_grouped_sums_f16(cfg, p, g, gy, st); break;
      case SF_BF16: rc = launch_grouped_sums_bf16(cfg, p, g, gy, st); break;
      default: rc = launch_grouped_sums_f32(cfg, p, g, gy, st); break;
    }
    if (rc != SF_OK) return rc;
  }
  if (grad_bias == nullptr) return SF_OK;
  return launch_group_colsum(grad, offsets, rows, groups, N, grad_bias, dtype, st);
}

int sf_act_backward(const void* grad, const void* pre, void* out, int64_t n, sf_dtype dtype, sf_epilogue act,
                    void* stream) {
  clear_error();
  if (!known(dtype)) return fail(SF_ERR_INVALID_ARG, "sf_act_backward: unknown dtype %d", (int)dtype);
  if (n < 0) return fail(SF_ERR_INVALID_ARG, "sf_act_backward: negative size");
  if (act != SF_EPI_SILU && act != SF_EPI_GELU_TANH)
    return fail(SF_ERR_INVALID_ARG, "sf_act_backward: act must be SF_EPI_SILU or SF_EPI_GELU_TANH, got %d", (int)act);
  if (n == 0) return SF_OK;
  if (grad == nullptr || pre == nullptr || out == nullptr)
    return fail(SF_ERR_INVALID_ARG, "sf_act_backward: null pointer");
  return launch_act_backward(epi_act(act), grad, pre, out, n, dtype, static_cast<hipStream_t>(stream));
}

static int q4_check(const char* name, int64_t rows, int64_t groups, int64_t N, int64_t K, int64_t group,
                    sf_dtype dtype) {
  int rc = grouped_check(name, rows, groups, N, K, dtype);
  if (rc != SF_OK) return rc;
  if (dtype == SF_F32) return fail(SF_ERR_UNSUPPORTED, "%s: scales and activations are F16 or BF16", name);
  if (K >= (int64_t(1) << 25)) return fail(SF_ERR_UNSUPPORTED, "%s: K must be < 2^25", name);
  if (group != 32 && group != 64 && (group < 128 || group % 128 != 0))
    return fail(SF_ERR_UNSUPPORTED, "%s: group %lld is not 32, 64 or a multiple of 128", name, (long long)group);
  if (K % group != 0)
    return fail(SF_ERR_INVALID_ARG, "%s: K = %lld is no multiple of the group %lld", name, (long long)K, (long long)group);
  return SF_OK;
}

int sf_linear_q4(const void* x, const void* q, const void* scales, const void* zeros, const int32_t* offsets,
                 const void* bias, void* y, int64_t rows, int64_t groups, int64_t N, int64_t K, int64_t group,
                 sf_dtype dtype, sf_epilogue epi, void* stream) {
  clear_error();
  const int rc = q4_check("sf_linear_q4", rows, groups, N, K, group, dtype);
  if (rc != SF_OK) return rc;
  if (offsets == nullptr && groups != 1)
    return fail(SF_ERR_INVALID_ARG, "sf_linear_q4: %lld weights need offsets", (long long)groups);
  if (epi < SF_EPI_NONE || epi > SF_EPI_GELU_TANH)
    return fail(SF_ERR_INVALID_ARG, "sf_linear_q4: unknown epilogue %d", (int)epi);
  if (epi_has_bias(epi) && bias == nullptr && groups > 0 && N > 0)
    return fail(SF_ERR_INVALID_ARG, "sf_linear_q4: the epilogue needs a bias");
  if (rows == 0 || N == 0) return SF_OK;
  if (y == nullptr || (K > 0 && (x == nullptr || (groups > 0 && (q == nullptr || scales == nullptr)))))
    return fail(SF_ERR_INVALID_ARG, "sf_linear_q4: null pointer");
  if (!aligned16(x) || !aligned16(q)) return fail(SF_ERR_UNSUPPORTED, "sf_linear_q4: x and q must be 16-byte aligned");
  return launch_q4(x, q, scales, zeros, bias, y, offsets, groups, rows, N, K, group, dtype, epi,
                   static_cast<hipStream_t>(stream));
}

int sf_linear_q4_plan(int64_t rows, int64_t groups, int64_t N, int64_t K, int64_t group, int zeros, int grouped,
                      char* buf, int len) {
  clear_error();
  if (buf == nullptr || len <= 0) return fail(SF_ERR_INVALID_ARG, "sf_linear_q4_plan: bad buffer");
  buf[0] = 0;
  const int rc = q4_check("sf_linear_q4_plan", rows, groups, N, K, group, SF_BF16);
  if (rc != SF_OK) return rc;
  if (grouped == 0 && groups != 1)
    return fail(SF_ERR_INVALID_ARG, "sf_linear_q4_plan: %lld weights need offsets", (long long)groups);
  if (rows == 0 || N == 0) {
    snprintf(buf, static_cast<size_t>(len), "noop");
    return SF_OK;
  }
  const Q4Variant v = q4_variant(rows, groups, grouped != 0, N, K, group, zeros != 0);
  snprintf(buf, static_cast<size_t>(len), "q4 16x%d %d waves, scales in %d", v.columns, v.waves, v.segments);
  return SF_OK;
}

int sf_q4_expand(const void* q, const void* scales, const void* zeros, void* w, int64_t groups, int64_t N, int64_t K,
                 int64_t group, sf_dtype dtype, void* stream) {
  clear_error();
  const int rc = q4_check("sf_q4_expand", 0, groups, N, K, group, dtype);
  if (rc != SF_OK || groups == 0 || N == 0 || K == 0) return rc;
  if (q == nullptr || scales == nullptr || w == nullptr)
    return fail(SF_ERR_INVALID_ARG, "sf_q4_expand: null pointer");
  if (!aligned16(q) || !aligned16(w)) return fail(SF_ERR_UNSUPPORTED, "sf_q4_expand: q and w must be 16-byte aligned");
  return launch_q4_expand(q, scales, zeros, w, groups, N, K, group, dtype, static_cast<hipStream_t>(stream));
}

}  // extern "C"
