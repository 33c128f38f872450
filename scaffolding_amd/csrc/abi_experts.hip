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
    case TILE32_SMALL2: bm = 16; bn = 32; return;
    default: bm = bn = 64; return;
  }
}

// Estimated us of a grouped product on 256 x 256 tiles (one a CU and round)
// and on 128 x 128 tiles (two a CU; the last of them by itself runs faster),
// for groups that each leave half a tile.  Fitted to sweeps (bf16, us, 256 /
// 128 measured): 8192 rows, 8 groups, K 1920 -> N 7680 282 / 298, 7680 -> 1920
// 370 / 285; 4096 rows 164 / 176, 198 / 227; 2048 rows, 7680 -> 1920 201 / 125;
// 16384 rows, 8 groups, 4096 -> 4096 520 / 625; 8192 rows, 64 groups, 2048 ->
// 1408 129 / 111; 512 rows, 8 groups, 4096 -> 4096 101 / 73.
static float big_us(int64_t rows, int64_t reached, int64_t N, int64_t K, int64_t cus) {
  const int64_t tiles = (2 * rows + 256 * reached) / 512 * cdiv(N, 256);
  return static_cast<float>(cdiv(tiles, cus)) * (12.4f + 0.0227f * static_cast<float>(K));
}
static float mid_us(int64_t rows, int64_t reached, int64_t N, int64_t K, int64_t cus) {
  const int64_t tiles = (2 * rows + 128 * reached) / 256 * cdiv(N, 128);
  const int64_t rem = tiles % (2 * cus);
  const float rounds = static_cast<float>(tiles / (2 * cus)) + (rem == 0 ? 0.0f : (rem <= cus ? 0.65f : 1.0f));
  return rounds * (2.6f + 0.018f * static_cast<float>(K));
}

// Tile of a grouped product whose `rows` rows fall into `reached` groups (the
// sizes themselves are on the device; `per` rows each on average).  `vec`:
// operands for the 16-byte direct loads; `dma`: for 4-byte ones (fp32).
static int rows_tile(int64_t rows, int64_t reached, int64_t N, int64_t K, bool vec, bool dma, bool f32,
                     bool b_kmajor) {
  const int64_t per = rows / reached, cus = cu_count_current();
  if (f32) {
    if (!dma) return TILE_GENERIC;
    if (!vec) return TILE32_RAG;
    // as sf_gemm: few 64 x 64 tiles with a short k loop run as 16 x 32 blocks
    // (64 rows, 4 groups, 512 -> 512: 17.6 us on 64 x 64 tiles, 6.0)
    const int64_t t64 = (2 * rows + 64 * reached) / 128 * cdiv(N, 64);
    return 4 * t64 <= cus && K <= 2048 ? TILE32_SMALL2 : TILE32_DMA;
  }
  if (!vec) return per > 96 ? TILE_RAG_128 : TILE_RAG_64;
  // 256 rows, 8 groups, 4096 -> 4096: 59 us on 32 x 64, 61 on 64 x 64, 71 on
  // 128 x 128 (dx, which has no 32 x 64: 61, 63)
  if (per <= 32) return b_kmajor ? TILE_MID_32 : TILE_MID_64;
  const bool big = N > 128 && K % 128 == 0 && K >= 128;
  return big && big_us(rows, reached, N, K, cus) <= mid_us(rows, reached, N, K, cus) ? TILE_NT_BIG : TILE_MID_128;
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
  if (rows >= INT32_MAX || N >= INT32_MAX || K >= INT32_MAX)
    return fail(SF_ERR_UNSUPPORTED, "%s: sizes must be < 2^31 - 1", name);
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
  const bool dma = f32 && N * K < (int64_t(1) << 28) && K < (int64_t(1) << 20);
  const bool vec = f32 ? dma && K % 4 == 0 && (b_kmajor || N % 4 == 0) && aligned16(A) && aligned16(B)
                       : K % 8 == 0 && (b_kmajor || N % 8 == 0) && aligned16(A) && aligned16(B) &&
                             N * K < (int64_t(1) << 30) && K < (int64_t(1) << 22);
  const int64_t reached = groups < rows ? (groups > 0 ? groups : 1) : rows;
  const int cfg = rows_tile(rows, reached, N, K, vec, dma, f32, b_kmajor);
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
