// abi_block.hip — C entry points of the causal transformer block: norms of
// queries and keys with the rotation, gated feed-forward layers, windowed
// attention.  Argument checks (before any HIP call) and the choice of kernels.
#include "sf_internal.hpp"

namespace sf {

static bool known(sf_dtype d) { return d == SF_F32 || d == SF_F16 || d == SF_BF16; }
static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr int64_t kMostRows = int64_t(1) << 30;

// ---- norms of queries and keys ----------------------------------------------

static int norm_rope_check(const char* name, const float* table, int64_t table_rows, int64_t rot, sf_norm norm,
                           float eps, int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads, int64_t D,
                           sf_dtype dtype) {
  if (!known(dtype)) return fail(SF_ERR_INVALID_ARG, "%s: unknown dtype %d", name, (int)dtype);
  if (norm != SF_NORM_RMS && norm != SF_NORM_LAYER) return fail(SF_ERR_INVALID_ARG, "%s: unknown norm %d", name, (int)norm);
  if (batch < 0 || rows < 0 || heads < 1 || kv_heads < 1 || D < 1)
    return fail(SF_ERR_INVALID_ARG, "%s: needs batch, rows >= 0 and heads, kv_heads, D >= 1 (%lld, %lld, %lld, %lld, %lld)",
                name, (long long)batch, (long long)rows, (long long)heads, (long long)kv_heads, (long long)D);
  if (D > 256 || heads > 4096 || kv_heads > 4096)
    return fail(SF_ERR_UNSUPPORTED, "%s: at most 256 columns a head and 4096 heads (D=%lld heads=%lld kv_heads=%lld)",
                name, (long long)D, (long long)heads, (long long)kv_heads);
  if (batch > 0 && rows > kMostRows / batch)
    return fail(SF_ERR_UNSUPPORTED, "%s: batch * rows must be at most 2^30", name);
  if (rot < 0 || rot > D || (rot & 1))
    return fail(SF_ERR_INVALID_ARG, "%s: the rotated columns must be an even number up to D (rot=%lld D=%lld)", name,
                (long long)rot, (long long)D);
  if (rot > 0 && (table == nullptr || table_rows < 1))
    return fail(SF_ERR_INVALID_ARG, "%s: the rotation needs a table", name);
  if (!(eps >= 0.0f) || eps > 3.0e38f) return fail(SF_ERR_INVALID_ARG, "%s: eps must be finite and >= 0", name);
  return SF_OK;
}

static void norm_rope_fill(NormRopeArgs& a, const void* x, int64_t ldx, const float* table, int64_t table_rows,
                           int64_t rot, const int32_t* positions, const void* weight, sf_norm norm, float eps,
                           int interleaved, int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads, int64_t D) {
  a = NormRopeArgs{};
  a.x = x;
  a.ldx = ldx;
  a.table = table;
  a.table_rows = table_rows;
  a.positions = positions;
  a.weight = weight;
  a.batch = batch;
  a.rows = rows;
  a.eps = eps;
  a.heads = (int)heads;
  a.kv_heads = (int)kv_heads;
  a.D = (int)D;
  a.rot = (int)rot;
  a.layer = norm == SF_NORM_LAYER;
  a.pairs = interleaved != 0;
}

// Whether na elements from `a` on and nb from `b` on share memory.
static bool ranges_meet(const void* a, __int128 na, const void* b, __int128 nb, int size) {
  const __int128 a0 = reinterpret_cast<uintptr_t>(a), b0 = reinterpret_cast<uintptr_t>(b);
  return a0 < b0 + nb * size && b0 < a0 + na * size;
}

// ---- gated feed-forward layers ----------------------------------------------

static int gated_check(const char* name, int64_t M, int64_t F, int64_t K, sf_dtype dtype, sf_epilogue act) {
  if (!known(dtype)) return fail(SF_ERR_INVALID_ARG, "%s: unknown dtype %d", name, (int)dtype);
  if (M < 0 || F < 0 || K < 0) return fail(SF_ERR_INVALID_ARG, "%s: negative size", name);
  if (act != SF_EPI_NONE && act != SF_EPI_SILU && act != SF_EPI_GELU_TANH)
    return fail(SF_ERR_INVALID_ARG, "%s: the activation must be SF_EPI_NONE, SF_EPI_SILU or SF_EPI_GELU_TANH, got %d",
                name, (int)act);
  if (M > kMostRows || F > kMostRows / 2 || K > kMostRows)
    return fail(SF_ERR_UNSUPPORTED, "%s: M and K must be at most 2^30, F 2^29", name);
  return SF_OK;
}

// Tiles of a gated product: lines of W a tile takes are half gate, half up.  The
// times are fitted to a sweep of 20 to 4096 rows over layers of F 352 to 11008
// and K 208 to 4096 (bf16): there the choice is within 1 % of the fastest in 82 of
// 88 sizes and within 7 % in all.
struct GatedTile {
  int cfg, bm, bn, occ;
  float tau[4];  // us per 64 k when r workgroups share each CU, in line between
};
static constexpr GatedTile kGatedDirect[] = {
    {TILE_MID_128, 128, 128, 2, {0.68f, 1.14f}},
    {TILE_MID_64, 64, 64, 3, {0.29f, 0.44f, 0.60f}},
    {TILE_MID_32, 32, 64, 3, {0.21f, 0.26f, 0.40f}},
};
static constexpr GatedTile kGatedStaged[] = {
    {TILE_RAG_128, 128, 128, 2, {0.90f, 1.50f}},
    {TILE_RAG_64, 64, 64, 4, {0.45f, 0.85f, 1.10f, 1.75f}},
};

static float gated_tiles_us(const GatedTile& c, int64_t tiles, int64_t K, int64_t cus) {
  const int64_t slots = c.occ * cus, rem = tiles % slots;
  float us = static_cast<float>(tiles / slots) * c.tau[c.occ - 1];
  if (rem > 0) {
    const int64_t r = rem / cus;
    const float part = static_cast<float>(rem % cus) / static_cast<float>(cus);
    us += r == 0 ? c.tau[0] : part == 0.0f ? c.tau[r - 1] : c.tau[r - 1] + part * (c.tau[r] - c.tau[r - 1]);
  }
  return us * static_cast<float>(cdiv(K, 64)) + 5.0f;  // launch, first loads, epilogue
}

// A round of 256 x 256 tiles; and one of `rem` of them, left whole or cut into
// quarters for a second launch.
static float gated_round_us(int64_t K) { return 12.4f + 0.0227f * static_cast<float>(K); }
static bool gated_quarters(int64_t rem, int64_t K, int64_t cus) {
  return rem > 0 && gated_tiles_us(kGatedDirect[0], 4 * rem, K, cus) < gated_round_us(K);
}

static int gated_tile(int64_t M, int64_t F, int64_t K, bool rows16, bool direct, int& bm, int& bn) {
  const int64_t cus = cu_count_current();
  if (rows16 && M <= 16) {  // the weight is read once, as fast as it comes
    bm = 16;
    bn = 32;
    return TILE_SKINNY;
  }
  float best = 3.0e38f;
  int cfg = -1;
  if (direct && K % 128 == 0 && K >= 128 && F > 64) {
    const int64_t tiles = cdiv(M, 256) * cdiv(F, 128), rem = tiles % cus;
    best = static_cast<float>(tiles / cus) * gated_round_us(K);
    if (tiles > cus && gated_quarters(rem, K, cus)) best += gated_tiles_us(kGatedDirect[0], 4 * rem, K, cus);
    else if (rem > 0) best += gated_round_us(K);
    cfg = TILE_NT_BIG;
    bm = bn = 256;
  }
  for (int i = 0; i < (direct ? 3 : 2); ++i) {
    const GatedTile& c = direct ? kGatedDirect[i] : kGatedStaged[i];
    const float us = gated_tiles_us(c, cdiv(M, c.bm) * cdiv(2 * F, c.bn), K, cus);
    if (us < best) {
      best = us;
      cfg = c.cfg;
      bm = c.bm;
      bn = c.bn;
    }
  }
  return cfg;
}

// The launches of a 16-bit layer: `tiles` of kernel cfg, of which a second launch
// takes those from `head` on as quarters.
struct GatedPlan {
  int cfg, bm, bn;
  int64_t tiles, head;
  bool persist;
};

static int gated_plan(const char* name, const void* x, const void* W, int64_t M, int64_t F, int64_t K, GatedPlan& g) {
  const bool rows16 = K % 8 == 0 && aligned16(x) && aligned16(W);
  // the direct loads' 32-bit offsets reach 2 GiB of either operand
  const bool direct = rows16 && K > 0 && 2 * F * K < kMostRows && M * K < kMostRows;
  g = GatedPlan{};
  g.cfg = gated_tile(M, F, K, rows16, direct, g.bm, g.bn);
  g.tiles = cdiv(M, g.bm) * cdiv(2 * F, g.bn);
  g.head = g.tiles;
  if (g.tiles > (int64_t(1) << 22)) return fail(SF_ERR_UNSUPPORTED, "%s: more than 2^22 tiles", name);
  if (g.cfg != TILE_NT_BIG) return SF_OK;
  // A part round that its tiles' quarters fill better runs as those: 4096 rows, F
  // 11008, K 4096 (5.4 rounds) 570 -> 552 us, F 2048 of 4352 rows (1.1) 172 -> 153;
  // past about half a round the quarters take as long.
  const int64_t cus = cu_count_current(), rem = g.tiles % cus;
  if (g.tiles > cus && gated_quarters(rem, K, cus)) g.head = g.tiles - rem;
  // One workgroup a CU walks the tiles where the last round is full or at most
  // half full, as sf_gemm's.
  g.persist = g.head > cus && cus % kNumXcd == 0 && 2 * (g.head % cus) <= cus;
  return SF_OK;
}

static int gated16(const void* x, const void* W, const void* bias, void* y, void* pre, int64_t M, int64_t F, int64_t K,
                   sf_dtype dtype, sf_epilogue act, hipStream_t st) {
  GatedPlan g;
  int rc = gated_plan("sf_gated_linear", x, W, M, F, K, g);
  if (rc != SF_OK) return rc;
  GatedParams p{};
  p.A = x;
  p.B = W;
  p.C = y;
  p.bias = bias;
  p.pre = pre;
  p.lda = p.ldb = K;
  p.ldc = F;
  p.M = (int)M;
  p.N = (int)(2 * F);
  p.F = (int)F;
  p.K = (int)K;
  p.alpha = 1.0f;
  p.epi = bias == nullptr ? act
          : act == SF_EPI_SILU ? SF_EPI_BIAS_SILU
          : act == SF_EPI_GELU_TANH ? SF_EPI_BIAS_GELU_TANH : SF_EPI_BIAS;
  p.tiles_m = (int)cdiv(M, g.bm);
  p.tiles_n = (int)cdiv(2 * F, g.bn);
  p.head = (int)g.head;
  p.persist = g.persist ? cu_count_current() : 0;
  const auto launch = [&](int c, unsigned gx) {
    return dtype == SF_BF16 ? launch_gated_bf16(c, p, gx, st) : launch_gated_f16(c, p, gx, st);
  };
  rc = launch(g.cfg, p.persist > 0 ? (unsigned)p.persist : (unsigned)g.head);
  if (rc != SF_OK || g.head == g.tiles) return rc;
  p.persist = 0;
  p.big_m = p.tiles_m;
  p.big_n = p.tiles_n;
  return launch(TILE_MID_128, (unsigned)(4 * (g.tiles - g.head)));
}

// fp32 layers of few rows, in one launch, bound by the weight's reading (F 5312, K
// 2416: 25 us for one row and 36 for 16, the product and the gate 86; F 11008, K
// 4096: 81 and 122, 145).
static bool gated_few32(const void* x, const void* W, int64_t M, int64_t F, int64_t K) {
  return M <= 16 && K > 0 && K % 4 == 0 && aligned16(x) && aligned16(W) && F < (int64_t(1) << 26);
}

// ---- windowed attention -------------------------------------------------------

// Sizes that every entry shares; *noop for an empty call.
static int window_sizes(const char* name, int64_t batch, int64_t heads, int64_t kv_heads, int64_t rows,
                        int64_t capacity, int64_t D, int64_t window, int64_t sinks, bool* noop) {
  *noop = false;
  if (batch < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || rows < 0 || capacity < 0)
    return fail(SF_ERR_INVALID_ARG, "%s: needs batch, rows >= 0 and heads a multiple of kv_heads >= 1 (%lld, %lld, %lld, %lld)",
                name, (long long)batch, (long long)rows, (long long)heads, (long long)kv_heads);
  if (window < 0 || sinks < 0) return fail(SF_ERR_INVALID_ARG, "%s: negative window or sinks", name);
  if (D < 8 || D > 128 || D % 8 != 0)
    return fail(SF_ERR_UNSUPPORTED, "%s: head size %lld (multiples of 8 up to 128)", name, (long long)D);
  if (rows > kMostRows / 2 || capacity > kMostRows / 2)
    return fail(SF_ERR_UNSUPPORTED, "%s: at most 2^29 rows", name);
  // workgroups of 256 threads, one more for the backward pass: a launch holds
  // fewer than 2^32 threads
  if (heads > (1 << 20) || batch > (1 << 24) || batch * heads >= (int64_t(1) << 24) / ((rows + 127) / 128 + 1))
    return fail(SF_ERR_UNSUPPORTED, "%s: batch * heads * (blocks of 128 rows + 1) must be below 2^24", name);
  *noop = batch == 0 || rows == 0;
  return SF_OK;
}

static int window_operand(const char* name, const char* what, const void* p, int64_t ld, int64_t stride, int64_t head,
                          int64_t D) {
  if (p == nullptr) return fail(SF_ERR_INVALID_ARG, "%s: null pointer (%s)", name, what);
  if (ld < D) return fail(SF_ERR_INVALID_ARG, "%s: row stride of %s below the head size", name, what);
  if (stride < 0 || head < 0) return fail(SF_ERR_INVALID_ARG, "%s: negative stride of %s", name, what);
  if (!aligned16(p) || ld % 8 || stride % 8 || head % 8)
    return fail(SF_ERR_UNSUPPORTED, "%s: rows of %s must be 16-byte aligned", name, what);
  if (ld >= (1 << 23)) return fail(SF_ERR_UNSUPPORTED, "%s: row stride of %s must be below 2^23", name, what);
  return SF_OK;
}

static int window_fill(const char* name, WinShape& a, const void* Q, int64_t ldq, int64_t strideQ, int64_t headQ,
                       const void* K, int64_t ldk, int64_t strideK, int64_t headK, const void* V, int64_t ldv,
                       int64_t strideV, int64_t headV, void* O, int64_t ldo, int64_t strideO, int64_t headO,
                       float scale, sf_dtype dtype) {
  if (!known(dtype)) return fail(SF_ERR_INVALID_ARG, "%s: unknown dtype %d", name, (int)dtype);
  if (dtype == SF_F32) return fail(SF_ERR_UNSUPPORTED, "%s: 16-bit dtypes only", name);
  if (!(scale >= -1.0e30f && scale <= 1.0e30f))
    return fail(SF_ERR_INVALID_ARG, "%s: the scale must be finite (at most 1e30 in size)", name);
  int rc = window_operand(name, "Q", Q, ldq, strideQ, headQ, a.D);
  if (rc == SF_OK) rc = window_operand(name, "K", K, ldk, strideK, headK, a.D);
  if (rc == SF_OK) rc = window_operand(name, "V", V, ldv, strideV, headV, a.D);
  if (rc == SF_OK) rc = window_operand(name, "O", O, ldo, strideO, headO, a.D);
  if (rc != SF_OK) return rc;
  a.Q = Q, a.ldq = ldq, a.sQ = strideQ, a.hQ = headQ;
  a.K = K, a.ldk = ldk, a.sK = strideK, a.hK = headK;
  a.V = V, a.ldv = ldv, a.sV = strideV, a.hV = headV;
  a.O = O, a.ldo = ldo, a.sO = strideO, a.hO = headO;
  a.scale = scale;
  return SF_OK;
}

static void window_shape(WinShape& a, int64_t batch, int64_t heads, int64_t kv_heads, int64_t rows, int64_t capacity,
                         int64_t D, int64_t window, int64_t sinks) {
  a = WinShape{};
  a.batch = batch, a.heads = heads, a.kv_heads = kv_heads;
  a.Sq = rows, a.Sk = capacity, a.D = D;
  a.window = window < kMostRows ? window : 0;  // past any position: none
  a.sinks = sinks < kMostRows ? sinks : kMostRows;
}

}  // namespace sf

using namespace sf;

extern "C" {

int sf_qk_norm_rope(const void* x, int64_t ldx, void* q, int64_t ldq, int64_t strideQ, void* k, int64_t ldk,
                    int64_t strideK, void* v, int64_t ldv, int64_t strideV, const float* table, int64_t table_rows,
                    int64_t rot, const int32_t* positions, const int32_t* lengths, int64_t capacity,
                    const void* weight, const void* bias, sf_norm norm, float eps, int interleaved, int64_t batch,
                    int64_t rows, int64_t heads, int64_t kv_heads, int64_t D, sf_dtype dtype, void* stream) {
  clear_error();
  const char* name = "sf_qk_norm_rope";
  const int rc = norm_rope_check(name, table, table_rows, rot, norm, eps, batch, rows, heads, kv_heads, D, dtype);
  if (rc != SF_OK || batch == 0 || rows == 0) return rc;
  if (x == nullptr || q == nullptr || k == nullptr) return fail(SF_ERR_INVALID_ARG, "%s: null pointer", name);
  if (ldx < (heads + (v != nullptr ? 2 : 1) * kv_heads) * D || ldq < heads * D || ldk < kv_heads * D ||
      (v != nullptr && ldv < kv_heads * D))
    return fail(SF_ERR_INVALID_ARG, "%s: a row is shorter than its heads", name);
  if (strideQ < 0 || strideK < 0 || strideV < 0) return fail(SF_ERR_INVALID_ARG, "%s: negative stride", name);
  if (capacity < 0 || capacity > kMostRows) return fail(SF_ERR_INVALID_ARG, "%s: capacity out of range", name);
  if (lengths != nullptr && capacity > 0) {  // a row would be written while another wave has yet to read it
    const int size = dtype == SF_F32 ? 4 : 2;
    const __int128 nx = static_cast<__int128>(batch * rows - 1) * ldx + (heads + (v != nullptr ? 2 : 1) * kv_heads) * D;
    const auto extent = [&](int64_t ld, int64_t stride) {
      return static_cast<__int128>(batch - 1) * stride + static_cast<__int128>(capacity - 1) * ld + kv_heads * D;
    };
    if (ranges_meet(x, nx, k, extent(ldk, strideK), size) ||
        (v != nullptr && ranges_meet(x, nx, v, extent(ldv, strideV), size)))
      return fail(SF_ERR_INVALID_ARG, "%s: with lengths, k and v may not overlap x", name);
  }
  NormRopeArgs a;
  norm_rope_fill(a, x, ldx, table, table_rows, rot, positions, weight, norm, eps, interleaved, batch, rows, heads,
                 kv_heads, D);
  a.q = q, a.ldq = ldq, a.sq = strideQ;
  a.k = k, a.ldk = ldk, a.sk = strideK;
  a.v = v, a.ldv = ldv, a.sv = strideV;
  a.lengths = lengths;
  a.capacity = capacity;
  a.bias = bias;
  return launch_norm_rope(a, dtype, false, static_cast<hipStream_t>(stream));
}

int sf_qk_norm_rope_plan(int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads, int64_t D, int64_t rot,
                         int values, int backward, char* buf, int len) {
  clear_error();
  const char* name = "sf_qk_norm_rope_plan";
  if (buf == nullptr || len <= 0) return fail(SF_ERR_INVALID_ARG, "%s: bad buffer", name);
  buf[0] = 0;
  const float none = 0.0f;  // stands for the table
  const int rc = norm_rope_check(name, &none, 1, rot, SF_NORM_RMS, 0.0f, batch, rows, heads, kv_heads, D, SF_BF16);
  if (rc != SF_OK) return rc;
  if (batch == 0 || rows == 0) {
    snprintf(buf, static_cast<size_t>(len), "noop");
    return SF_OK;
  }
  NormRopeArgs a;
  norm_rope_fill(a, nullptr, 0, nullptr, 0, rot, nullptr, nullptr, SF_NORM_RMS, 0.0f, 0, batch, rows, heads, kv_heads, D);
  a.v = values != 0 || backward != 0 ? buf : nullptr;  // not followed
  const NormRopePlan p = norm_rope_plan(a, backward != 0);
  snprintf(buf, static_cast<size_t>(len), "chunks of %d, %u workgroups", p.chunk, p.blocks);
  return SF_OK;
}

int64_t sf_qk_norm_rope_backward_work(int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads, int64_t D,
                                      int64_t rot) {
  if (batch < 1 || rows < 1 || heads < 1 || kv_heads < 1 || D < 1 || D > 256 || rot < 0 || rot > D || (rot & 1) ||
      heads > 4096 || kv_heads > 4096 || rows > kMostRows / batch)
    return 0;
  return norm_rope_work(batch, rows, (int)heads, (int)kv_heads, (int)D, (int)rot);
}

int sf_qk_norm_rope_backward(const void* grad, const void* x, const float* table, int64_t table_rows, int64_t rot,
                             const int32_t* positions, const void* weight, sf_norm norm, float eps, int interleaved,
                             void* grad_x, void* grad_weight, void* grad_bias, int64_t batch, int64_t rows,
                             int64_t heads, int64_t kv_heads, int64_t D, sf_dtype dtype, void* work, void* stream) {
  clear_error();
  const char* name = "sf_qk_norm_rope_backward";
  const int rc = norm_rope_check(name, table, table_rows, rot, norm, eps, batch, rows, heads, kv_heads, D, dtype);
  if (rc != SF_OK) return rc;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (batch == 0 || rows == 0) {
    const size_t bytes = static_cast<size_t>(2 * D) * (dtype == SF_F32 ? 4 : 2);
    int z = grad_weight != nullptr ? launch_zero(grad_weight, bytes, st) : SF_OK;
    if (z == SF_OK && grad_bias != nullptr) z = launch_zero(grad_bias, bytes, st);
    return z;
  }
  const bool sums = grad_weight != nullptr || grad_bias != nullptr;
  if (grad == nullptr || x == nullptr || grad_x == nullptr || (sums && work == nullptr))
    return fail(SF_ERR_INVALID_ARG, "%s: null pointer", name);
  NormRopeArgs a;
  const int64_t ld = (heads + 2 * kv_heads) * D;
  norm_rope_fill(a, x, ld, table, table_rows, rot, positions, weight, norm, eps, interleaved, batch, rows, heads,
                 kv_heads, D);
  a.g = grad, a.ldg = ld;
  a.q = grad_x, a.ldq = ld;
  a.v = grad_x;  // the values' gradient goes through
  a.capacity = rows;
  a.dw = grad_weight, a.db = grad_bias;
  a.part = sums ? static_cast<float*>(work) : nullptr;
  return launch_norm_rope(a, dtype, true, st);
}

int sf_window_attention(const void* Q, int64_t ldq, int64_t strideQ, int64_t headQ, const void* K, int64_t ldk,
                        int64_t strideK, int64_t headK, const void* V, int64_t ldv, int64_t strideV, int64_t headV,
                        void* O, int64_t ldo, int64_t strideO, int64_t headO, float* lse, const int32_t* lengths,
                        int64_t batch, int64_t heads, int64_t kv_heads, int64_t rows, int64_t D, int64_t window,
                        int64_t sinks, float scale, sf_dtype dtype, void* stream) {
  clear_error();
  const char* name = "sf_window_attention";
  bool noop;
  int rc = window_sizes(name, batch, heads, kv_heads, rows, rows, D, window, sinks, &noop);
  if (rc != SF_OK || noop) return rc;
  WinShape a;
  window_shape(a, batch, heads, kv_heads, rows, rows, D, window, sinks);
  rc = window_fill(name, a, Q, ldq, strideQ, headQ, K, ldk, strideK, headK, V, ldv, strideV, headV, O, ldo, strideO,
                   headO, scale, dtype);
  if (rc != SF_OK) return rc;
  a.lse = lse;
  a.lengths = lengths;
  return launch_window(a, dtype, nullptr, static_cast<hipStream_t>(stream));
}

int64_t sf_window_attention_backward_work(int64_t batch, int64_t heads, int64_t kv_heads, int64_t rows, int64_t D,
                                          int64_t window, int64_t sinks) {
  bool noop;
  if (window_sizes("", batch, heads, kv_heads, rows, rows, D, window, sinks, &noop) != SF_OK || noop) {
    clear_error();
    return 0;
  }
  WinShape a;
  window_shape(a, batch, heads, kv_heads, rows, rows, D, window, sinks);
  return win_back_work(a);
}

int sf_window_attention_backward(const void* dO, int64_t lddo, int64_t strideDO, int64_t headDO, const void* Q,
                                 int64_t ldq, int64_t strideQ, int64_t headQ, const void* K, int64_t ldk,
                                 int64_t strideK, int64_t headK, const void* V, int64_t ldv, int64_t strideV,
                                 int64_t headV, const void* O, int64_t ldo, int64_t strideO, int64_t headO,
                                 const float* lse, const int32_t* lengths, void* dQ, int64_t lddq, int64_t strideDQ,
                                 int64_t headDQ, void* dK, int64_t lddk, int64_t strideDK, int64_t headDK, void* dV,
                                 int64_t lddv, int64_t strideDV, int64_t headDV, int64_t batch, int64_t heads,
                                 int64_t kv_heads, int64_t rows, int64_t D, int64_t window, int64_t sinks, float scale,
                                 sf_dtype dtype, void* work, void* stream) {
  clear_error();
  const char* name = "sf_window_attention_backward";
  bool noop;
  int rc = window_sizes(name, batch, heads, kv_heads, rows, rows, D, window, sinks, &noop);
  if (rc != SF_OK || noop) return rc;
  WinShape a;
  window_shape(a, batch, heads, kv_heads, rows, rows, D, window, sinks);
  rc = window_fill(name, a, Q, ldq, strideQ, headQ, K, ldk, strideK, headK, V, ldv, strideV, headV,
                   const_cast<void*>(O), ldo, strideO, headO, scale, dtype);
  if (rc == SF_OK) rc = window_operand(name, "dO", dO, lddo, strideDO, headDO, D);
  if (rc == SF_OK) rc = window_operand(name, "dQ", dQ, lddq, strideDQ, headDQ, D);
  if (rc == SF_OK) rc = window_operand(name, "dK", dK, lddk, strideDK, headDK, D);
  if (rc == SF_OK) rc = window_operand(name, "dV", dV, lddv, strideDV, headDV, D);
  if (rc != SF_OK) return rc;
  if (lse == nullptr || work == nullptr) return fail(SF_ERR_INVALID_ARG, "%s: null pointer (lse or work)", name);
  if (!aligned16(work)) return fail(SF_ERR_INVALID_ARG, "%s: work must be 16-byte aligned", name);
  a.lse = const_cast<float*>(lse);
  a.lengths = lengths;
  WinBack g;
  g.dO = dO, g.ldg = lddo, g.sG = strideDO, g.hG = headDO;
  g.dQ = dQ, g.lddq = lddq, g.sDQ = strideDQ, g.hDQ = headDQ;
  g.dK = dK, g.lddk = lddk, g.sDK = strideDK, g.hDK = headDK;
  g.dV = dV, g.lddv = lddv, g.sDV = strideDV, g.hDV = headDV;
  return launch_window_back(a, g, dtype, work, static_cast<hipStream_t>(stream));
}

int64_t sf_window_attention_cached_work(int64_t batch, int64_t heads, int64_t kv_heads, int64_t rows, int64_t capacity,
                                        int64_t D, int64_t window, int64_t sinks) {
  bool noop;
  if (window_sizes("", batch, heads, kv_heads, rows, capacity, D, window, sinks, &noop) != SF_OK || noop ||
      capacity == 0) {
    clear_error();
    return 0;
  }
  WinShape a;
  window_shape(a, batch, heads, kv_heads, rows, capacity, D, window, sinks);
  return win_cached_work(a);
}

int sf_window_attention_cached(const void* Q, int64_t ldq, int64_t strideQ, int64_t headQ, const void* K, int64_t ldk,
                               int64_t strideK, int64_t headK, const void* V, int64_t ldv, int64_t strideV,
                               int64_t headV, void* O, int64_t ldo, int64_t strideO, int64_t headO,
                               const int32_t* lengths, int64_t batch, int64_t heads, int64_t kv_heads, int64_t rows,
                               int64_t capacity, int64_t D, int64_t window, int64_t sinks, float scale, sf_dtype dtype,
                               void* work, void* stream) {
  clear_error();
  const char* name = "sf_window_attention_cached";
  bool noop;
  int rc = window_sizes(name, batch, heads, kv_heads, rows, capacity, D, window, sinks, &noop);
  if (rc != SF_OK || noop) return rc;
  if (capacity == 0) return fail(SF_ERR_INVALID_ARG, "%s: a cache without rows", name);
  WinShape a;
  window_shape(a, batch, heads, kv_heads, rows, capacity, D, window, sinks);
  rc = window_fill(name, a, Q, ldq, strideQ, headQ, K, ldk, strideK, headK, V, ldv, strideV, headV, O, ldo, strideO,
                   headO, scale, dtype);
  if (rc != SF_OK) return rc;
  if (lengths == nullptr || (work == nullptr && win_cached_work(a) > 0))
    return fail(SF_ERR_INVALID_ARG, "%s: null pointer (lengths or work)", name);
  if (!aligned16(work)) return fail(SF_ERR_INVALID_ARG, "%s: work must be 16-byte aligned", name);
  a.lengths = lengths;
  a.cached = 1;
  return launch_window(a, dtype, static_cast<float*>(work), static_cast<hipStream_t>(stream));
}

int sf_window_attention_plan(int64_t batch, int64_t heads, int64_t kv_heads, int64_t rows, int64_t capacity, int64_t D,
                             int64_t window, int64_t sinks, char* buf, int len) {
  clear_error();
  const char* name = "sf_window_attention_plan";
  if (buf == nullptr || len <= 0) return fail(SF_ERR_INVALID_ARG, "%s: bad buffer", name);
  buf[0] = 0;
  bool noop;
  const int rc = window_sizes(name, batch, heads, kv_heads, rows, capacity, D, window, sinks, &noop);
  if (rc != SF_OK) return rc;
  const size_t n = static_cast<size_t>(len);
  if (noop) {
    snprintf(buf, n, "noop");
    return SF_OK;
  }
  WinShape a;
  window_shape(a, batch, heads, kv_heads, rows, capacity > 0 ? capacity : rows, D, window, sinks);
  a.cached = capacity > 0;
  const WinPlan p = win_plan(a);
  if (p.parts > 0) snprintf(buf, n, "window split %d, heads up to %d", p.parts, p.width);
  else snprintf(buf, n, "window %d rows, heads up to %d", p.few ? 64 : 128, p.width);
  return SF_OK;
}

int sf_gated_linear(const void* x, const void* W, const void* bias, void* y, void* pre, int64_t M, int64_t F, int64_t K,
                    sf_dtype dtype, sf_epilogue act, void* stream) {
  clear_error();
  const char* name = "sf_gated_linear";
  int rc = gated_check(name, M, F, K, dtype, act);
  if (rc != SF_OK || M == 0 || F == 0) return rc;
  if (y == nullptr || (K > 0 && (x == nullptr || W == nullptr)) || (dtype == SF_F32 && pre == nullptr))
    return fail(SF_ERR_INVALID_ARG, "%s: null pointer", name);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype != SF_F32) return gated16(x, W, bias, y, pre, M, F, K, dtype, act, st);
  if (gated_few32(x, W, M, F, K)) return launch_gated_skinny32(x, W, bias, y, pre, M, F, K, epi_act(act), st);
  rc = sf_gemm(0, 1, M, 2 * F, K, 1, x, K > 0 ? K : 1, 0, W, K > 0 ? K : 1, 0, pre, 2 * F, 0, SF_F32, SF_F32, 1.0f,
               bias, bias != nullptr ? SF_EPI_BIAS : SF_EPI_NONE, stream);
  if (rc != SF_OK) return rc;
  return launch_gate(epi_act(act), false, nullptr, pre, y, M, F, dtype, st);
}

int sf_gated_linear_plan(const void* x, const void* W, int64_t M, int64_t F, int64_t K, sf_dtype dtype, char* buf,
                         int len) {
  clear_error();
  const char* name = "sf_gated_linear_plan";
  if (buf == nullptr || len <= 0) return fail(SF_ERR_INVALID_ARG, "%s: bad buffer", name);
  buf[0] = 0;
  int rc = gated_check(name, M, F, K, dtype, SF_EPI_NONE);
  if (rc != SF_OK) return rc;
  const size_t n = static_cast<size_t>(len);
  if (M == 0 || F == 0) {
    snprintf(buf, n, "noop");
  } else if (dtype == SF_F32) {
    snprintf(buf, n, "gated fp32 %s", gated_few32(x, W, M, F, K) ? "16 rows" : "product, then gate");
  } else {
    GatedPlan g;
    rc = gated_plan(name, x, W, M, F, K, g);
    if (rc != SF_OK) return rc;
    const bool staged = g.cfg == TILE_RAG_128 || g.cfg == TILE_RAG_64;
    char quarters[32] = "";
    if (g.head < g.tiles) snprintf(quarters, sizeof(quarters), ", %lld quartered", (long long)(g.tiles - g.head));
    snprintf(buf, n, "gated %dx%d%s%s%s", g.bm, g.bn, staged ? " staged" : "", g.persist ? " persistent" : "", quarters);
  }
  return SF_OK;
}

int64_t sf_gated_backward_work(int64_t M, int64_t F) {
  if (M < 1 || F < 1 || M > kMostRows || F > kMostRows / 2) return 0;
  return gate_sums_work(M, F);
}

int sf_gated_backward(const void* grad, const void* pre, void* grad_pre, void* grad_bias, int64_t M, int64_t F,
                      sf_dtype dtype, sf_epilogue act, void* work, void* stream) {
  clear_error();
  const char* name = "sf_gated_backward";
  const int rc = gated_check(name, M, F, 0, dtype, act);
  if (rc != SF_OK || F == 0) return rc;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (M == 0) return grad_bias == nullptr ? SF_OK
                     : launch_zero(grad_bias, static_cast<size_t>(2 * F) * (dtype == SF_F32 ? 4 : 2), st);
  if (grad == nullptr || pre == nullptr || grad_pre == nullptr || (grad_bias != nullptr && work == nullptr))
    return fail(SF_ERR_INVALID_ARG, "%s: null pointer", name);
  if (grad_bias == nullptr) return launch_gate(epi_act(act), true, grad, pre, grad_pre, M, F, dtype, st);
  return launch_gate_sums(epi_act(act), grad, pre, grad_pre, grad_bias, static_cast<float*>(work), M, F, dtype, st);
}

}  // extern "C"
