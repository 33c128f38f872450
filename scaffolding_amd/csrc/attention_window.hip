// attention_window.hip — launchers of attention_window.hpp's kernels.
#include "sf_internal.hpp"
#include "attention_window.hpp"

namespace sf {

static int win_width(int64_t D) { return D <= 64 ? 64 : (D <= 96 ? 96 : 128); }

static int64_t cdiv64(int64_t a, int64_t b) { return (a + b - 1) / b; }

void win_fill_params(const WinShape& a, WinParams& p) {
  p = WinParams{};
  p.Q = a.Q, p.K = a.K, p.V = a.V, p.O = a.O;
  p.lse = a.lse;
  p.lengths = a.lengths;
  p.sQ = a.sQ, p.sK = a.sK, p.sV = a.sV, p.sO = a.sO;
  p.hQ = a.hQ, p.hK = a.hK, p.hV = a.hV, p.hO = a.hO;
  p.ldq = (int)a.ldq, p.ldk = (int)a.ldk, p.ldv = (int)a.ldv, p.ldo = (int)a.ldo;
  p.B = (int)a.batch, p.H = (int)a.heads, p.Hk = (int)a.kv_heads, p.G = p.H / p.Hk;
  p.Sq = (int)a.Sq, p.Sk = (int)a.Sk, p.D = (int)a.D;
  p.window = a.window > 0 && a.window < (1 << 30) ? (int)a.window : 1 << 30;
  p.sinks = a.sinks < (1 << 30) ? (int)a.sinks : 1 << 30;
  p.cached = a.cached;
  p.QB = (int)cdiv64(a.Sq, WinCfg<64>::ROWS);
  p.scale_log2e = a.scale * 1.4426950408889634f;
}

// The key ranges of win_split_kernel, or 0 where whole rows of 128 queries are
// the better choice.  Estimated us: a workgroup of the split kernel (one a CU
// at head sizes past 64, else two) takes 3 and 2.6 per four blocks of 32 keys
// (its share of the memory's rate), the merge 3; one of win_attn_kernel (two a
// CU, 128 rows) 5 and 1 per block of 64 keys.  Both sides measured over 216 caches
// (1, 8, 32 sequences of 256 to 4096 tokens, 1 to 64 new ones, 8 or 32 heads of 64
// and 128 on 1 to 8 key heads): the choice is within 6 % of the better one in 153
// and within 30 % in 207.  It misses where several row blocks share a key head,
// whose keys the second one finds in L2 while the estimate counts them again: 16
// tokens over 32 x 4096, 32 heads of 64 on one, take 167 us in whole rows and 54
// split.  The other way by at most 29 %: 16 tokens over 8 x 1024, 32 heads of 64 on
// 8, 18.8 us in two ranges, 14.5 in workgroups of 64 rows.
static int win_split_parts(const WinShape& a, int cus) {
  const int64_t G = a.heads / a.kv_heads, RB = cdiv64(a.Sq * G, 16), items = a.batch * a.kv_heads * RB;
  const int64_t W = a.window > 0 ? a.window : a.Sk;
  const int64_t keys = W + a.Sq + a.sinks < a.Sk ? W + a.Sq + a.sinks : a.Sk;
  const int64_t blocks = cdiv64(keys, 32) + 1, slots = (a.D > 64 ? 1 : 2) * cus;
  const double whole = (double)cdiv64(a.batch * a.heads * cdiv64(a.Sq, WinCfg<64>::ROWS), 2 * cus) *
                       (5.0 + 1.0 * (double)cdiv64(keys, 64));
  double best = whole;
  int parts = 0;
  // (workgroups of 256 threads: a launch holds fewer than 2^32; the merge takes
  // up to four an item)
  for (int64_t q = 1; q <= 64 && (q == 1 || 8 * q <= blocks) && items * (q > 4 ? q : 4) < (int64_t(1) << 24); ++q) {
    const double us = (double)cdiv64(items * q, slots) * (3.0 + 2.6 * (double)cdiv64(blocks, 4 * q)) +
                      (q > 1 ? 3.0 + 0.05 * (double)q : 0.0);
    if (us < best) {
      best = us;
      parts = (int)q;
    }
  }
  return parts;
}

static size_t win_part_floats(int64_t D) {
  switch (win_width(D)) {
    case 64: return WinSplitCfg<64>::PART;
    case 96: return WinSplitCfg<96>::PART;
  }
  return WinSplitCfg<128>::PART;
}

int64_t win_cached_work(const WinShape& a) {
  const int parts = win_split_parts(a, cu_count_current());
  if (parts < 2) return 0;
  return a.batch * a.kv_heads * cdiv64(a.Sq * (a.heads / a.kv_heads), 16) * parts *
         (int64_t)(win_part_floats(a.D) * sizeof(float));
}

template <typename T, int DW, bool FEW>
static int launch_win_rows(const WinParams& p, hipStream_t st) {
  const dim3 g((unsigned)((int64_t)p.B * p.H * p.QB));
  if (p.lse != nullptr) hipLaunchKernelGGL((win_attn_kernel<T, DW, true, FEW>), g, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((win_attn_kernel<T, DW, false, FEW>), g, dim3(256), 0, st, p);
  return check_launch("window attention");
}

template <typename T, int DW>
static int launch_win(const WinParams& p, int parts, bool few, hipStream_t st) {
  if (parts > 0) {
    const int64_t items = (int64_t)p.B * p.Hk * p.RB;
    hipLaunchKernelGGL((win_split_kernel<T, DW>), dim3((unsigned)(items * parts)), dim3(256), 0, st, p);
    int rc = check_launch("window attention (split)");
    if (rc != SF_OK || parts == 1) return rc;
    hipLaunchKernelGGL((win_merge_kernel<T, DW>), dim3((unsigned)(items * (DW / 32))), dim3(256), 0, st, p);
    return check_launch("window attention (merge)");
  }
  return few ? launch_win_rows<T, DW, true>(p, st) : launch_win_rows<T, DW, false>(p, st);
}

WinPlan win_plan(const WinShape& a) {
  const int cus = cu_count_current();
  const int64_t halves = a.batch * a.heads * cdiv64(a.Sq, WinCfg<64, true>::ROWS);
  return {win_width(a.D), a.cached ? win_split_parts(a, cus) : 0, halves <= (a.D > 64 ? 1 : 2) * cus};
}

int launch_window(const WinShape& a, sf_dtype dt, float* ws, hipStream_t st) {
  WinParams p;
  win_fill_params(a, p);
  const WinPlan plan = win_plan(a);
  const int parts = plan.parts;
  const bool few = plan.few;
  if (a.cached) {
    p.parts = parts;
    p.RB = (int)cdiv64(a.Sq * p.G, 16);
    p.ws = ws;
  }
  if (few) p.QB = (int)cdiv64(a.Sq, WinCfg<64, true>::ROWS);
  const bool h = dt == SF_F16;
  switch (plan.width) {
    case 64: return h ? launch_win<F16, 64>(p, parts, few, st) : launch_win<BF16, 64>(p, parts, few, st);
    case 96: return h ? launch_win<F16, 96>(p, parts, few, st) : launch_win<BF16, 96>(p, parts, few, st);
  }
  return h ? launch_win<F16, 128>(p, parts, few, st) : launch_win<BF16, 128>(p, parts, few, st);
}

}  // namespace sf
