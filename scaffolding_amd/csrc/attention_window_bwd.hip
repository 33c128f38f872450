// attention_window_bwd.hip — launcher of attention_window_bwd.hpp's kernels.
#include "sf_internal.hpp"
#include "attention_window_bwd.hpp"

namespace sf {

static int64_t cdiv64(int64_t a, int64_t b) { return (a + b - 1) / b; }
static int win_width(int64_t D) { return D <= 64 ? 64 : (D <= 96 ? 96 : 128); }

// Ranges of win_dkv_kernel's work: one a CU (its eight waves fill it), but at
// least 4 products a range on average (each leaves at most 2 sums to be added).
// All three launches, us, for at least 8 / 4 / 2: 2 x 20 rows of 3 + 1 heads
// 27 / 23 / 20, 1024 of 8 + 8, window 256, 73 / 61 / 61, 512 of 16 + 4 60 / 62 /
// 81.
static int64_t win_ranges(const WinShape& a) {
  const int64_t blocks = cdiv64(a.Sk, 128), G = a.heads / a.kv_heads;
  const int64_t seen = a.window > 0 && a.window + 127 < a.Sq ? a.window + 127 : a.Sq;
  const int64_t products = a.batch * a.kv_heads * blocks * (cdiv64(seen, 64) + 1) * G;  // at most, but for the sinks'
  int64_t n = cu_count_current();
  if (n > products / 4) n = products / 4;
  return n < 1 ? 1 : n;
}

static int64_t round256(int64_t n) { return cdiv64(n, 256) * 256; }
static size_t part_floats(int64_t D) { return static_cast<size_t>(2 * 128) * win_width(D); }

// The rows' statistics, the ranges' starts, their sums.
int64_t win_back_work(const WinShape& a) {
  const int64_t n = win_ranges(a);
  return round256(2 * a.batch * a.heads * a.Sq * 4) + round256((n + 1) * static_cast<int64_t>(sizeof(WinStart))) +
         2 * n * static_cast<int64_t>(part_floats(a.D) * sizeof(float));
}

template <typename T, int DW>
static int launch_win_back_t(const WinBackParams& p, hipStream_t st) {
  hipLaunchKernelGGL((win_dq_kernel<T, DW>), dim3((unsigned)((int64_t)p.w.B * p.w.H * p.w.QB + 1)), dim3(256), 0, st, p);
  int rc = check_launch("window attention gradient (queries)");
  if (rc != SF_OK) return rc;
  hipLaunchKernelGGL((win_dkv_kernel<T, DW>), dim3((unsigned)p.ranges), dim3(512), 0, st, p);
  rc = check_launch("window attention gradient (keys)");
  if (rc != SF_OK || p.ranges == 1) return rc;
  hipLaunchKernelGGL((win_dkv_merge_kernel<T, DW>), dim3((unsigned)(2 * p.ranges)), dim3(512), 0, st, p);
  return check_launch("window attention gradient (merge)");
}

int launch_window_back(const WinShape& a, const WinBack& g, sf_dtype dt, void* work, hipStream_t st) {
  WinBackParams p{};
  win_fill_params(a, p.w);
  p.dO = g.dO, p.ldg = (int)g.ldg, p.sG = g.sG, p.hG = g.hG;
  p.dQ = g.dQ, p.lddq = (int)g.lddq, p.sDQ = g.sDQ, p.hDQ = g.hDQ;
  p.dK = g.dK, p.lddk = (int)g.lddk, p.sDK = g.sDK, p.hDK = g.hDK;
  p.dV = g.dV, p.lddv = (int)g.lddv, p.sDV = g.sDV, p.hDV = g.hDV;
  p.scale = a.scale;
  p.KBS = (int)cdiv64(a.Sk, 128);
  p.ranges = (int)win_ranges(a);
  p.stat = static_cast<float*>(work);
  char* at = static_cast<char*>(work) + round256(2 * a.batch * a.heads * a.Sq * 4);
  p.start = reinterpret_cast<WinStart*>(at);
  p.ws = reinterpret_cast<float*>(at + round256((p.ranges + 1) * static_cast<int64_t>(sizeof(WinStart))));
  const bool h = dt == SF_F16;
  switch (win_width(a.D)) {
    case 64: return h ? launch_win_back_t<F16, 64>(p, st) : launch_win_back_t<BF16, 64>(p, st);
    case 96: return h ? launch_win_back_t<F16, 96>(p, st) : launch_win_back_t<BF16, 96>(p, st);
  }
  return h ? launch_win_back_t<F16, 128>(p, st) : launch_win_back_t<BF16, 128>(p, st);
}

}  // namespace sf
