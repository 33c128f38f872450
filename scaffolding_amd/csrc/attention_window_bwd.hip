// attention_window_bwd.hip — launcher of attention_window_bwd.hpp's kernels.
#include "sf_internal.hpp"
#include "attention_window_bwd.hpp"

namespace sf {

static int64_t cdiv64(int64_t a, int64_t b) { return (a + b - 1) / b; }
static int win_width(int64_t D) { return D <= 64 ? 64 : (D <= 96 ? 96 : 128); }

// Which key blocks run in parts, and in how many.  A key block of 128 is seen
// by the rows up to its window's end, one with sinks by every later row: with a
// window the blocks of the sinks are cut to about the others' rows, without
// one the first half of all blocks is cut in two.
static void win_cut(const WinShape& a, int* heavy, int* parts) {
  const int64_t blocks = cdiv64(a.Sk, 128), seen = a.window > 0 && a.window + 127 < a.Sq ? a.window + 127 : a.Sq;
  *heavy = 0;
  *parts = 1;
  if (seen < a.Sq) {
    const int64_t most = cdiv64(a.Sq, seen + 128);
    if (a.sinks > 0 && most > 1) {
      const int64_t with = cdiv64(a.sinks, 128);
      *heavy = (int)(with < blocks ? with : blocks);
      *parts = (int)(most < 16 ? most : 16);
    }
  } else if (blocks > 1) {
    *heavy = (int)(blocks / 2);
    *parts = 2;
  }
}

static size_t part_floats(int64_t D) { return static_cast<size_t>(2 * 128) * win_width(D); }

int64_t win_back_work(const WinShape& a) {
  int heavy, parts;
  win_cut(a, &heavy, &parts);
  const int64_t stats = cdiv64(a.batch * a.heads * a.Sq * 4, 256) * 256;
  return stats + (heavy > 0 ? a.batch * a.kv_heads * heavy * parts * (int64_t)(part_floats(a.D) * sizeof(float)) : 0);
}

template <typename T, int DW>
static int launch_win_back_t(const WinBackParams& p, hipStream_t st) {
  hipLaunchKernelGGL((win_dq_kernel<T, DW>), dim3((unsigned)((int64_t)p.w.B * p.w.H * p.w.QB)), dim3(256), 0, st, p);
  int rc = check_launch("window attention gradient (queries)");
  if (rc != SF_OK) return rc;
  const int64_t kv = (int64_t)p.w.B * p.w.Hk;
  hipLaunchKernelGGL((win_dkv_kernel<T, DW>), dim3((unsigned)(kv * (p.heavy * p.parts + p.KBS - p.heavy))), dim3(256), 0,
                     st, p);
  rc = check_launch("window attention gradient (keys)");
  if (rc != SF_OK || p.heavy == 0) return rc;
  hipLaunchKernelGGL((win_dkv_merge_kernel<T, DW>), dim3((unsigned)(kv * p.heavy)), dim3(256), 0, st, p);
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
  win_cut(a, &p.heavy, &p.parts);
  if (a.batch * a.kv_heads * ((int64_t)p.heavy * p.parts + p.KBS) > (int64_t(1) << 30))
    return fail(SF_ERR_UNSUPPORTED, "window attention gradient: more than 2^30 workgroups");
  p.delta = static_cast<float*>(work);
  p.ws = p.delta + cdiv64(a.batch * a.heads * a.Sq * 4, 256) * 64;
  const bool h = dt == SF_F16;
  switch (win_width(a.D)) {
    case 64: return h ? launch_win_back_t<F16, 64>(p, st) : launch_win_back_t<BF16, 64>(p, st);
    case 96: return h ? launch_win_back_t<F16, 96>(p, st) : launch_win_back_t<BF16, 96>(p, st);
  }
  return h ? launch_win_back_t<F16, 128>(p, st) : launch_win_back_t<BF16, 128>(p, st);
}

}  // namespace sf
