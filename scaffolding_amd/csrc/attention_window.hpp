// attention_window.hpp — causal attention over a sliding window and a few
// first keys ("sinks"), 16-bit operands, fp32 accumulation and softmax:
//
//   O[i] = sum_j p_ij V[j],  p_i = softmax over the j that i sees of
//   scale Q[i] . K[j];  the query at position i sees j <= i with j > i -
//   window or j < sinks, and j < the sequence's length
//
// Query head h reads key head h / (heads / kv_heads).  Two users: whole
// sequences (query i at position i) and caches (query i at lengths[b] + i).
//
// win_attn_kernel: attn_wide_kernel's scheme (attention_wide.hpp): 128 query
// rows a workgroup in four waves, blocks of 64 keys through an LDS ring by
// direct loads, S^T = K Q^T so that P stays in the lane that made it, lazily
// raised row references.  A workgroup walks the blocks that any of its rows
// sees, the sinks' first; only blocks at the edge of what a wave's rows see are
// compared key by key, and a wave leaves out those that none of its rows sees.
// Keys past the sequence's end are never read (the buffers end there), so what
// a cache holds behind it does not matter.  A NaN or infinite V that a row does
// not see meets its weight 0 in the products: rows that come out other than
// finite, or past the type's largest value, are formed again over their own keys
// (win_exact_rows).
//
// The scale is applied to the fp32 scores (attn_wide_kernel's rounding of a
// scaled Q would show in the rows' log-sums), and with the log-sums wanted a
// row's sum is that of the unrounded weights.
//
// win_split_kernel: few query rows over many keys (decoding), see there.
#pragma once

#include "gemm16nt_pp.hpp"

namespace sf {

struct WinParams {
  const void* Q;
  const void* K;
  const void* V;
  void* O;
  float* lse;          // [B, H, Sq], or NULL
  const int* lengths;  // of the sequences (caches: before the new rows), or NULL
  int64_t sQ, sK, sV, sO, hQ, hK, hV, hO;  // batch and head strides, elements
  int ldq, ldk, ldv, ldo;
  int B, H, Hk, G;     // G = H / Hk
  int Sq, Sk, D;       // Sk: rows of K and V
  int window, sinks;   // window >= 1 (2^30: none)
  int cached;
  int QB;              // row blocks of a head
  float scale_log2e;
  // win_split_kernel
  float* ws;
  int parts, RB;
};

struct WinSeq {
  int off;   // position of row 0
  int keys;  // keys of the sequence
  int rows;  // rows of it that queries stand on (the others give 0)
};
__device__ __forceinline__ WinSeq win_seq(const WinParams& p, int64_t b) {
  WinSeq s;
  int n = p.lengths != nullptr ? p.lengths[b] : p.Sk;
  n = n < 0 ? 0 : (n < p.Sk ? n : p.Sk);
  if (p.cached) {
    s.off = n;
    s.keys = n + p.Sq < p.Sk ? n + p.Sq : p.Sk;
    s.rows = p.Sq;
  } else {
    s.off = 0;
    s.keys = n;
    s.rows = n;
  }
  return s;
}

// The blocks of KB keys that rows r0 .. r1 - 1 see: `sinks` first ones, then
// from `first` on.
template <int KB>
struct WinBlocks {
  int sinks, first, n;
  __device__ __forceinline__ int at(int i) const { return i < sinks ? i : first + (i - sinks); }
};
template <int KB>
__device__ __forceinline__ WinBlocks<KB> win_blocks(const WinParams& p, const WinSeq& s, int r0, int r1) {
  WinBlocks<KB> w;
  const int end = s.off + r1 < s.keys ? s.off + r1 : s.keys;
  int lo = s.off + r0 - p.window + 1;
  lo = lo > 0 ? lo : 0;
  w.first = lo / KB;
  const int last = end > lo ? (end + KB - 1) / KB : w.first;
  const int sk = p.sinks < end ? p.sinks : end;
  const int sb = (sk + KB - 1) / KB;
  w.sinks = sb < w.first ? sb : w.first;
  w.n = w.sinks + last - w.first;
  return w;
}

// (Without branches: it stands in the middle of code that must stay in one
// piece to be scheduled.)
__device__ __forceinline__ bool win_sees(const WinParams& p, const WinSeq& s, int pos, int key) {
  return (key <= pos) & (key < s.keys) & ((key > pos - p.window) | (key < p.sinks));
}

// Workgroup -> (row block, batch entry, query head).  The last row blocks, which
// see the most keys, start first; the heads that share keys, and with eight or
// more key heads all row blocks of one, run on one XCD (its L2 holds them).
__device__ __forceinline__ void win_item(const WinParams& p, int pid, int& qb, int& b, int& h) {
  const int heads = p.B * p.H;
  const int r = pid % heads;
  qb = p.QB - 1 - pid / heads;
  const int whole = p.B * p.Hk / kNumXcd * kNumXcd;  // key heads dealt out to XCDs
  int kv, g;
  if (r < whole * p.G) {
    const int t = r / kNumXcd;
    kv = t / p.G * kNumXcd + r % kNumXcd;
    g = t % p.G;
  } else {
    const int t = r - whole * p.G;
    kv = whole + t / p.G;
    g = t % p.G;
  }
  b = kv / p.Hk;
  h = kv % p.Hk * p.G + g;
}

// One 16-bit row times another, fp32.
template <typename T>
__device__ __forceinline__ float win_dot(const uint16_t* a, const uint16_t* b, int D) {
  float dot = 0.f;
#pragma nounroll
  for (int d = 0; d < D; d += 8) {
    const u32x4 x = *reinterpret_cast<const u32x4*>(a + d), y = *reinterpret_cast<const u32x4*>(b + d);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t u = x[e], v = y[e];
      dot = __builtin_fmaf(Elem<T>::to_f32((uint16_t)(u & 0xffffu)), Elem<T>::to_f32((uint16_t)(v & 0xffffu)), dot);
      dot = __builtin_fmaf(Elem<T>::to_f32((uint16_t)(u >> 16)), Elem<T>::to_f32((uint16_t)(v >> 16)), dot);
    }
  }
  return dot;
}

// The least size that rounds to infinity in T.  A row's weights are rounded for
// their product with V and its sum is not (or held unnormalised, up to 2^8 times
// the result), so a row of values next to T's largest one can come out past it,
// which an average cannot.
template <typename T>
__device__ __forceinline__ float win_top() {
  return std::is_same<T, F16>::value ? 65520.f : __builtin_bit_cast(float, 0x7f7f8000u);
}

// Output rows term by term over their own keys alone, scores and values from
// global memory.  One wave; bit i of `rows` is the row at position pos0 + i,
// whose query and output lie at Q + i ldq and O + i ldo.  Slow, for rows
// beside values that are not finite and rows that came out past T's largest
// value: the weights are normalised ahead of their products and the terms added
// 64 at a time, so that a sum over n keys is off by at most (n / 64 + 128) 2^-24 of
// its terms' sizes (half a step of fp16 at n = 2^18).  Not inlined: it would cost
// the kernels registers.  Columns d0 .. d1 - 1 are stored.
template <typename T>
__device__ __attribute__((noinline)) void win_exact_rows(const WinParams& p, const uint16_t* Q, int64_t ldq,
                                                         uint16_t* O, int64_t ldo, const uint16_t* K,
                                                         const uint16_t* V, WinSeq s, int pos0, uint64_t rows, int d0,
                                                         int d1) {
  const int lane = threadIdx.x & 63;
  const bool dok = 2 * lane < p.D;  // lane: columns 2 lane, 2 lane + 1
  while (rows != 0) {
    const int i = __builtin_ctzll(rows);
    rows &= rows - 1;
    const int pos = pos0 + i;
    const uint16_t* q = Q + (int64_t)i * ldq;
    const int end = pos + 1 < s.keys ? pos + 1 : s.keys;
    int lo = pos - p.window + 1;
    lo = lo > 0 ? lo : 0;
    const int head = p.sinks < lo ? (p.sinks < end ? p.sinks : end) : (lo < end ? lo : end);  // keys [0, head) are sinks
    const int n = head + (end > lo ? end - lo : 0);
    auto key = [&](int t) { return t < head ? t : lo + (t - head); };
    float mx = -INFINITY;
    bool bad = false;
#pragma nounroll
    for (int t = lane; t < n; t += 64) {
      const float x = win_dot<T>(q, K + (int64_t)key(t) * p.ldk, p.D) * p.scale_log2e;
      bad |= x != x;
      mx = fmaxf(mx, x);
    }
    mx = wave_max(mx);
    bad = __builtin_amdgcn_ballot_w64(bad) != 0 || !(mx > -INFINITY) || mx == INFINITY;
    auto weight = [&](int t) {
      return __builtin_amdgcn_exp2f(win_dot<T>(q, K + (int64_t)key(t) * p.ldk, p.D) * p.scale_log2e - mx);
    };
    float a0 = bad && n > 0 ? __builtin_nanf("") : 0.f, a1 = a0;
    if (!bad) {
      float l = 0.f;
#pragma nounroll
      for (int t = lane; t < n; t += 64) l += weight(t);
      const float inv = 1.0f / wave_sum(l);
#pragma nounroll
      for (int t0 = 0; t0 < n; t0 += 64) {
        const int m = n - t0 < 64 ? n - t0 : 64;
        const float pt = lane < m ? weight(t0 + lane) * inv : 0.f;
        float b0 = 0.f, b1 = 0.f;
#pragma nounroll
        for (int u = 0; u < m; ++u) {
          const float pu = __shfl(pt, u, 64);
          const uint32_t w =
              *reinterpret_cast<const uint32_t*>(V + (int64_t)key(t0 + u) * p.ldv + (dok ? 2 * lane : 0));
          b0 = __builtin_fmaf(pu, Elem<T>::to_f32((uint16_t)(w & 0xffffu)), b0);
          b1 = __builtin_fmaf(pu, Elem<T>::to_f32((uint16_t)(w >> 16)), b1);
        }
        a0 += b0;
        a1 += b1;
      }
    }
    if (dok && 2 * lane >= d0 && 2 * lane < d1)
      *reinterpret_cast<uint32_t*>(O + (int64_t)i * ldo + 2 * lane) = pack2<T>(a0, a1);
  }
}

// FEW: where all workgroups of half the rows run at once, one a CU (two at head
// sizes up to 64): a workgroup's few blocks do not hide their loads' latency, so
// three of them are under way.  3 x 777 rows, 6 + 2 heads of 72, window 100: 10.2
// us (else 14.2); 1024 rows, 16 + 4 heads of 128: 22.6 (27.0); 4096 rows of 4 + 1:
// 73.7 (86.2).  Where twice as many would run, 25.2 instead of 20.6 (2 x 1024 rows,
// 16 + 4 heads of 128, window 200).
template <int DW, bool FEW = false>
struct WinCfg {
  static constexpr int MB = FEW ? 1 : 2;       // 16-row query blocks per wave
  static constexpr int ROWS = 4 * MB * 16;     // query rows per workgroup
  static constexpr int HALVES = (DW + 63) / 64;
  static constexpr int NS = FEW ? 4 : (DW > 64 ? 2 : 3);  // key blocks of 64 in LDS
};

template <typename T, int DW, bool LSE, bool FEW>
__global__ __launch_bounds__(256, FEW && DW > 64 ? 1 : 2) void win_attn_kernel(WinParams p) {
  using C = WinCfg<DW, FEW>;
  constexpr int MB = C::MB, HV = C::HALVES, NS = C::NS;
  constexpr int KC = DW / 32, DB = DW / 16;
  constexpr int KB = 64;
  constexpr int HB = KB * 128;  // one half of a key block
  constexpr int LPB = 4 * HV;   // direct loads per wave and key block
  constexpr float THRESH = 8.0f, UNSET = -3.0e38f;
  __shared__ __attribute__((aligned(1024))) uint8_t sK[NS][HV * HB];
  __shared__ __attribute__((aligned(1024))) uint8_t sV[NS][HV * HB];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int qb, b, h;
  win_item(p, (int)blockIdx.x, qb, b, h);
  const int hk = h / p.G;
  const WinSeq sq = win_seq(p, b);
  const int r0 = qb * C::ROWS, q0 = r0 + wave * (MB * 16);
  const int r1 = r0 + C::ROWS < sq.rows ? r0 + C::ROWS : sq.rows;
  const WinBlocks<KB> kbs = win_blocks<KB>(p, sq, r0, r1 > r0 ? r1 : r0);
  const int nkb = r1 > r0 ? kbs.n : 0;
  const uint16_t* Qb = static_cast<const uint16_t*>(p.Q) + b * p.sQ + h * p.hQ;
  const uint16_t* Kb = static_cast<const uint16_t*>(p.K) + b * p.sK + hk * p.hK;
  const uint16_t* Vb = static_cast<const uint16_t*>(p.V) + b * p.sV + hk * p.hV;
  uint16_t* Ob = static_cast<uint16_t*>(p.O) + b * p.sO + h * p.hO;

  // Loads: 16-byte chunk hch of rows drow and drow + 8 of a block, per half of
  // 64 d; chunks at or past D and rows past the last key lie outside the
  // block's buffer and read as zeros.
  const int drow = wave * 16 + (lane >> 3);
  const int hch = (lane & 7) ^ (lane >> 3);
  uint32_t vk0[HV], vv0[HV];
#pragma unroll
  for (int hf = 0; hf < HV; ++hf) {
    const int d = hf * 64 + hch * 8;
    vk0[hf] = d < p.D ? (uint32_t)drow * (uint32_t)p.ldk * 2u + (uint32_t)d * 2u : 0x80000000u;
    vv0[hf] = d < p.D ? (uint32_t)drow * (uint32_t)p.ldv * 2u + (uint32_t)d * 2u : 0x80000000u;
  }
  const uint32_t k8 = 8u * (uint32_t)p.ldk * 2u, v8 = 8u * (uint32_t)p.ldv * 2u;
  auto issue = [&](int i) {
    const int s = i % NS, j = kbs.at(i);
    const int left = sq.keys - j * KB < KB ? sq.keys - j * KB : KB;  // >= 1
    const __amdgpu_buffer_rsrc_t rK = __builtin_amdgcn_make_buffer_rsrc(
        (void*)(Kb + (int64_t)j * KB * p.ldk), (short)0, (int)(((uint32_t)(left - 1) * (uint32_t)p.ldk + (uint32_t)p.D) * 2u),
        0x00020000);
    const __amdgpu_buffer_rsrc_t rV = __builtin_amdgcn_make_buffer_rsrc(
        (void*)(Vb + (int64_t)j * KB * p.ldv), (short)0, (int)(((uint32_t)(left - 1) * (uint32_t)p.ldv + (uint32_t)p.D) * 2u),
        0x00020000);
#pragma unroll
    for (int hf = 0; hf < HV; ++hf) {
      uint8_t* k = &sK[s][0] + hf * HB + wave * 2048;
      uint8_t* v = &sV[s][0] + hf * HB + wave * 2048;
      const uint32_t ok = vk0[hf], ov = vv0[hf];
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rK, (lds_ptr_t)k, 16, ok, 0, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rK, (lds_ptr_t)(k + 1024), 16, ok + k8, 0, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rV, (lds_ptr_t)v, 16, ov, 0, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rV, (lds_ptr_t)(v + 1024), 16, ov + v8, 0, 0, 0);
    }
  };
#pragma unroll
  for (int i = 0; i < NS - 1; ++i)
    if (i < nkb) issue(i);

  u32x4 qf[MB][KC];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    int r = q0 + mb * 16 + (lane & 15);
    r = r < p.Sq ? r : p.Sq - 1;
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
      const int d0 = kc * 32 + 8 * (lane >> 4);
      qf[mb][kc] = d0 < p.D ? *reinterpret_cast<const u32x4*>(Qb + (int64_t)r * p.ldq + d0) : u32x4{0u, 0u, 0u, 0u};
    }
  }

  f32x4 o[MB][DB], osum[MB];
  float nq[MB], th[MB];  // -reference; a row is raised when one of its exponents exceeds th
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    osum[mb] = f32x4{0.f, 0.f, 0.f, 0.f};
    nq[mb] = 0.f;
    th[mb] = UNSET;
#pragma unroll
    for (int db = 0; db < DB; ++db) o[mb][db] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const uint32_t one2 = (uint32_t)Elem<T>::from_f32(1.0f) * 0x10001u;
  const u32x4 ones = u32x4{one2, one2, one2, one2};

  const uint32_t kfo = (uint32_t)((lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) << 4));
  const int vs = lane & 15, vg = lane >> 4;
  const int vrow0 = 4 * vg + (vs >> 2);
  const uint32_t vfo_base = (uint32_t)vrow0 * 128u + (uint32_t)((vs & 1) * 8);
  const int vch = (vs & 3) >> 1;
  const int vsw = vrow0 & 7;
  const int pw0 = sq.off + q0, pw1 = pw0 + MB * 16 - 1;  // positions of the wave's rows

  for (int i = 0; i < nkb; ++i) {
    const int st = i % NS, j = kbs.at(i);
    __builtin_amdgcn_sched_barrier(0);
    if (NS == 4 && i + 2 < nkb)
      __builtin_amdgcn_s_waitcnt(waitcnt_imm(2 * LPB, 0));
    else if (NS >= 3 && i + 1 < nkb)
      __builtin_amdgcn_s_waitcnt(waitcnt_imm(LPB, 0));
    else
      __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 0));
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    if (i + NS - 1 < nkb) issue(i + NS - 1);
    __builtin_amdgcn_sched_barrier(0);
    // none of the wave's rows sees a key of this block
    const int k0 = j * KB, k1 = k0 + KB - 1;
    if (k0 > pw1 || (k1 <= pw0 - p.window && k0 >= p.sinks)) continue;
    const bool edge = k1 > pw0 || k1 >= sq.keys || (k0 <= pw1 - p.window && k1 >= p.sinks);

    // ---- S = Q K^T ---------------------------------------------------------
    f32x4 s[MB][4];
    const uint32_t ka = lds_addr(&sK[st][0]) + kfo;
    auto read_k = [&](auto nb_c, u32x4 (&f)[KC]) {
      constexpr int NBK = decltype(nb_c)::value;
      static_for<KC>([&](auto kc_c) {
        constexpr int KCI = decltype(kc_c)::value;
        f[KCI] = ds_read16<(KCI >> 1) * HB + NBK * 2048>((KCI & 1) ? (ka ^ 64u) : ka);
      });
    };
    {
      u32x4 kf[KC];
      read_k(std::integral_constant<int, 0>{}, kf);
      static_for<4>([&](auto nbc) {
        constexpr int NBK = decltype(nbc)::value;
        u32x4 nk[KC];
        if constexpr (NBK < 3) {
          read_k(std::integral_constant<int, (NBK < 3 ? NBK + 1 : 0)>{}, nk);
          __builtin_amdgcn_s_waitcnt(waitcnt_imm(63, KC));
        } else {
          __builtin_amdgcn_s_waitcnt(waitcnt_imm(63, 0));
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) s[mb][NBK] = Mfma16<T>::run(kf[0], qf[mb][0], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
        for (int kc = 1; kc < KC; ++kc)
#pragma unroll
          for (int mb = 0; mb < MB; ++mb) s[mb][NBK] = Mfma16<T>::run(kf[kc], qf[mb][kc], s[mb][NBK]);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (NBK < 3) {
#pragma unroll
          for (int kc = 0; kc < KC; ++kc) kf[kc] = nk[kc];
        }
      });
    }

    // ---- V fragments of d 0-63 (they land under the softmax) ---------------
    const uint32_t va = lds_addr(&sV[st][0]) + vfo_base;
    u32x4 vf[4][2];
    auto read_v = [&](auto h_c, auto n_c) {
      constexpr int HF = decltype(h_c)::value;
      static_for<decltype(n_c)::value>([&](auto dbc) {
        constexpr int D4 = decltype(dbc)::value;
        const uint32_t a0 = va + (uint32_t)(((2 * D4 + vch) ^ vsw) << 4);
        const u32x2 t00 = ds_read_tr16<HF * HB + 0>(a0);
        const u32x2 t01 = ds_read_tr16<HF * HB + 16 * 128>(a0);
        const u32x2 t10 = ds_read_tr16<HF * HB + 32 * 128>(a0);
        const u32x2 t11 = ds_read_tr16<HF * HB + 48 * 128>(a0);
        vf[D4][0] = u32x4{t00.x, t00.y, t01.x, t01.y};
        vf[D4][1] = u32x4{t10.x, t10.y, t11.x, t11.y};
      });
    };
    __builtin_amdgcn_sched_barrier(0);
    read_v(std::integral_constant<int, 0>{}, std::integral_constant<int, 4>{});
    __builtin_amdgcn_sched_barrier(0);

    // exponents against the rows' references
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int nb = 0; nb < 4; ++nb)
#pragma unroll
        for (int q = 0; q < 4; ++q) s[mb][nb][q] = __builtin_fmaf(s[mb][nb][q], p.scale_log2e, nq[mb]);
    if (edge) {
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        const int pos = pw0 + mb * 16 + (lane & 15);
#pragma unroll
        for (int nb = 0; nb < 4; ++nb)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (!win_sees(p, sq, pos, k0 + nb * 16 + 4 * (lane >> 4) + q)) s[mb][nb][q] = -INFINITY;
      }
    }

    // ---- lazy row references -----------------------------------------------
    bool need = false;
    float lmx[MB];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      float mx = s[mb][0][0];
#pragma unroll
      for (int e = 1; e < 16; ++e) mx = __builtin_elementwise_maximum(mx, s[mb][e >> 2][e & 3]);
      lmx[mb] = mx;
      need |= mx > th[mb];
    }
    if (__builtin_amdgcn_ballot_w64(need) != 0) {
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        float mx = fmaxf(lmx[mb], __shfl_xor(lmx[mb], 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        // A row without a reference takes its first maximum (O and its sum are
        // still zero); later ones only raise it.
        const bool unset = th[mb] < 0.f, found = mx > UNSET;
        const float sub = unset ? (found ? mx : 0.f) : fmaxf(mx, 0.f);
        const float corr = unset ? 1.0f : __builtin_amdgcn_exp2f(-sub);
        nq[mb] -= sub;
        if (found) th[mb] = THRESH;
#pragma unroll
        for (int nb = 0; nb < 4; ++nb)
#pragma unroll
          for (int q = 0; q < 4; ++q) s[mb][nb][q] -= sub;
        osum[mb] *= corr;
#pragma unroll
        for (int db = 0; db < DB; ++db) o[mb][db] *= corr;
      }
    }

    // ---- P = 2^x in 16 bits, O += P V, row sums -----------------------------
    u32x4 pf[MB][2];
    auto expo = [&](int mb) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t w[4];
#pragma unroll
        for (int hh = 0; hh < 2; ++hh)
#pragma unroll
          for (int q2 = 0; q2 < 2; ++q2) {
            const float e0 = __builtin_amdgcn_exp2f(s[mb][2 * c + hh][2 * q2]);
            const float e1 = __builtin_amdgcn_exp2f(s[mb][2 * c + hh][2 * q2 + 1]);
            if constexpr (LSE) {
              osum[mb][2 * q2] += e0;
              osum[mb][2 * q2 + 1] += e1;
            }
            w[hh * 2 + q2] = pack2<T>(e0, e1);
          }
        pf[mb][c] = u32x4{w[0], w[1], w[2], w[3]};
      }
    };
    auto sums = [&](int mb) {
      if constexpr (!LSE) {
        osum[mb] = Mfma16<T>::run(ones, pf[mb][0], osum[mb]);
        osum[mb] = Mfma16<T>::run(ones, pf[mb][1], osum[mb]);
      }
    };
    auto pv = [&](int mb, auto h_c, auto n_c) {
      constexpr int HF = decltype(h_c)::value, N = decltype(n_c)::value;
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int d4 = 0; d4 < N; ++d4)
          o[mb][HF * 4 + d4] = Mfma16<T>::run(vf[d4][c], pf[mb][c], o[mb][HF * 4 + d4]);
    };
    constexpr std::integral_constant<int, 0> h0{};
    constexpr std::integral_constant<int, 4> n0{};
    expo(0);
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(63, 0));  // V fragments landed
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
    sums(0);
    pv(0, h0, n0);
    if constexpr (MB > 1) {
      expo(1);
#pragma unroll
      for (int g = 0; g < 10; ++g) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, LSE ? 4 : 3, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
      sums(1);
      pv(1, h0, n0);
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (HV > 1) {
      constexpr std::integral_constant<int, 1> h1{};
      constexpr std::integral_constant<int, DB - 4> n1{};
      read_v(h1, n1);
      __builtin_amdgcn_s_waitcnt(waitcnt_imm(63, 0));
      __builtin_amdgcn_sched_barrier(0);
      pv(0, h1, n1);
      if constexpr (MB > 1) pv(1, h1, n1);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
  }

  uint64_t odd = 0;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    float l = osum[mb][0];
    if constexpr (LSE) {
      l = (l + osum[mb][1]) + (osum[mb][2] + osum[mb][3]);
      l += __shfl_xor(l, 16, 64);
      l += __shfl_xor(l, 32, 64);
    }
    const int r = q0 + mb * 16 + (lane & 15), pos = sq.off + r;
    // a row has a key unless it is past the sequence, or its window is past the
    // cache's end and no sink is there
    const bool row = r < p.Sq, any = r < sq.rows && sq.keys > 0 && (sq.keys > pos - p.window + 1 || p.sinks > 0);
    const float inv = 1.0f / l;
    float most = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        o[mb][db][q] *= inv;
        most = __builtin_elementwise_maximum(most, __builtin_fabsf(o[mb][db][q]));
      }
    }
    uint64_t bad = __builtin_amdgcn_ballot_w64(row && any && !(most < win_top<T>()));  // NaN too
    bad |= bad >> 32;
    bad = (bad | bad >> 16) & 0xffffull;
    odd |= bad << (16 * mb);
    if (row && ((bad >> (lane & 15)) & 1) == 0) {
      uint16_t* orow = Ob + (int64_t)r * p.ldo;
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const int d = db * 16 + 4 * (lane >> 4);
        if (d < p.D)
          *reinterpret_cast<u32x2*>(orow + d) =
              any ? u32x2{pack2<T>(o[mb][db][0], o[mb][db][1]), pack2<T>(o[mb][db][2], o[mb][db][3])} : u32x2{0u, 0u};
      }
    }
    if constexpr (LSE) {
      // (log2 l - nq) ln 2: the reference and the sum's logarithm
      if (row && lane < 16)
        p.lse[((int64_t)b * p.H + h) * p.Sq + r] =
            any ? (__builtin_amdgcn_logf(l) - nq[mb]) * 0.6931471805599453f : -INFINITY;
    }
  }
  if (__builtin_expect(odd != 0, 0)) {
    const WinParams& kp = *(const WinParams*)__builtin_amdgcn_kernarg_segment_ptr();
    win_exact_rows<T>(kp, Qb + (int64_t)q0 * p.ldq, p.ldq, Ob + (int64_t)q0 * p.ldo, p.ldo, Kb, Vb, sq, pw0, odd, 0,
                      p.D);
  }
}

// ---------------------------------------------------------------------
// win_split_kernel: few query rows over many keys (decoding).
//
// The G query heads of one key head share its keys, so the rows of one product
// are G heads x the new tokens, 16 at a time (row r: token r / G, head r % G); a
// workgroup takes one such block and one range of the keys, its four waves every
// fourth block of 32 keys.  Reading K and V once is the bound, so nothing waits
// for anything but memory: each wave has its own ring of four slots (K, V, K, V
// of two blocks) and no barrier, and asks for a slot's next block as soon as it
// has read the slot, so three of four slots are always in flight (24 KB a wave,
// 96 KB a CU at head size 128).  Blocks past the wave's last one are asked for
// from an empty buffer: zeros without memory traffic, and the counts of loads in
// flight stay constant.
//
// The waves' sums are merged in LDS; with more than one range of keys (chosen so
// that the CUs are full) the ranges' sums go to `ws` and win_merge_kernel, a
// second launch, merges them in order.
// ---------------------------------------------------------------------
template <int DW>
struct WinSplitCfg {
  static constexpr int HALVES = (DW + 63) / 64;
  static constexpr int SLOT = HALVES * 4096;           // 32 keys
  static constexpr int LPB = HALVES * 4;               // direct loads per slot
  static constexpr int PART_O = DW / 16 * 64 * 4;      // floats of one part's O
  static constexpr int PART = PART_O + 32;             // and its references and sums
};

// Row r's query (and output) offset and position.
struct WinRow {
  int token, head;
};
__device__ __forceinline__ WinRow win_row(const WinParams& p, int hk, int r) {
  WinRow w;
  w.token = r / p.G;
  w.head = hk * p.G + r % p.G;
  return w;
}

// Normalises and stores 16 rows' blocks of 16 columns db0, db0 + step, ... (NB
// of them, those below DB); rows that are not below win_top are formed again
// (columns d0 .. d1 - 1, all that the workgroup stores) by wave 0.  l: the sum of
// the lane's row.
template <typename T, int DB, int NB>
__device__ __forceinline__ void win_finish_rows(const WinParams& p, const WinSeq& sq, int b, int hk, int rb, int wave,
                                                int lane, int db0, int step, int d0, int d1, const f32x4 (&o)[NB],
                                                float l, uint32_t* flag) {
  const int rows = p.Sq * p.G, r = rb * 16 + (lane & 15);
  const WinRow w = win_row(p, hk, r < rows ? r : rows - 1);
  const int pos = sq.off + w.token;
  const bool row = r < rows, any = sq.keys > 0 && (sq.keys > pos - p.window + 1 || p.sinks > 0);
  const float inv = 1.0f / l;
  float most = 0.f;
  u32x2 v[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    float x[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      x[q] = o[i][q] * inv;
      if (db0 + step * i < DB) most = __builtin_elementwise_maximum(most, __builtin_fabsf(x[q]));
    }
    v[i] = any ? u32x2{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])} : u32x2{0u, 0u};
  }
  uint64_t bad = __builtin_amdgcn_ballot_w64(row && any && !(most < win_top<T>()));  // NaN too
  bad |= bad >> 32;
  bad = (bad | bad >> 16) & 0xffffull;
  if (bad != 0 && lane == 0) __hip_atomic_fetch_or(flag, (uint32_t)bad, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  __syncthreads();
  const uint32_t odd = *flag;
  uint16_t* Ob = static_cast<uint16_t*>(p.O) + b * p.sO;
  if (row && ((odd >> (lane & 15)) & 1) == 0) {
    uint16_t* orow = Ob + (int64_t)w.token * p.ldo + w.head * p.hO;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int db = db0 + step * i, d = db * 16 + 4 * (lane >> 4);
      if (db < DB && d < p.D) *reinterpret_cast<u32x2*>(orow + d) = v[i];
    }
  }
  if (__builtin_expect(odd != 0, 0) && wave == 0) {
    const WinParams& kp = *(const WinParams*)__builtin_amdgcn_kernarg_segment_ptr();
    const uint16_t* Qb = static_cast<const uint16_t*>(p.Q) + b * p.sQ;
    const uint16_t* Kb = static_cast<const uint16_t*>(p.K) + b * p.sK + hk * p.hK;
    const uint16_t* Vb = static_cast<const uint16_t*>(p.V) + b * p.sV + hk * p.hV;
    for (int i = 0; i < 16; ++i)
      if ((odd >> i) & 1) {
        const WinRow x = win_row(p, hk, rb * 16 + i);
        win_exact_rows<T>(kp, Qb + (int64_t)x.token * p.ldq + x.head * p.hQ, 0,
                          Ob + (int64_t)x.token * p.ldo + x.head * p.hO, 0, Kb, Vb, sq, sq.off + x.token, 1, d0, d1);
      }
  }
}

template <typename T, int DW>
__global__ __launch_bounds__(256) void win_split_kernel(WinParams p) {
  using C = WinSplitCfg<DW>;
  constexpr int HV = C::HALVES, KC = DW / 32, DB = DW / 16, KB = 32, LPB = C::LPB;
  constexpr float THRESH = 8.0f, UNSET = -3.0e38f;
  __shared__ __attribute__((aligned(1024))) uint8_t ring[4][4 * C::SLOT];
  __shared__ float sm[4][16], sl[4][16];
  __shared__ uint32_t flag;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int t = (int)blockIdx.x;
  const int part = t % p.parts;
  t /= p.parts;
  const int rb = t % p.RB;
  t /= p.RB;
  const int hk = t % p.Hk, b = t / p.Hk;
  const WinSeq sq = win_seq(p, b);
  const int rows = p.Sq * p.G;
  const int t0 = rb * 16 / p.G, t1 = (rb * 16 + 15 < rows ? rb * 16 + 15 : rows - 1) / p.G;  // tokens t0 .. t1
  const WinBlocks<KB> kbs = win_blocks<KB>(p, sq, t0, t1 + 1);
  const int i0 = (int)((int64_t)kbs.n * part / p.parts), i1 = (int)((int64_t)kbs.n * (part + 1) / p.parts);
  const int cnt = i1 - i0 - wave > 0 ? (i1 - i0 - wave + 3) / 4 : 0;  // this wave's blocks
  const uint16_t* Kb = static_cast<const uint16_t*>(p.K) + b * p.sK + hk * p.hK;
  const uint16_t* Vb = static_cast<const uint16_t*>(p.V) + b * p.sV + hk * p.hV;
  if (threadIdx.x == 0) flag = 0;

  uint8_t* my = &ring[wave][0];
  const int hch = (lane & 7) ^ (lane >> 3);
  uint32_t vk0[HV], vv0[HV];
#pragma unroll
  for (int hf = 0; hf < HV; ++hf) {
    const int d = hf * 64 + hch * 8;
    vk0[hf] = d < p.D ? (uint32_t)(lane >> 3) * (uint32_t)p.ldk * 2u + (uint32_t)d * 2u : 0x80000000u;
    vv0[hf] = d < p.D ? (uint32_t)(lane >> 3) * (uint32_t)p.ldv * 2u + (uint32_t)d * 2u : 0x80000000u;
  }
  // Block u of this wave (K or V) into slot `s`; past the last: from an empty
  // buffer.
  auto issue = [&](const uint16_t* base, int ld, const uint32_t (&v0)[HV], int u, int s) {
    const int j = kbs.at(u < cnt ? i0 + wave + 4 * u : i0);
    const int left = sq.keys - j * KB < KB ? sq.keys - j * KB : KB;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        (void*)(base + (int64_t)j * KB * ld), (short)0,
        u < cnt ? (int)(((uint32_t)(left - 1) * (uint32_t)ld + (uint32_t)p.D) * 2u) : 0, 0x00020000);
    const uint32_t step = 16u * (uint32_t)ld;
#pragma unroll
    for (int hf = 0; hf < HV; ++hf) {
      uint8_t* dst = my + s * C::SLOT + hf * 4096;
      uint32_t o = v0[hf];
#pragma unroll
      for (int rr = 0; rr < 4; ++rr) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)(dst + rr * 1024), 16, o, 0, 0, 0);
        o += step;
      }
    }
  };
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    issue(Kb, p.ldk, vk0, u, 2 * u);
    issue(Vb, p.ldv, vv0, u, 2 * u + 1);
  }
  __builtin_amdgcn_sched_barrier(0);

  // Queries and positions of the lane's row.
  const int r = rb * 16 + (lane & 15);
  const WinRow w = win_row(p, hk, r < rows ? r : rows - 1);
  const uint16_t* qrow = static_cast<const uint16_t*>(p.Q) + b * p.sQ + (int64_t)w.token * p.ldq + w.head * p.hQ;
  const int pos = sq.off + w.token;
  u32x4 qf[KC];
#pragma unroll
  for (int kc = 0; kc < KC; ++kc) {
    const int d0 = kc * 32 + 8 * (lane >> 4);
    qf[kc] = d0 < p.D ? *reinterpret_cast<const u32x4*>(qrow + d0) : u32x4{0u, 0u, 0u, 0u};
  }
  // The wait for the queries would wait for every load: once, here.
  __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 63));

  f32x4 o[DB];
  float l = 0.f, nq = 0.f, th = UNSET;
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
  const uint32_t kfo = (uint32_t)((lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) << 4));
  const int vs = lane & 15, vg = lane >> 4;
  const int vrow0 = 4 * vg + (vs >> 2);
  const uint32_t vfo = (uint32_t)vrow0 * 128u + (uint32_t)((vs & 1) * 8);
  const int vch = (vs & 3) >> 1;
  const int vsw = vrow0 & 7;
  const uint32_t ra = lds_addr(my);
  const int pw0 = sq.off + t0, pw1 = sq.off + t1;

  for (int u = 0; u < cnt; ++u) {
    const int j = kbs.at(i0 + wave + 4 * u), k0 = j * KB, k1 = k0 + KB - 1;
    const uint32_t ks = ra + (uint32_t)((u & 1) * 2 * C::SLOT), vsl = ks + C::SLOT;
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(3 * LPB, 63));
    __builtin_amdgcn_sched_barrier(0);
    u32x4 kf[2][KC];
    static_for<2>([&](auto nb_c) {
      constexpr int NB = decltype(nb_c)::value;
      static_for<KC>([&](auto kc_c) {
        constexpr int KCI = decltype(kc_c)::value;
        kf[NB][KCI] = ds_read16<(KCI >> 1) * 4096 + NB * 2048>((KCI & 1) ? ((ks + kfo) ^ 64u) : ks + kfo);
      });
    });
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(63, 0));
    __builtin_amdgcn_sched_barrier(0);
    issue(Kb, p.ldk, vk0, u + 2, (u & 1) * 2);
    __builtin_amdgcn_sched_barrier(0);
    f32x4 s[2];
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
      s[nb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kc = 0; kc < KC; ++kc) s[nb] = Mfma16<T>::run(kf[nb][kc], qf[kc], s[nb]);
    }
#pragma unroll
    for (int nb = 0; nb < 2; ++nb)
#pragma unroll
      for (int q = 0; q < 4; ++q) s[nb][q] = __builtin_fmaf(s[nb][q], p.scale_log2e, nq);
    if (k1 > pw0 || k1 >= sq.keys || (k0 <= pw1 - p.window && k1 >= p.sinks)) {
#pragma unroll
      for (int nb = 0; nb < 2; ++nb)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (!win_sees(p, sq, pos, k0 + nb * 16 + 4 * (lane >> 4) + q)) s[nb][q] = -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int e = 1; e < 8; ++e) mx = __builtin_elementwise_maximum(mx, s[e >> 2][e & 3]);
    if (__builtin_amdgcn_ballot_w64(mx > th) != 0) {
      float m = fmaxf(mx, __shfl_xor(mx, 16, 64));
      m = fmaxf(m, __shfl_xor(m, 32, 64));
      const bool unset = th < 0.f, found = m > UNSET;
      const float sub = unset ? (found ? m : 0.f) : fmaxf(m, 0.f);
      const float corr = unset ? 1.0f : __builtin_amdgcn_exp2f(-sub);
      nq -= sub;
      if (found) th = THRESH;
#pragma unroll
      for (int nb = 0; nb < 2; ++nb)
#pragma unroll
        for (int q = 0; q < 4; ++q) s[nb][q] -= sub;
      l *= corr;
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] *= corr;
    }
    u32x4 pf;
#pragma unroll
    for (int nb = 0; nb < 2; ++nb)
#pragma unroll
      for (int q2 = 0; q2 < 2; ++q2) {
        const float e0 = __builtin_amdgcn_exp2f(s[nb][2 * q2]), e1 = __builtin_amdgcn_exp2f(s[nb][2 * q2 + 1]);
        l += e0 + e1;
        pf[nb * 2 + q2] = pack2<T>(e0, e1);
      }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(3 * LPB, 63));
    __builtin_amdgcn_sched_barrier(0);
    u32x4 vf[DB];
    static_for<DB>([&](auto db_c) {
      constexpr int DBI = decltype(db_c)::value;
      const uint32_t a0 = vsl + vfo + (uint32_t)(((2 * (DBI & 3) + vch) ^ vsw) << 4);
      const u32x2 x = ds_read_tr16<(DBI >> 2) * 4096>(a0), y = ds_read_tr16<(DBI >> 2) * 4096 + 16 * 128>(a0);
      vf[DBI] = u32x4{x.x, x.y, y.x, y.y};
    });
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(63, 0));
    __builtin_amdgcn_sched_barrier(0);
    issue(Vb, p.ldv, vv0, u + 2, (u & 1) * 2 + 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] = Mfma16<T>::run(vf[db], pf, o[db]);
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);

  // ---- the four waves' sums ------------------------------------------------
  __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 0));  // the last (empty) loads write zeros to this wave's ring
  f32x4* park = reinterpret_cast<f32x4*>(my);
  const float m = th < 0.f ? -INFINITY : -nq;  // no key, or only scores of -inf or NaN
#pragma unroll
  for (int db = 0; db < DB; ++db) park[db * 64 + lane] = o[db];
  if (lane < 16) {
    sm[wave][lane] = m;
    sl[wave][lane] = l;
  }
  __syncthreads();
  const int lr = lane & 15;
  float big = fmaxf(fmaxf(sm[0][lr], sm[1][lr]), fmaxf(sm[2][lr], sm[3][lr]));
  float wt[4], lt = 0.f;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    wt[x] = sm[x][lr] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(sm[x][lr] - big);  // its sums are 0 (or NaN)
    lt += wt[x] * sl[x][lr];
  }
  f32x4 mine[(DB + 3) / 4];
#pragma unroll
  for (int i = 0; i < (DB + 3) / 4; ++i) {
    const int db = wave + 4 * i;
    mine[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (db < DB)
#pragma unroll
      for (int x = 0; x < 4; ++x) mine[i] += wt[x] * reinterpret_cast<const f32x4*>(&ring[x][0])[db * 64 + lane];
  }
  if (p.parts == 1) {
    win_finish_rows<T, DB>(p, sq, b, hk, rb, wave, lane, wave, 4, 0, p.D, mine, lt, &flag);
    return;
  }
  float* ws = p.ws + (int64_t)blockIdx.x * C::PART;
#pragma unroll
  for (int i = 0; i < (DB + 3) / 4; ++i)
    if (wave + 4 * i < DB) reinterpret_cast<f32x4*>(ws)[(wave + 4 * i) * 64 + lane] = mine[i];
  if (wave == 0 && lane < 16) {
    ws[C::PART_O + lane] = big;
    ws[C::PART_O + 16 + lane] = lt;
  }
}

// The parts of one block of rows.  A workgroup merges 32 columns, so that a few
// sequences' many parts (1 of 131072 tokens, 8 key heads: 32 parts of each) are
// read by enough of them; its waves take every fourth part, and their sums are
// added in wave order.
template <typename T, int DW>
__global__ __launch_bounds__(256) void win_merge_kernel(WinParams p) {
  using C = WinSplitCfg<DW>;
  constexpr int DB = DW / 16;
  __shared__ f32x4 so[4][2][64];
  __shared__ float sl[4][16];
  __shared__ uint32_t flag;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c2 = (int)blockIdx.x % (DB / 2), item = (int)blockIdx.x / (DB / 2);
  const int rb = item % p.RB, hk = item / p.RB % p.Hk, b = item / p.RB / p.Hk;
  if (threadIdx.x == 0) flag = 0;
  const WinSeq sq = win_seq(p, b);
  const float* ws = p.ws + (int64_t)item * p.parts * C::PART;
  const int lr = lane & 15;
  float big = -INFINITY;
#pragma unroll 8
  for (int q = 0; q < p.parts; ++q) big = fmaxf(big, ws[(int64_t)q * C::PART + C::PART_O + lr]);
  float lt = 0.f;
  f32x4 mine[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll 4
  for (int q = wave; q < p.parts; q += 4) {
    const float* pq = ws + (int64_t)q * C::PART;
    const float m = pq[C::PART_O + lr], wt = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - big);
    lt += wt * pq[C::PART_O + 16 + lr];
#pragma unroll
    for (int i = 0; i < 2; ++i) mine[i] += wt * reinterpret_cast<const f32x4*>(pq)[(2 * c2 + i) * 64 + lane];
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) so[wave][i][lane] = mine[i];
  if (lane < 16) sl[wave][lane] = lt;
  __syncthreads();
  lt = (sl[0][lr] + sl[1][lr]) + (sl[2][lr] + sl[3][lr]);
  // waves 0 and 1 store a block of 16 columns each
  f32x4 out[1] = {f32x4{0.f, 0.f, 0.f, 0.f}};
  if (wave < 2) out[0] = (so[0][wave][lane] + so[1][wave][lane]) + (so[2][wave][lane] + so[3][wave][lane]);
  win_finish_rows<T, DB>(p, sq, b, hk, rb, wave, lane, wave < 2 ? 2 * c2 + wave : DB, 1, 32 * c2, 32 * c2 + 32, out, lt,
                         &flag);
}

}  // namespace sf
