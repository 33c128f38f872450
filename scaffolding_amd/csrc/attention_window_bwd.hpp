// attention_window_bwd.hpp — gradients of win_attn_kernel (attention_window.hpp).
//
// With P = exp(scale Q K^T - lse) (0 where a query does not see a key), dO the
// gradient of O, and delta[i] = dO[i] . O[i]:
//
//   dV = P^T dO,  dP = dO V^T,  dS = P (dP - delta),
//   dQ = scale dS K,  dK = scale dS^T Q
//
// Two launches, each forming S and dP again (14 D flop a pair of query and key
// instead of 10 D): the sums of dQ run over keys, those of dK and dV over
// queries, so one launch for all would need atomic sums of one of them, whose
// order changes the bits.
//
//   win_dq_kernel   128 query rows a workgroup (32 a wave), Q and dO in
//                   registers, blocks of 64 keys of K and V through LDS; it
//                   forms delta first and leaves it, and lse as the exponents
//                   want it, for the other launch
//   win_dkv_kernel  128 keys a workgroup, 32 for two waves, their K and V in
//                   registers, blocks of 64 rows of Q and dO of every query head
//                   of the group through LDS: the sum over heads is part of it.
//                   Of two waves each forms P and dS of half the rows, hands
//                   them to the other through LDS and sums dK and dV of half the
//                   columns: 320 KB of LDS a block where 16 keys a wave alone
//                   read 512 (190 -> 179 us below)
//
// 2 x 4096 rows, 16 + 4 heads of 128, window 1024, 4 sinks, bf16: 132 us (90 GF,
// 690 TF/s), 179 us (121 GF, 675 TF/s) and 17 for the cut blocks' sums, 130 MB
// written and read.  Both products and LDS reading are busy about a third of the
// time and hardly overlap: two waves a SIMD is what the sums' registers leave, and
// the barriers keep them in step.  Forming the weights beside the products with V
// gains 2 % of the second launch and nothing in the first.  A third stage of
// tiles, or Q's rows asked for a tile ahead, takes more registers or LDS than
// there are.
//
// Both take the forward kernel's operand layouts: scores come out with the
// summed index (keys here, rows there) across a lane's registers, where the
// next product wants them, and the other operand of that product is read
// transposed from the LDS tile that the scores were formed from.
//
// P and dS are rounded to the operands' type for the products (half a step
// each); P of fp16 is held times 2^8, so that the weights of thousands of keys
// stay normal numbers.  Everything else, sums included, is fp32.
//
// How many rows see a block of keys differs widely (sinks, no window, short
// sequences), so win_dkv_kernel's work is cut evenly whatever it is: the (key
// block, row block, head) products of all key blocks in one list, as many equal
// ranges of it as workgroups fit the chip (win_plan_ranges: one more workgroup
// of the first launch, while the others work).  A key block whose products lie
// in one range is stored by it; of one that is cut each range leaves its fp32
// sums, and a third launch adds them in order (win_dkv_merge_kernel).
#pragma once

#include "attention_window.hpp"

namespace sf {

// A place in the list: product `at` of key block `block` (of (batch entry, key
// head, key block) in this order).
struct WinStart {
  int block, at;
};

struct WinBackParams {
  WinParams w;      // O: the forward output; lse its log-sums
  const void* dO;   // strides as O's
  void *dQ, *dK, *dV;  // strides as Q's, K's and V's
  int64_t sG, hG, sDQ, hDQ, sDK, hDK, sDV, hDV;
  int ldg, lddq, lddk, lddv;
  float* stat;      // [2, B, H, Sq]: -lse / ln 2 (P's scale added), then -delta
  float* ws;        // two sums (WinDkvCfg::PART floats) a range: its first and its last key block's
  WinStart* start;  // where each range begins, and the end of the last
  int ranges;
  int KBS;          // key blocks of 128 of a sequence
  float scale;
};

// The rows that see a key of block kb (128 keys): blocks of 64 rows from
// `first`; `products` of the list (every query head of the group times those,
// or 1 for a block past the sequence's end, whose gradient is 0).
struct WinKeyRows {
  int first, n, products;
};
__device__ __forceinline__ WinKeyRows win_key_rows(const WinParams& p, const WinSeq& s, int kb) {
  WinKeyRows r;
  const int k0 = kb * 128;
  int last = s.rows - 1;
  if (k0 >= p.sinks && k0 + 127 + p.window - 1 < last) last = k0 + 127 + p.window - 1;
  r.first = k0 / 64;
  r.n = last >= k0 ? last / 64 - r.first + 1 : 0;
  r.products = r.n > 0 ? r.n * p.G : 1;
  return r;
}

template <typename T>
struct WinBackScale {
  static constexpr float up = 1.0f, down = 1.0f, log2 = 0.0f;
};
template <>
struct WinBackScale<F16> {
  static constexpr float up = 256.0f, down = 1.0f / 256.0f, log2 = 8.0f;
};

// Fragment offsets of a tile of 128-byte rows (64 d each half), as
// win_attn_kernel's: rows of 16 (straight) and 16 columns of 32 rows
// (transposed).
struct WinFrag {
  uint32_t row;   // straight, chunk l >> 4 of row l & 15
  uint32_t trow;  // transposed
  int tch, tsw;
  __device__ __forceinline__ void set(int lane) {
    row = (uint32_t)((lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) << 4));
    const int vs = lane & 15, vrow = 4 * (lane >> 4) + (vs >> 2);
    trow = (uint32_t)vrow * 128u + (uint32_t)((vs & 1) * 8);
    tch = (vs & 3) >> 1;
    tsw = vrow & 7;
  }
};

// Rows NB 16 .. + 15 of the tile at `base`: KC chunks of 32 d.
template <int NB, int KC, int HB>
__device__ __forceinline__ void win_frag_rows(uint32_t base, const WinFrag& f, u32x4 (&out)[KC]) {
  static_for<KC>([&](auto kc_c) {
    constexpr int I = decltype(kc_c)::value;
    out[I] = ds_read16<(I >> 1) * HB + NB * 2048>((I & 1) ? ((base + f.row) ^ 64u) : base + f.row);
  });
}
// Columns 16 DBI .. + 15 of rows 32 C .. + 31, transposed.
template <int C, int DBI, int HB>
__device__ __forceinline__ u32x4 win_frag_cols(uint32_t base, const WinFrag& f) {
  const uint32_t a = base + f.trow + (uint32_t)(((2 * (DBI & 3) + f.tch) ^ f.tsw) << 4);
  const u32x2 x = ds_read_tr16<(DBI >> 2) * HB + C * 4096>(a), y = ds_read_tr16<(DBI >> 2) * HB + C * 4096 + 2048>(a);
  return u32x4{x.x, x.y, y.x, y.y};
}

// One wave's share (16 rows) of the direct loads of a 64-row tile: rows from
// row0 of `base`, those from `end` on and columns from D on read as zeros.
template <int HV>
__device__ __forceinline__ void win_load_tile(const uint16_t* base, int ld, int row0, int end, int D, uint8_t* dst,
                                              int wave, int lane) {
  constexpr int HB = 64 * 128;
  const int left = end - row0 < 64 ? end - row0 : 64;  // >= 1
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(base + (int64_t)row0 * ld), (short)0, (int)(((uint32_t)(left - 1) * (uint32_t)ld + (uint32_t)D) * 2u),
      0x00020000);
  const int ch = (lane & 7) ^ (lane >> 3);
  const uint32_t r0 = (uint32_t)(wave * 16 + (lane >> 3)) * (uint32_t)ld * 2u, r8 = 16u * (uint32_t)ld;
#pragma unroll
  for (int hf = 0; hf < HV; ++hf) {
    const int d = hf * 64 + ch * 8;
    const uint32_t o = d < D ? r0 + (uint32_t)d * 2u : 0x80000000u;
    uint8_t* p = dst + hf * HB + wave * 2048;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)p, 16, o, 0, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)(p + 1024), 16, o + r8, 0, 0, 0);
  }
}

// Fragments of 16 rows from global memory (rows at or past `end` as zeros).
template <int KC>
__device__ __forceinline__ void win_load_rows(const uint16_t* base, int ld, int row0, int end, int D, int lane,
                                              u32x4 (&out)[KC]) {
  const int r = row0 + (lane & 15);
#pragma unroll
  for (int kc = 0; kc < KC; ++kc) {
    const int d = kc * 32 + 8 * (lane >> 4);
    out[kc] = r < end && d < D ? *reinterpret_cast<const u32x4*>(base + (int64_t)r * ld + d) : u32x4{0u, 0u, 0u, 0u};
  }
}

// Cuts the list of products into bp.ranges equal ranges.  One workgroup.
__device__ __forceinline__ void win_plan_ranges(const WinBackParams& bp, int64_t* scan) {
  const WinParams& p = bp.w;
  const int tid = (int)threadIdx.x, nt = (int)blockDim.x;
  const int64_t all = (int64_t)p.B * p.Hk * bp.KBS;
  auto products = [&](int64_t e) -> int64_t {
    const int kb = (int)(e % bp.KBS);
    return win_key_rows(p, win_seq(p, e / bp.KBS / p.Hk), kb).products;
  };
  // the sum over the threads' values up to this one; every thread calls it
  auto running = [&](int64_t v) {
    scan[tid] = v;
    __syncthreads();
    for (int off = 1; off < nt; off <<= 1) {
      const int64_t o = tid >= off ? scan[tid - off] : 0;
      __syncthreads();
      scan[tid] += o;
      __syncthreads();
    }
    return scan[tid];
  };
  int64_t v = 0;
  for (int64_t e = tid; e < all; e += nt) v += products(e);
  running(v);
  const int64_t total = scan[nt - 1];
  __syncthreads();
  int64_t base = 0;
  for (int64_t e0 = 0; e0 < all; e0 += nt) {
    const int64_t e = e0 + tid, c = e < all ? products(e) : 0;
    const int64_t end = base + running(c), begin = end - c;
    base += scan[nt - 1];
    __syncthreads();
    // range w begins at product w total / ranges
    for (int64_t w = (begin * bp.ranges + total - 1) / total; w < bp.ranges; ++w) {
      const int64_t at = w * total / bp.ranges;
      if (at >= end) break;
      bp.start[w] = WinStart{(int)e, (int)(at - begin)};
    }
  }
  if (tid == 0) bp.start[bp.ranges] = WinStart{(int)all, 0};
}

// Stores the lane's part of 16 rows (row: the lane's) of a gradient; rows at or
// past `end` get 0, those past `rows` are not there.
template <typename T, int DB>
__device__ __forceinline__ void win_store_16(uint16_t* base, int ld, int row, int end, int rows, int D, float scale,
                                             int lane, const f32x4 (&v)[DB]) {
  if (row >= rows) return;
  uint16_t* out = base + (int64_t)row * ld;
#pragma unroll
  for (int db = 0; db < DB; ++db) {
    const int d = db * 16 + 4 * (lane >> 4);
    const f32x4 x = v[db];
    if (d < D)
      *reinterpret_cast<u32x2*>(out + d) =
          row < end ? u32x2{pack2<T>(x[0] * scale, x[1] * scale), pack2<T>(x[2] * scale, x[3] * scale)} : u32x2{0u, 0u};
  }
}

template <typename T, int DW>
__global__ __launch_bounds__(256, 2) void win_dq_kernel(WinBackParams bp) {
  using C = WinCfg<DW>;
  using S = WinBackScale<T>;
  constexpr int MB = 2, HV = C::HALVES, KC = DW / 32, DB = DW / 16, KB = 64, HB = KB * 128, NS = 2;
  const WinParams& p = bp.w;
  __shared__ __attribute__((aligned(1024))) uint8_t sK[NS][HV * HB];
  __shared__ __attribute__((aligned(1024))) uint8_t sV[NS][HV * HB];
  if (blockIdx.x == 0) {  // the other launch's plan
    win_plan_ranges(bp, reinterpret_cast<int64_t*>(&sK[0][0]));
    return;
  }
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int qb, b, h;
  win_item(p, (int)blockIdx.x - 1, qb, b, h);
  const int hk = h / p.G;
  const WinSeq sq = win_seq(p, b);
  const int r0 = qb * 128, q0 = r0 + wave * 32;
  const int r1 = r0 + 128 < sq.rows ? r0 + 128 : sq.rows;
  const WinBlocks<KB> kbs = win_blocks<KB>(p, sq, r0, r1 > r0 ? r1 : r0);
  const int nkb = r1 > r0 ? kbs.n : 0;
  const uint16_t* Qb = static_cast<const uint16_t*>(p.Q) + b * p.sQ + h * p.hQ;
  const uint16_t* Kb = static_cast<const uint16_t*>(p.K) + b * p.sK + hk * p.hK;
  const uint16_t* Vb = static_cast<const uint16_t*>(p.V) + b * p.sV + hk * p.hV;
  const uint16_t* Ob = static_cast<const uint16_t*>(p.O) + b * p.sO + h * p.hO;
  const uint16_t* Gb = static_cast<const uint16_t*>(bp.dO) + b * bp.sG + h * bp.hG;
  auto issue = [&](int i) {
    const int j = kbs.at(i) * KB;
    win_load_tile<HV>(Kb, p.ldk, j, sq.keys, p.D, &sK[i & 1][0], wave, lane);
    win_load_tile<HV>(Vb, p.ldv, j, sq.keys, p.D, &sV[i & 1][0], wave, lane);
  };
  if (nkb > 0) issue(0);

  u32x4 qf[MB][KC], gf[MB][KC];
  float nl[MB], dl[MB];
  const int64_t stat = ((int64_t)b * p.H + h) * p.Sq;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    u32x4 of[KC];
    const int row = q0 + mb * 16 + (lane & 15);
    win_load_rows<KC>(Qb, p.ldq, q0 + mb * 16, sq.rows, p.D, lane, qf[mb]);
    win_load_rows<KC>(Gb, bp.ldg, q0 + mb * 16, sq.rows, p.D, lane, gf[mb]);
    win_load_rows<KC>(Ob, p.ldo, q0 + mb * 16, sq.rows, p.D, lane, of);
    float d = 0.f;
#pragma unroll
    for (int kc = 0; kc < KC; ++kc)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t x = gf[mb][kc][e], y = of[kc][e];
        d = __builtin_fmaf(Elem<T>::to_f32((uint16_t)(x & 0xffffu)), Elem<T>::to_f32((uint16_t)(y & 0xffffu)), d);
        d = __builtin_fmaf(Elem<T>::to_f32((uint16_t)(x >> 16)), Elem<T>::to_f32((uint16_t)(y >> 16)), d);
      }
    d += __shfl_xor(d, 16, 64);
    d += __shfl_xor(d, 32, 64);
    dl[mb] = -d;
    nl[mb] = row < sq.rows ? S::log2 - p.lse[stat + row] * 1.4426950408889634f : 0.f;
    if (row < sq.rows && lane < 16) {
      bp.stat[stat + row] = nl[mb];
      bp.stat[(int64_t)p.B * p.H * p.Sq + stat + row] = -d;
    }
  }
  f32x4 dq[MB][DB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int db = 0; db < DB; ++db) dq[mb][db] = f32x4{0.f, 0.f, 0.f, 0.f};
  WinFrag fr;
  fr.set(lane);
  const int pw0 = q0, pw1 = q0 + 31;

  for (int i = 0; i < nkb; ++i) {
    const int k0 = kbs.at(i) * KB, k1 = k0 + KB - 1;
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 0));
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    if (i + 1 < nkb) issue(i + 1);
    __builtin_amdgcn_sched_barrier(0);
    if (k0 > pw1 || (k1 <= pw0 - p.window && k0 >= p.sinks)) continue;
    const bool edge = k1 > pw0 || k1 >= sq.keys || (k0 <= pw1 - p.window && k1 >= p.sinks);
    const uint32_t ka = lds_addr(&sK[i & 1][0]), va = lds_addr(&sV[i & 1][0]);
    static_for<2>([&](auto c_c) {
      constexpr int CH = decltype(c_c)::value;  // keys 32 CH .. + 31 of the block
      f32x4 s[MB][2], dp[MB][2];
      static_for<2>([&](auto n_c) {
        constexpr int N = decltype(n_c)::value, NB = 2 * CH + N;
        u32x4 kf[KC], vf[KC];
        win_frag_rows<NB, KC, HB>(ka, fr, kf);
        win_frag_rows<NB, KC, HB>(va, fr, vf);
        __builtin_amdgcn_s_waitcnt(waitcnt_imm(63, KC));
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          s[mb][N] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int kc = 0; kc < KC; ++kc) s[mb][N] = Mfma16<T>::run(kf[kc], qf[mb][kc], s[mb][N]);
        }
        __builtin_amdgcn_s_waitcnt(waitcnt_imm(63, 0));
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          dp[mb][N] = f32x4{dl[mb], dl[mb], dl[mb], dl[mb]};
#pragma unroll
          for (int kc = 0; kc < KC; ++kc) dp[mb][N] = Mfma16<T>::run(vf[kc], gf[mb][kc], dp[mb][N]);
        }
      });
      u32x4 kt[DB];
      __builtin_amdgcn_sched_barrier(0);
      static_for<DB>([&](auto db_c) {
        constexpr int I = decltype(db_c)::value;
        kt[I] = win_frag_cols<CH, I, HB>(ka, fr);
      });
      __builtin_amdgcn_sched_barrier(0);
      u32x4 ds[MB];
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        const int pos = pw0 + mb * 16 + (lane & 15);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          float v[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[mb][n][q], p.scale_log2e, nl[mb]));
            v[q] = e * (dp[mb][n][q] * S::down);
            if (edge && !win_sees(p, sq, pos, k0 + CH * 32 + n * 16 + 4 * (lane >> 4) + q)) v[q] = 0.f;
          }
          ds[mb][2 * n] = pack2<T>(v[0], v[1]);
          ds[mb][2 * n + 1] = pack2<T>(v[2], v[3]);
        }
      }
      __builtin_amdgcn_s_waitcnt(waitcnt_imm(63, 0));
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) dq[mb][db] = Mfma16<T>::run(kt[db], ds[mb], dq[mb][db]);
      __builtin_amdgcn_sched_barrier(0);
    });
  }
  uint16_t* Db = static_cast<uint16_t*>(bp.dQ) + b * bp.sDQ + h * bp.hDQ;
#pragma unroll
  for (int mb = 0; mb < 2; ++mb)
    win_store_16<T, DB>(Db, bp.lddq, q0 + mb * 16 + (lane & 15), sq.rows, p.Sq, p.D, bp.scale, lane, dq[mb]);
}

template <int DW>
struct WinDkvCfg {
  static constexpr int PART = 2 * 128 * DW;  // floats of the sums of a workgroup's 128 keys, dK and dV
};

// 16 bytes a lane to LDS, in the order of the ds_read16 around it.
__device__ __forceinline__ void ds_write16(uint32_t addr, u32x4 v) {
  asm volatile("ds_write_b128 %0, %1" ::"v"(addr), "v"(v) : "memory");
}

template <typename T, int DW>
__global__ __launch_bounds__(512, 2) void win_dkv_kernel(WinBackParams bp) {
  using S = WinBackScale<T>;
  constexpr int HV = WinCfg<DW>::HALVES, KC = DW / 32, DB = DW / 16, DH = DB / 2, RB = 64, HB = RB * 128, NS = 2;
  const WinParams& p = bp.w;
  __shared__ __attribute__((aligned(1024))) uint8_t sQ[NS][HV * HB];
  __shared__ __attribute__((aligned(1024))) uint8_t sG[NS][HV * HB];
  __shared__ __attribute__((aligned(256))) float sL[NS][2][RB];
  __shared__ __attribute__((aligned(1024))) u32x4 sX[8][4][64];  // a wave's P and dS
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = wave & 1;  // of a tile's rows, and of the columns of D
  // Each XCD takes a contiguous share of the ranges: neighbouring key blocks
  // read the same rows.
  const int w = xcd_remap((int)blockIdx.x, (int)gridDim.x);
  const WinStart from = bp.start[w], to = bp.start[w + 1];
  WinFrag fr;
  fr.set(lane);
  uint32_t col[DH];  // transposed fragments of the wave's columns
#pragma unroll
  for (int x = 0; x < DH; ++x) {
    const int db = half * DH + x;
    col[x] = fr.trow + (uint32_t)(((2 * (db & 3) + fr.tch) ^ fr.tsw) << 4) + (uint32_t)((db >> 2) * HB);
  }
  const uint32_t xa = lds_addr(&sX[wave][0][0]) + (uint32_t)lane * 16u;
  const uint32_t xb = lds_addr(&sX[wave ^ 1][0][0]) + (uint32_t)lane * 16u;
  for (int e = from.block; e < to.block || (e == to.block && to.at > 0); ++e) {
    const int kv = e / bp.KBS, kb = e % bp.KBS;
    const int b = kv / p.Hk, hk = kv % p.Hk;
    const WinSeq sq = win_seq(p, b);
    const int n = sq.rows;
    const WinKeyRows kr = win_key_rows(p, sq, kb);
    const int begin = e == from.block ? from.at : 0, end = e == to.block ? to.at : kr.products;
    const int t0 = begin, t1 = kr.n > 0 ? end : begin;  // past the sequence: nothing to add up
    const int kw0 = kb * 128 + (wave >> 1) * 32;
    const uint16_t* Kb = static_cast<const uint16_t*>(p.K) + b * p.sK + hk * p.hK;
    const uint16_t* Vb = static_cast<const uint16_t*>(p.V) + b * p.sV + hk * p.hV;
    const uint16_t* Qb = static_cast<const uint16_t*>(p.Q) + b * p.sQ + (int64_t)hk * p.G * p.hQ;
    const uint16_t* Gb = static_cast<const uint16_t*>(bp.dO) + b * bp.sG + (int64_t)hk * p.G * bp.hG;
    // waves 0-3 load Q's tile, 4-7 that of dO
    auto issue = [&](int t) {
      const int g = t / kr.n, row0 = (kr.first + t % kr.n) * RB, st = (t - t0) % NS;
      if (wave < 4) win_load_tile<HV>(Qb + g * p.hQ, p.ldq, row0, n, p.D, &sQ[st][0], wave, lane);
      else win_load_tile<HV>(Gb + g * bp.hG, bp.ldg, row0, n, p.D, &sG[st][0], wave - 4, lane);
      if (wave < 2) {
        const int left = n - row0 < RB ? n - row0 : RB;
        const float* src = bp.stat + (((int64_t)wave * p.B + b) * p.H + hk * p.G + g) * p.Sq + row0;
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)src, (short)0, left * 4, 0x00020000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)&sL[st][wave][0], 4, (uint32_t)lane * 4u, 0, 0, 0);
      }
    };
    __syncthreads();  // every wave has read the last block's tiles
    if (t0 < t1) issue(t0);
    u32x4 kf[2][KC], vf[2][KC];
    f32x4 dk[2][DH], dv[2][DH];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      win_load_rows<KC>(Kb, p.ldk, kw0 + 16 * j, n, p.D, lane, kf[j]);
      win_load_rows<KC>(Vb, p.ldv, kw0 + 16 * j, n, p.D, lane, vf[j]);
#pragma unroll
      for (int x = 0; x < DH; ++x) dk[j][x] = dv[j][x] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    for (int t = t0; t < t1; ++t) {
      const int row0 = (kr.first + t % kr.n) * RB, st = (t - t0) % NS;
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 0));
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
      if (t + 1 < t1) issue(t + 1);
      __builtin_amdgcn_sched_barrier(0);
      // whether rows c0 .. c0 + 31 see one of the wave's keys
      auto meet = [&](int c0) {
        return !(c0 + 31 < kw0 || (kw0 + 31 <= c0 - p.window && kw0 >= p.sinks) || c0 >= n);
      };
      const uint32_t qa = lds_addr(&sQ[st][0]), ga = lds_addr(&sG[st][0]);
      // The gradients of the wave's columns from rows 32 c .. + 31: the reading,
      // and the products.
      auto columns = [&](uint32_t base, uint32_t c, u32x4 (&f)[DH]) {
        static_for<DH>([&](auto x_c) {
          constexpr int X = decltype(x_c)::value;
          const uint32_t a = base + col[X] + c * 4096u;
          const u32x2 lo = ds_read_tr16<0>(a), hi = ds_read_tr16<2048>(a);
          f[X] = u32x4{lo.x, lo.y, hi.x, hi.y};
        });
      };
      auto add = [&](const u32x4 (&f)[DH], const u32x4 (&pt)[2], f32x4 (&out)[2][DH]) {
#pragma unroll
        for (int x = 0; x < DH; ++x)
#pragma unroll
          for (int j = 0; j < 2; ++j) out[j][x] = Mfma16<T>::run(f[x], pt[j], out[j][x]);
      };
      const int c0 = row0 + half * 32;
      if (meet(c0)) {
        const bool edge = kw0 + 31 > c0 || c0 + 31 >= n || (kw0 <= c0 + 31 - p.window && kw0 + 31 >= p.sinks);
        const uint32_t la = lds_addr(&sL[st][0][0]) + (uint32_t)half * 128u + (uint32_t)(lane >> 4) * 16u;
        const uint32_t q0 = qa + (uint32_t)half * 4096u, g0 = ga + (uint32_t)half * 4096u;
        u32x4 qf[2][KC], gf[2][KC], ls[2], dl[2], pf[2], ds[2], gt[DH], qt[DH];
        f32x4 s[2][2], dp[2][2];
        static_for<2>([&](auto i) { win_frag_rows<decltype(i)::value, KC, HB>(q0, fr, qf[decltype(i)::value]); });
        static_for<2>([&](auto i) {
          constexpr int I = decltype(i)::value;
          ls[I] = ds_read16<I * 64>(la);
          dl[I] = ds_read16<RB * 4 + I * 64>(la);
          win_frag_rows<I, KC, HB>(g0, fr, gf[I]);
        });
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(waitcnt_imm(63, 2 * KC + 4));  // Q's rows
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) s[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kc = 0; kc < KC; ++kc)
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) s[i][j] = Mfma16<T>::run(qf[i][kc], kf[j][kc], s[i][j]);
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(waitcnt_imm(63, 0));
        __builtin_amdgcn_sched_barrier(0);
        columns(ga, (uint32_t)half, gt);
        __builtin_amdgcn_sched_barrier(0);
        // the weights are formed while the products with V run
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const f32x4 nl = __builtin_bit_cast(f32x4, ls[i]);
            dp[i][j] = __builtin_bit_cast(f32x4, dl[i]);
#pragma unroll
            for (int q = 0; q < 4; ++q)
              s[i][j][q] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][j][q], p.scale_log2e, nl[q]));
          }
#pragma unroll
        for (int kc = 0; kc < KC; ++kc)
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) dp[i][j] = Mfma16<T>::run(gf[i][kc], vf[j][kc], dp[i][j]);
#pragma unroll
        for (int g = 0; g < 4 * KC; ++g) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        columns(qa, (uint32_t)half, qt);
        __builtin_amdgcn_sched_barrier(0);
        if (edge) {
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int key = kw0 + 16 * j + (lane & 15), row = c0 + i * 16 + 4 * (lane >> 4);
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const bool see = (row + q < n) & win_sees(p, sq, row + q, key);
                s[i][j][q] = see ? s[i][j][q] : 0.f;
                dp[i][j][q] = see ? dp[i][j][q] : 0.f;
              }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            pf[j][2 * i] = pack2<T>(s[i][j][0], s[i][j][1]);
            pf[j][2 * i + 1] = pack2<T>(s[i][j][2], s[i][j][3]);
          }
        __builtin_amdgcn_s_waitcnt(waitcnt_imm(63, 2 * DH));  // dO's columns
        __builtin_amdgcn_sched_barrier(0);
        add(gt, pf, dv);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float v[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = s[i][j][q] * (dp[i][j][q] * S::down);
            ds[j][2 * i] = pack2<T>(v[0], v[1]);
            ds[j][2 * i + 1] = pack2<T>(v[2], v[3]);
          }
#pragma unroll
        for (int g = 0; g < 2 * DH; ++g) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x002, 3, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          ds_write16(xa + j * 1024, pf[j]);
          ds_write16(xa + (2 + j) * 1024, ds[j]);
        }
        __builtin_amdgcn_s_waitcnt(waitcnt_imm(63, 4));  // Q's columns
        __builtin_amdgcn_sched_barrier(0);
        add(qt, ds, dk);
      }
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(waitcnt_imm(63, 0));
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
      if (meet(row0 + (half ^ 1) * 32)) {  // the neighbour's rows, for the wave's columns
        u32x4 pf[2], ds[2], gt[DH], qt[DH];
        pf[0] = ds_read16<0>(xb), pf[1] = ds_read16<1024>(xb);
        columns(ga, (uint32_t)(half ^ 1), gt);
        ds[0] = ds_read16<2048>(xb), ds[1] = ds_read16<3 * 1024>(xb);
        columns(qa, (uint32_t)(half ^ 1), qt);
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(waitcnt_imm(63, 2 * DH + 2));
        __builtin_amdgcn_sched_barrier(0);
        add(gt, pf, dv);
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(waitcnt_imm(63, 0));
        __builtin_amdgcn_sched_barrier(0);
        add(qt, ds, dk);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (begin == 0 && end == kr.products) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int key = kw0 + 16 * j + (lane & 15), d0 = half * DH * 16;
        win_store_16<T, DH>(static_cast<uint16_t*>(bp.dK) + b * bp.sDK + hk * bp.hDK + d0, bp.lddk, key, n, p.Sk,
                            p.D - d0, bp.scale, lane, dk[j]);
        win_store_16<T, DH>(static_cast<uint16_t*>(bp.dV) + b * bp.sDV + hk * bp.hDV + d0, bp.lddv, key, n, p.Sk,
                            p.D - d0, S::down, lane, dv[j]);
      }
    } else {
      f32x4* out = reinterpret_cast<f32x4*>(bp.ws + (int64_t)(2 * w + (begin == 0 ? 1 : 0)) * WinDkvCfg<DW>::PART) +
                   ((wave >> 1) * 2 * DB + half * DH) * 64 + lane;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int x = 0; x < DH; ++x) {
          out[(j * DB + x) * 64] = dk[j][x];
          out[(8 * DB + j * DB + x) * 64] = dv[j][x];
        }
    }
  }
}

// The key block that range w begins and does not end: its sums and those of the
// ranges behind it that hold more of the block, added in order.
template <typename T, int DW>
__global__ __launch_bounds__(512) void win_dkv_merge_kernel(WinBackParams bp) {
  using S = WinBackScale<T>;
  constexpr int DB = DW / 16, PART = WinDkvCfg<DW>::PART / 4;
  const WinParams& p = bp.w;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int w = (int)blockIdx.x / 2, dv = (int)blockIdx.x % 2;
  const WinStart from = bp.start[w], to = bp.start[w + 1];
  const int e = to.block;
  if (to.at == 0 || (from.block == e && from.at > 0) || (from.block == e && from.at == to.at)) return;
  const int kv = e / bp.KBS, kb = e % bp.KBS;
  const int b = kv / p.Hk, hk = kv % p.Hk;
  const WinSeq sq = win_seq(p, b);
  const f32x4* in = reinterpret_cast<const f32x4*>(bp.ws) + (dv * 8 * DB + wave * DB) * 64 + lane;
  f32x4 v[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) v[db] = in[(int64_t)(2 * w + 1) * PART + db * 64];
  WinStart at = to;
  for (int f = w + 1; f < bp.ranges; ++f) {
    const WinStart next = bp.start[f + 1];
    if (next.block != at.block || next.at != at.at) {  // a range with products
#pragma unroll
      for (int db = 0; db < DB; ++db) v[db] += in[(int64_t)2 * f * PART + db * 64];
      if (next.block != e) break;
      at = next;
    }
  }
  const int key = kb * 128 + wave * 16 + (lane & 15);
  if (dv == 0)
    win_store_16<T, DB>(static_cast<uint16_t*>(bp.dK) + b * bp.sDK + hk * bp.hDK, bp.lddk, key, sq.rows, p.Sk, p.D,
                          bp.scale, lane, v);
  else
    win_store_16<T, DB>(static_cast<uint16_t*>(bp.dV) + b * bp.sDV + hk * bp.hDV, bp.lddv, key, sq.rows, p.Sk, p.D,
                          S::down, lane, v);
}

}  // namespace sf
