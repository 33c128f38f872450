// qknorm.hip — norms of queries and keys per head with the position rotation
// in the same pass, and the backward pass.
//
// A head's D columns are normed (rms: x r, r = rsqrt(mean x^2 + eps); layer:
// (x - mean) r with the variance under r), scaled (and shifted), and its first
// `rot` columns turned in pairs (a, b) -> (a cos - b sin, b cos + a sin) by the
// token's row of a table.  One read and one write of the projection: bound by
// HBM.
//
// A lane owns two chunks of V columns: the two halves of V rotated pairs
// (columns c and c + rot / 2, or neighbouring chunks where pairs are
// neighbouring columns), so the rotation needs no other lane.  L lanes hold a
// head, 64 / L heads are in flight in a wave, and the mean runs over L lanes.
// A wave keeps to heads of one kind (queries, keys or values), so it holds one
// row of the weight and, backward, one row of its gradient's sums.
//
// Backward, with hat the normed head, d the gradient turned back and e = d w:
//   dw += d hat, db += d, dx = r (e - hat mean(e hat) [layer: - mean(e)])
// The sums over tokens stay in fp32 registers, are added over the block's
// waves in LDS, parked per block, and added in block order by a second launch:
// no atomics, the same bits every time.
#include "rowio.hpp"
#include "sf_internal.hpp"

namespace sf {

// V elements of type T at element alignment, as loaded.
template <typename T, int V> struct Vec;
struct __attribute__((packed, aligned(2))) H4u {
  u32x2 v;
};
template <typename T> struct Vec<T, 8> {
  u32x4 w;
  __device__ __forceinline__ void load(const void* b, int64_t i) {
    w = reinterpret_cast<const H8u*>(static_cast<const uint16_t*>(b) + i)->v;
  }
  __device__ __forceinline__ void zero() { w = u32x4{0u, 0u, 0u, 0u}; }
  __device__ __forceinline__ float get(int e) const {
    return Elem<T>::to_f32(static_cast<uint16_t>(w[e >> 1] >> ((e & 1) * 16)));
  }
  __device__ __forceinline__ static void store(void* b, int64_t i, const float* v) { store8u<T>(b, i, v); }
};
template <typename T> struct Vec<T, 4> {
  u32x2 w;
  __device__ __forceinline__ void load(const void* b, int64_t i) {
    w = reinterpret_cast<const H4u*>(static_cast<const uint16_t*>(b) + i)->v;
  }
  __device__ __forceinline__ void zero() { w = u32x2{0u, 0u}; }
  __device__ __forceinline__ float get(int e) const {
    return Elem<T>::to_f32(static_cast<uint16_t>(w[e >> 1] >> ((e & 1) * 16)));
  }
  __device__ __forceinline__ static void store(void* b, int64_t i, const float* v) {
    reinterpret_cast<H4u*>(static_cast<uint16_t*>(b) + i)->v = u32x2{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])};
  }
};
template <typename T> struct Vec<T, 1> {
  uint16_t w;
  __device__ __forceinline__ void load(const void* b, int64_t i) { w = static_cast<const uint16_t*>(b)[i]; }
  __device__ __forceinline__ void zero() { w = 0; }
  __device__ __forceinline__ float get(int) const { return Elem<T>::to_f32(w); }
  __device__ __forceinline__ static void store(void* b, int64_t i, const float* v) {
    static_cast<uint16_t*>(b)[i] = Elem<T>::from_f32(v[0]);
  }
};
template <int V> struct VecF {
  f32x4 w[V / 4];
  __device__ __forceinline__ void load(const void* b, int64_t i) {
#pragma unroll
    for (int e = 0; e < V / 4; ++e) w[e] = reinterpret_cast<const F4u*>(static_cast<const float*>(b) + i)[e].v;
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int e = 0; e < V / 4; ++e) w[e] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  __device__ __forceinline__ float get(int e) const { return w[e >> 2][e & 3]; }
  __device__ __forceinline__ static void store(void* b, int64_t i, const float* v) {
#pragma unroll
    for (int e = 0; e < V / 4; ++e)
      reinterpret_cast<F4u*>(static_cast<float*>(b) + i)[e].v = f32x4{v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]};
  }
};
template <> struct Vec<float, 8> : VecF<8> {};
template <> struct Vec<float, 4> : VecF<4> {};
template <> struct Vec<float, 1> {
  float w;
  __device__ __forceinline__ void load(const void* b, int64_t i) { w = static_cast<const float*>(b)[i]; }
  __device__ __forceinline__ void zero() { w = 0.f; }
  __device__ __forceinline__ float get(int) const { return w; }
  __device__ __forceinline__ static void store(void* b, int64_t i, const float* v) { static_cast<float*>(b)[i] = v[0]; }
};

struct NormRopeParams {
  NormRopeArgs a;
  int lg;             // log2 of the lanes of a head
  int per;            // heads of a slice
  int nq, nk, nv;     // slices of the query, key and value heads
  int64_t stride;     // tokens between a wave's units
};

// A lane's columns.
template <int V, int PL, bool PAIRS>
struct Lanes {
  int ca[PL], cb[PL];  // first column of either chunk, -1: none
  int tix[PL];         // the chunks' first angle, -1: not rotated
  __device__ __forceinline__ void set(int sub, int L, int D, int rot) {
    constexpr bool NEXT = PAIRS && V > 1;  // pairs within a chunk
    const int rp = rot / (2 * V);
#pragma unroll
    for (int u = 0; u < PL; ++u) {
      const int p = sub + u * L;
      tix[u] = p < rp ? p * V : -1;
      if (NEXT || p >= rp) {
        ca[u] = NEXT ? 2 * p * V : rot + 2 * (p - rp) * V;
        cb[u] = ca[u] + V;
      } else {
        ca[u] = PAIRS ? 2 * p : p * V;
        cb[u] = PAIRS ? 2 * p + 1 : p * V + rot / 2;
      }
      if (ca[u] >= D) ca[u] = -1;
      if (cb[u] >= D) cb[u] = -1;
    }
  }
};

template <int V>
__device__ __forceinline__ void load_angles(const float* p, float* out) {
  if constexpr (V == 1) {
    out[0] = p[0];
  } else {
#pragma unroll
    for (int e = 0; e < V / 4; ++e) {
      const f32x4 v = reinterpret_cast<const F4u*>(p)[e].v;
#pragma unroll
      for (int q = 0; q < 4; ++q) out[4 * e + q] = v[q];
    }
  }
}

// (a, b) turned by (c, s), in place.  NEXT: the pairs are neighbours within a,
// then within b.
template <int V, bool NEXT>
__device__ __forceinline__ void turn(float* a, float* b, const float* c, const float* s) {
  if constexpr (NEXT) {
#pragma unroll
    for (int e = 0; e < V / 2; ++e) {
      const float a0 = a[2 * e], a1 = a[2 * e + 1], b0 = b[2 * e], b1 = b[2 * e + 1];
      a[2 * e] = a0 * c[e] - a1 * s[e];
      a[2 * e + 1] = a1 * c[e] + a0 * s[e];
      b[2 * e] = b0 * c[V / 2 + e] - b1 * s[V / 2 + e];
      b[2 * e + 1] = b1 * c[V / 2 + e] + b0 * s[V / 2 + e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float x = a[e], y = b[e];
      a[e] = x * c[e] - y * s[e];
      b[e] = y * c[e] + x * s[e];
    }
  }
}

// The sum over L = 2^n neighbouring lanes, in each of them: up to 16 by the
// lane network (pairs, quads, halves and rows mirrored), without the trip
// through LDS that a permute takes.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float sum_lanes(float v, int L) {
  if (L >= 2) v += dpp<0xb1>(v);    // quad_perm 1 0 3 2
  if (L >= 4) v += dpp<0x4e>(v);    // quad_perm 2 3 0 1
  if (L >= 8) v += dpp<0x141>(v);   // row_half_mirror
  if (L >= 16) v += dpp<0x140>(v);  // row_mirror
  if (L >= 32) v += __shfl_xor(v, 16, 64);
  if (L >= 64) v += __shfl_xor(v, 32, 64);
  return v;
}

// Where the unit's wave stands: its slice's kind (0 queries, 1 keys, 2
// values), first head and number of heads.
struct Slice {
  int kind, first, count;
};
__device__ __forceinline__ Slice slice_of(const NormRopeParams& p, int s) {
  Slice r;
  r.kind = s < p.nq ? 0 : s < p.nq + p.nk ? 1 : 2;
  r.first = (s - (r.kind > 0 ? p.nq : 0) - (r.kind > 1 ? p.nk : 0)) * p.per;
  const int heads = r.kind == 0 ? p.a.heads : p.a.kv_heads;
  r.count = heads - r.first < p.per ? heads - r.first : p.per;
  return r;
}

// Columns of the head in the packed row.
__device__ __forceinline__ int64_t head_col(const NormRopeArgs& a, int kind, int h) {
  return (int64_t)(h + (kind > 0 ? a.heads : 0) + (kind > 1 ? a.kv_heads : 0)) * a.D;
}

// Token t's position as the table counts it; cos and sin of the lane's pairs.
template <int V, int PL>
__device__ __forceinline__ void angles(const NormRopeArgs& a, int64_t pos, const int (&tix)[PL], float (&c)[PL][V],
                                       float (&s)[PL][V]) {
  const bool in = pos >= 0 && pos < a.table_rows;  // uniform
#pragma unroll
  for (int u = 0; u < PL; ++u) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      c[u][e] = 1.f;
      s[u][e] = 0.f;
    }
    if (tix[u] >= 0) {
      if (in) {
        const float* row = a.table + pos * a.rot + tix[u];
        load_angles<V>(row, c[u]);
        load_angles<V>(row + a.rot / 2, s[u]);
      } else {  // no such row: NaN
#pragma unroll
        for (int e = 0; e < V; ++e) c[u][e] = s[u][e] = __builtin_nanf("");
      }
    }
  }
}

// Waves of a block share a slice; block b takes slice b % slices and tokens
// 4 (b / slices) + wave, then every stride-th.
template <typename T, int V, int PL, bool PAIRS>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(NormRopeParams p) {
  const NormRopeArgs& a = p.a;
  constexpr bool NEXT = PAIRS && V > 1;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slices = p.nq + p.nk + p.nv;
  const Slice sl = slice_of(p, (int)(blockIdx.x % (unsigned)slices));
  const int L = 1 << p.lg, D = a.D, hpw = 64 >> p.lg, hg = lane >> p.lg;
  Lanes<V, PL, PAIRS> ln;
  ln.set(lane & (L - 1), L, D, a.rot);
  Vec<T, V> wa[PL], wb[PL], ba[PL], bb[PL];
  if (sl.kind < 2) {
#pragma unroll
    for (int u = 0; u < PL; ++u) {
      wa[u].zero(), wb[u].zero(), ba[u].zero(), bb[u].zero();
      if (a.weight != nullptr) {
        if (ln.ca[u] >= 0) wa[u].load(a.weight, sl.kind * D + ln.ca[u]);
        if (ln.cb[u] >= 0) wb[u].load(a.weight, sl.kind * D + ln.cb[u]);
      }
      if (a.bias != nullptr) {
        if (ln.ca[u] >= 0) ba[u].load(a.bias, sl.kind * D + ln.ca[u]);
        if (ln.cb[u] >= 0) bb[u].load(a.bias, sl.kind * D + ln.cb[u]);
      }
    }
  }
  const float inv_d = 1.0f / (float)D;
  const int64_t tokens = a.batch * a.rows;
  typedef typename Elem<T>::storage S;
  for (int64_t t = (int64_t)(blockIdx.x / (unsigned)slices) * 4 + wave; t < tokens; t += p.stride) {
    const int64_t b = t / a.rows, i = t - b * a.rows;
    const int64_t at = i + (a.lengths != nullptr ? a.lengths[b] : 0);
    S* out;  // the kind's row of the output
    if (sl.kind == 0) out = static_cast<S*>(a.q) + b * a.sq + i * a.ldq;
    else if (at < 0 || at >= a.capacity) continue;  // uniform: no such row
    else if (sl.kind == 1) out = static_cast<S*>(a.k) + b * a.sk + at * a.ldk;
    else out = static_cast<S*>(a.v) + b * a.sv + at * a.ldv;
    float c[PL][V], s[PL][V];
    if (sl.kind < 2) angles<V, PL>(a, a.positions != nullptr ? (int64_t)a.positions[t] : at, ln.tix, c, s);
    const S* row = static_cast<const S*>(a.x) + t * a.ldx + head_col(a, sl.kind, sl.first);
    for (int h0 = 0; h0 < sl.count; h0 += hpw) {
      const int h = h0 + hg;
      const bool live = h < sl.count;
      float xa[PL][V], xb[PL][V];
#pragma unroll
      for (int u = 0; u < PL; ++u) {
        Vec<T, V> va, vb;
        va.zero(), vb.zero();
        if (live && ln.ca[u] >= 0) va.load(row, (int64_t)h * D + ln.ca[u]);
        if (live && ln.cb[u] >= 0) vb.load(row, (int64_t)h * D + ln.cb[u]);
#pragma unroll
        for (int e = 0; e < V; ++e) xa[u][e] = va.get(e), xb[u][e] = vb.get(e);
      }
      if (sl.kind < 2) {
        if (a.layer) {
          float m = 0.f;
#pragma unroll
          for (int u = 0; u < PL; ++u)
#pragma unroll
            for (int e = 0; e < V; ++e) m += xa[u][e] + xb[u][e];
          m = sum_lanes(m, L) * inv_d;
#pragma unroll
          for (int u = 0; u < PL; ++u)
#pragma unroll
            for (int e = 0; e < V; ++e) {
              xa[u][e] = ln.ca[u] >= 0 ? xa[u][e] - m : 0.f;
              xb[u][e] = ln.cb[u] >= 0 ? xb[u][e] - m : 0.f;
            }
        }
        float q = 0.f;
#pragma unroll
        for (int u = 0; u < PL; ++u)
#pragma unroll
          for (int e = 0; e < V; ++e) q += xa[u][e] * xa[u][e] + xb[u][e] * xb[u][e];
        const float r = 1.0f / sqrtf(sum_lanes(q, L) * inv_d + a.eps);
#pragma unroll
        for (int u = 0; u < PL; ++u) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            xa[u][e] *= r;
            xb[u][e] *= r;
            if (a.weight != nullptr) {
              xa[u][e] *= wa[u].get(e);
              xb[u][e] *= wb[u].get(e);
            }
            if (a.bias != nullptr) {
              xa[u][e] += ba[u].get(e);
              xb[u][e] += bb[u].get(e);
            }
          }
          if (ln.tix[u] >= 0) turn<V, NEXT>(xa[u], xb[u], c[u], s[u]);
        }
      }
      const int64_t col = (int64_t)(sl.first + h) * D;
#pragma unroll
      for (int u = 0; u < PL; ++u) {
        if (live && ln.ca[u] >= 0) Vec<T, V>::store(out, col + ln.ca[u], xa[u]);
        if (live && ln.cb[u] >= 0) Vec<T, V>::store(out, col + ln.cb[u], xb[u]);
      }
    }
  }
}

// part: [block][dw | db][D] fp32, blocks of value slices none.
template <typename T, int V, int PL, bool PAIRS>
__global__ __launch_bounds__(256) void qk_norm_rope_backward_kernel(NormRopeParams p) {
  const NormRopeArgs& a = p.a;
  constexpr bool NEXT = PAIRS && V > 1;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slices = p.nq + p.nk + p.nv;
  const Slice sl = slice_of(p, (int)(blockIdx.x % (unsigned)slices));
  const int L = 1 << p.lg, D = a.D, hpw = 64 >> p.lg, hg = lane >> p.lg;
  Lanes<V, PL, PAIRS> ln;
  ln.set(lane & (L - 1), L, D, a.rot);
  Vec<T, V> wa[PL], wb[PL];
  float sa[2][PL][V], sb[2][PL][V];  // this lane's sums of dw, db
#pragma unroll
  for (int u = 0; u < PL; ++u) {
    wa[u].zero(), wb[u].zero();
    if (a.weight != nullptr && sl.kind < 2) {
      if (ln.ca[u] >= 0) wa[u].load(a.weight, sl.kind * D + ln.ca[u]);
      if (ln.cb[u] >= 0) wb[u].load(a.weight, sl.kind * D + ln.cb[u]);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) sa[0][u][e] = sa[1][u][e] = sb[0][u][e] = sb[1][u][e] = 0.f;
  }
  const float inv_d = 1.0f / (float)D;
  const int64_t tokens = a.batch * a.rows;
  typedef typename Elem<T>::storage S;
  for (int64_t t = (int64_t)(blockIdx.x / (unsigned)slices) * 4 + wave; t < tokens; t += p.stride) {
    const int64_t b = t / a.rows, i = t - b * a.rows;
    const int64_t col0 = head_col(a, sl.kind, sl.first);
    const S* grow = static_cast<const S*>(a.g) + t * a.ldg + col0;
    const S* row = static_cast<const S*>(a.x) + t * a.ldx + col0;
    S* out = static_cast<S*>(a.q) + t * a.ldq + col0;
    float c[PL][V], s[PL][V];
    if (sl.kind < 2) {
      angles<V, PL>(a, a.positions != nullptr ? (int64_t)a.positions[t] : i, ln.tix, c, s);
#pragma unroll
      for (int u = 0; u < PL; ++u)
#pragma unroll
        for (int e = 0; e < V; ++e) s[u][e] = -s[u][e];  // turned back
    }
    for (int h0 = 0; h0 < sl.count; h0 += hpw) {
      const int h = h0 + hg;
      const bool live = h < sl.count;
      float da[PL][V], db[PL][V], xa[PL][V], xb[PL][V];
#pragma unroll
      for (int u = 0; u < PL; ++u) {
        Vec<T, V> va, vb, ga, gb;
        va.zero(), vb.zero(), ga.zero(), gb.zero();
        if (live && ln.ca[u] >= 0) {
          ga.load(grow, (int64_t)h * D + ln.ca[u]);
          if (sl.kind < 2) va.load(row, (int64_t)h * D + ln.ca[u]);
        }
        if (live && ln.cb[u] >= 0) {
          gb.load(grow, (int64_t)h * D + ln.cb[u]);
          if (sl.kind < 2) vb.load(row, (int64_t)h * D + ln.cb[u]);
        }
#pragma unroll
        for (int e = 0; e < V; ++e)
          xa[u][e] = va.get(e), xb[u][e] = vb.get(e), da[u][e] = ga.get(e), db[u][e] = gb.get(e);
      }
      if (sl.kind < 2) {
        if (a.layer) {
          float m = 0.f;
#pragma unroll
          for (int u = 0; u < PL; ++u)
#pragma unroll
            for (int e = 0; e < V; ++e) m += xa[u][e] + xb[u][e];
          m = sum_lanes(m, L) * inv_d;
#pragma unroll
          for (int u = 0; u < PL; ++u)
#pragma unroll
            for (int e = 0; e < V; ++e) {
              xa[u][e] = ln.ca[u] >= 0 ? xa[u][e] - m : 0.f;
              xb[u][e] = ln.cb[u] >= 0 ? xb[u][e] - m : 0.f;
            }
        }
        float q = 0.f;
#pragma unroll
        for (int u = 0; u < PL; ++u)
#pragma unroll
          for (int e = 0; e < V; ++e) q += xa[u][e] * xa[u][e] + xb[u][e] * xb[u][e];
        // Lanes past the last head add zeros to the sums, also where eps is 0 (their
        // r would be infinite) or the angles are not finite.
        const float r = live ? 1.0f / sqrtf(sum_lanes(q, L) * inv_d + a.eps) : 0.f;
        float m1 = 0.f, m2 = 0.f;
#pragma unroll
        for (int u = 0; u < PL; ++u) {
          if (live && ln.tix[u] >= 0) turn<V, NEXT>(da[u], db[u], c[u], s[u]);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            xa[u][e] *= r;  // hat
            xb[u][e] *= r;
            sa[0][u][e] += da[u][e] * xa[u][e];
            sb[0][u][e] += db[u][e] * xb[u][e];
            sa[1][u][e] += da[u][e];
            sb[1][u][e] += db[u][e];
            if (a.weight != nullptr) {
              da[u][e] *= wa[u].get(e);
              db[u][e] *= wb[u].get(e);
            }
            m1 += da[u][e] * xa[u][e] + db[u][e] * xb[u][e];
            m2 += da[u][e] + db[u][e];
          }
        }
        m1 = sum_lanes(m1, L) * inv_d;
        m2 = a.layer ? sum_lanes(m2, L) * inv_d : 0.f;
#pragma unroll
        for (int u = 0; u < PL; ++u)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            da[u][e] = r * (da[u][e] - xa[u][e] * m1 - m2);
            db[u][e] = r * (db[u][e] - xb[u][e] * m1 - m2);
          }
      }
#pragma unroll
      for (int u = 0; u < PL; ++u) {
        if (live && ln.ca[u] >= 0) Vec<T, V>::store(out, (int64_t)h * D + ln.ca[u], da[u]);
        if (live && ln.cb[u] >= 0) Vec<T, V>::store(out, (int64_t)h * D + ln.cb[u], db[u]);
      }
    }
  }
  if (a.part == nullptr || sl.kind == 2) return;  // workgroup-uniform
  // Sums over the wave's heads, then over the waves.
  __shared__ float red[4][2][256];
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int u = 0; u < PL; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float x = sa[w][u][e], y = sb[w][u][e];
        for (int off = L; off < 64; off <<= 1) {
          x += __shfl_xor(x, off, 64);
          y += __shfl_xor(y, off, 64);
        }
        if (hg == 0) {
          if (ln.ca[u] >= 0) red[wave][w][ln.ca[u] + e] = x;
          if (ln.cb[u] >= 0) red[wave][w][ln.cb[u] + e] = y;
        }
      }
  __syncthreads();
  for (int j = threadIdx.x; j < 2 * D; j += 256) {
    const int w = j >= D, d = j - w * D;
    a.part[(int64_t)blockIdx.x * 2 * D + j] = (red[0][w][d] + red[1][w][d]) + (red[2][w][d] + red[3][w][d]);
  }
}

// dw, db [2, D] from the blocks' sums: one block of 1024 threads per 32 columns,
// 32 threads of every column; the blocks of one kind are those whose number mod
// slices is in its range.
template <typename T>
__global__ __launch_bounds__(1024) void qk_norm_sums_kernel(NormRopeParams p, unsigned blocks) {
  const NormRopeArgs& a = p.a;
  const int D = a.D, per = (D + 31) / 32, x = threadIdx.x & 31;
  const int kind = blockIdx.x / (2 * per), w = blockIdx.x / per % 2, d = blockIdx.x % per * 32 + x;
  const int row = threadIdx.x >> 5;
  const unsigned slices = p.nq + p.nk + p.nv, first = kind ? p.nq : 0, count = kind ? p.nk : p.nq;
  const unsigned n = blocks / slices * count;
  float v = 0.f;
  if (d < D) {
#pragma unroll 8
    for (unsigned j = row; j < n; j += 32)
      v += a.part[((int64_t)(j / count) * slices + first + j % count) * 2 * D + w * D + d];
  }
  __shared__ float red[32][33];
  red[row][x] = v;
  __syncthreads();
  if (threadIdx.x < 32 && d < D) {
    float s = 0.f;
    for (int j = 0; j < 32; ++j) s += red[j][x];
    void* out = w ? a.db : a.dw;
    if (out != nullptr) static_cast<typename Elem<T>::storage*>(out)[kind * D + d] = Elem<T>::from_f32(s);
  }
}

// The widest chunk that the sizes take: chunks divide the head and, in twos,
// what is rotated of it.  Backward at most 4 columns (124 registers, four waves a
// SIMD): with 8, the sums of both parameters and the operands take 231, and half
// as many waves are there to hide the memory's latency.  (The kernel takes either
// norm at run time and sums both parameters; one for the rms norm without its
// bias would take 94, and 150 with 8 columns.  None is built.)
static int chunk_of(int D, int rot, bool back) {
  if (!back && D % 8 == 0 && rot % 16 == 0) return 8;
  if (D % 4 == 0 && rot % 8 == 0) return 4;
  return 1;
}

// Fills the split of the work; returns its blocks.
static unsigned norm_rope_split(NormRopeParams& p, bool back) {
  const NormRopeArgs& a = p.a;
  const int V = chunk_of(a.D, a.rot, back);
  int pairs = a.rot / (2 * V) + (a.D - a.rot + 2 * V - 1) / (2 * V);
  p.lg = 0;
  while ((1 << p.lg) < pairs && p.lg < 6) ++p.lg;
  const int hpw = 64 >> p.lg;
  const int64_t tokens = a.batch * a.rows, cus = cu_count_current();
  // One pass of the wave over a slice where tokens are few (decoding: latency),
  // four where they fill the chip: the angles are loaded once for them.
  p.per = hpw * (tokens < 16 * cus ? 1 : 4);
  auto cdiv = [](int64_t x, int64_t y) { return (x + y - 1) / y; };
  p.nq = (int)cdiv(a.heads, p.per);
  p.nk = (int)cdiv(a.kv_heads, p.per);
  p.nv = a.v != nullptr ? p.nk : 0;
  const int64_t slices = p.nq + p.nk + p.nv;
  // Blocks of four tokens at a time.  Forward up to 64 a CU and slice; backward
  // 4 a CU over all slices, what the registers let run at once, since each
  // leaves sums to be added (8 a CU: the same time here, twice the sums).
  int64_t groups = cdiv(tokens, 4);
  const int64_t most = back ? cdiv(4 * cus, slices) : 64 * cus;
  if (groups > most) groups = most;
  const int64_t fit = ((int64_t(1) << 24) - 1) / slices;  // a launch holds fewer than 2^32 threads
  if (groups > fit) groups = fit;
  if (groups < 1) groups = 1;
  p.stride = groups * 4;
  return (unsigned)(groups * slices);
}

int64_t norm_rope_work(int64_t batch, int64_t rows, int heads, int kv_heads, int D, int rot) {
  NormRopeParams p{};
  p.a.batch = batch, p.a.rows = rows, p.a.heads = heads, p.a.kv_heads = kv_heads, p.a.D = D, p.a.rot = rot;
  p.a.v = &p;  // not followed
  return (int64_t)norm_rope_split(p, true) * 2 * D * 4;
}

NormRopePlan norm_rope_plan(const NormRopeArgs& a, bool back) {
  NormRopeParams p{};
  p.a = a;
  const unsigned blocks = norm_rope_split(p, back);
  return {chunk_of(a.D, a.rot, back), blocks};
}

template <typename T, int V, int PL>
static void launch_norm_rope_v(const NormRopeParams& p, bool back, unsigned blocks, hipStream_t st) {
  const dim3 g(blocks), b(256);
  if (back) {
    if (p.a.pairs) hipLaunchKernelGGL((qk_norm_rope_backward_kernel<T, V, PL, true>), g, b, 0, st, p);
    else hipLaunchKernelGGL((qk_norm_rope_backward_kernel<T, V, PL, false>), g, b, 0, st, p);
  } else {
    if (p.a.pairs) hipLaunchKernelGGL((qk_norm_rope_kernel<T, V, PL, true>), g, b, 0, st, p);
    else hipLaunchKernelGGL((qk_norm_rope_kernel<T, V, PL, false>), g, b, 0, st, p);
  }
}

template <typename T>
static void launch_norm_rope_8(const NormRopeParams& p, unsigned blocks, hipStream_t st) {
  if (p.a.pairs) hipLaunchKernelGGL((qk_norm_rope_kernel<T, 8, 1, true>), dim3(blocks), dim3(256), 0, st, p);
  else hipLaunchKernelGGL((qk_norm_rope_kernel<T, 8, 1, false>), dim3(blocks), dim3(256), 0, st, p);
}

template <typename T>
static int launch_norm_rope_t(const NormRopeArgs& a, bool back, hipStream_t st) {
  NormRopeParams p{};
  p.a = a;
  const unsigned blocks = norm_rope_split(p, back);
  switch (chunk_of(a.D, a.rot, back)) {
    case 8: launch_norm_rope_8<T>(p, blocks, st); break;
    case 4: launch_norm_rope_v<T, 4, 1>(p, back, blocks, st); break;
    default: launch_norm_rope_v<T, 1, 2>(p, back, blocks, st); break;
  }
  int rc = check_launch("query and key norm");
  if (rc != SF_OK || !back || a.part == nullptr) return rc;
  hipLaunchKernelGGL((qk_norm_sums_kernel<T>), dim3(4 * ((a.D + 31) / 32)), dim3(1024), 0, st, p, blocks);
  return check_launch("query and key norm sums");
}

int launch_norm_rope(const NormRopeArgs& a, sf_dtype dt, bool back, hipStream_t st) {
  switch (dt) {
    case SF_F16: return launch_norm_rope_t<F16>(a, back, st);
    case SF_BF16: return launch_norm_rope_t<BF16>(a, back, st);
    default: return launch_norm_rope_t<float>(a, back, st);
  }
}

}  // namespace sf
