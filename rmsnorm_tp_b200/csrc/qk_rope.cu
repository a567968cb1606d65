// Norms of query and key heads with the position rotation in the same pass,
// the same pass written into a paged cache, and the backward pass.
//
//   forward   y = R(p) (x inv w),  inv = rsqrt(mean_D(x^2) + eps)
//   backward  g = R(p)^T dy;  dx = inv g w - x inv^3 mean_D(g w x);
//             dw = sum over tokens and heads of g x inv
//   cache     a row's amax gives its scale, its codes are e4m3(y * 448 / amax)
#include "heads_common.cuh"

namespace rtp {
namespace {

struct Rows {            // one [tokens, heads, head_dim] operand
  const void* p;
  int64_t st, sh;        // token and head stride, elements
};
struct OutRows {
  void* p;
  int64_t st, sh;
};

struct QkArgs {
  Rows q, k, v;
  OutRows qo, ko;
  const void* qw;
  const void* kw;
  const float* rope;
  const int64_t* positions;
  const int64_t* slots;
  void* kc;              // cache
  void* vc;
  float* ks;
  float* vs;
  int64_t tokens, max_pos, num_slots;
  int page, hq, hk, d, r;
  int interleaved, norm, e4m3;
  float eps;
};

struct QkBackArgs {
  Rows dqo, dko, q, k;
  void* dq;
  void* dk;
  const void* qw;
  const void* kw;
  const float* rope;
  const int64_t* positions;
  float* ws;             // [grid][2 * d] fp32 partials of dweight
  int64_t tokens, max_pos;
  int hq, hk, d, r;
  int interleaved, norm;
  float eps;
};

constexpr int kBlock = 256;
constexpr int kWarps = kBlock / 32;

// Elements of pair u of a head: a turned pair for u < r / 2, else two (or one)
// neighbours that are not turned; `b` is -1 where the head ends on `a`.
__device__ __forceinline__ void pair_of(int u, int d, int r, int interleaved, int& a, int& b) {
  const int half = r / 2;
  if (u < half) {
    a = interleaved ? 2 * u : u;
    b = interleaved ? 2 * u + 1 : u + half;
  } else {
    a = r + 2 * (u - half);
    b = a + 1 < d ? a + 1 : -1;
  }
}

// Element offset of a cache row.
__device__ __forceinline__ int64_t cache_row(int64_t slot, int head, const QkArgs& a) {
  int64_t pg;
  int off;
  page_of(slot, a.page, a.num_slots, pg, off);
  return (pg * a.hk + head) * a.page + off;
}

// ---- any head_dim, alignment and stride: one warp per row ----------------------
// Lane l holds the pairs l, l + 32, ...; a row is read twice (its sum of squares,
// then its elements), the second time from L1.
template <typename T, bool kWrite>
__global__ void __launch_bounds__(kBlock) qk_rope_any_kernel(const __grid_constant__ QkArgs a) {
  ptx::grid_dep_wait();
  const int tid = thread_here(), lane = tid & 31;
  const int heads = a.hq + a.hk + (kWrite ? a.hk : 0);
  const int64_t row = (int64_t)blockIdx.x * kWarps + (tid >> 5);
  if (row >= a.tokens * heads) return;
  const int64_t t = (unsigned)row / (unsigned)heads;   // at most 2^31 rows
  const int h = (int)(row - t * heads);
  const bool is_q = h < a.hq, is_v = kWrite && h >= a.hq + a.hk;
  const int hh = is_q ? h : is_v ? h - a.hq - a.hk : h - a.hq;
  const Rows& in = is_q ? a.q : is_v ? a.v : a.k;
  const T* x = static_cast<const T*>(in.p) + t * in.st + hh * in.sh;
  const T* w = static_cast<const T*>(is_q ? a.qw : a.kw);
  const int pairs = a.r / 2 + (a.d - a.r + 1) / 2;
  const int64_t pos = a.positions[t];
  const bool known = pos >= 0 && pos < a.max_pos;
  const float* turn = a.rope + (known ? pos : 0) * a.r;

  float inv = 1.f;
  if (a.norm && !is_v) {
    float ss = 0.f;
    for (int i = lane; i < a.d; i += 32) {
      const float f = Pack<T>::to_f(x[i]);
      ss = fmaf(f, f, ss);
    }
    inv = rsqrtf(warp_allreduce_sum(ss) / (float)a.d + a.eps);
  }
  auto value = [&](int u, int& ia, int& ib, float& ya, float& yb) {
    pair_of(u, a.d, a.r, a.interleaved, ia, ib);
    ya = Pack<T>::to_f(x[ia]);
    yb = ib >= 0 ? Pack<T>::to_f(x[ib]) : 0.f;
    if (is_v) return;
    if (a.norm) {
      ya = (ya * inv) * Pack<T>::to_f(w[ia]);
      if (ib >= 0) yb = (yb * inv) * Pack<T>::to_f(w[ib]);
    }
    if (u < a.r / 2) {
      const float c = known ? turn[u] : quiet_nan(), s = known ? turn[a.r / 2 + u] : quiet_nan();
      const float p = ya * c - yb * s;
      yb = ya * s + yb * c;
      ya = p;
    }
  };

  if (!kWrite || is_q) {
    const OutRows& o = is_q ? a.qo : a.ko;
    T* y = static_cast<T*>(o.p) + t * o.st + hh * o.sh;
    for (int u = lane; u < pairs; u += 32) {
      int ia, ib;
      float ya, yb;
      value(u, ia, ib, ya, yb);
      y[ia] = Pack<T>::from_f(ya);
      if (ib >= 0) y[ib] = Pack<T>::from_f(yb);
    }
    return;
  }
  const int64_t slot = a.slots[t];
  if (slot < 0 || slot >= a.num_slots) return;
  const int64_t at = cache_row(slot, hh, a);
  void* cache = is_v ? a.vc : a.kc;
  if (!a.e4m3) {
    T* y = static_cast<T*>(cache) + at * a.d;
    for (int u = lane; u < pairs; u += 32) {
      int ia, ib;
      float ya, yb;
      value(u, ia, ib, ya, yb);
      y[ia] = Pack<T>::from_f(ya);
      if (ib >= 0) y[ib] = Pack<T>::from_f(yb);
    }
    return;
  }
  float most = kE4M3Floor;
  for (int u = lane; u < pairs; u += 32) {
    int ia, ib;
    float ya, yb;
    value(u, ia, ib, ya, yb);
    most = fmaxf(most, fmaxf(fabsf(ya), fabsf(yb)));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
  const float to = kE4M3Max / most;
  unsigned char* y = static_cast<unsigned char*>(cache) + at * a.d;
  for (int u = lane; u < pairs; u += 32) {
    int ia, ib;
    float ya, yb;
    value(u, ia, ib, ya, yb);
    y[ia] = e4m3_of(ya * to);
    if (ib >= 0) y[ib] = e4m3_of(yb * to);
  }
  if (lane == 0) (is_v ? a.vs : a.ks)[at] = most / kE4M3Max;
}

// One CTA per 1/gridDim-th of the rows of each operand; every lane adds its
// pairs' dw into its warp's own slice of shared memory, the warps' slices are
// added in warp order.
template <typename T>
__global__ void __launch_bounds__(kBlock)
qk_rope_backward_any_kernel(const __grid_constant__ QkBackArgs a) {
  extern __shared__ float dw[];     // [kWarps][d]
  ptx::grid_dep_wait();
  const int tid = thread_here(), lane = tid & 31, warp = tid >> 5;
  const int pairs = a.r / 2 + (a.d - a.r + 1) / 2;
  float* mine = dw + warp * a.d;
  for (int part = 0; part < 2; ++part) {
    const int heads = part == 0 ? a.hq : a.hk;
    const Rows& xr = part == 0 ? a.q : a.k;
    const Rows& gr = part == 0 ? a.dqo : a.dko;
    T* dx = static_cast<T*>(part == 0 ? a.dq : a.dk);
    const T* w = static_cast<const T*>(part == 0 ? a.qw : a.kw);
    if (a.norm)
      for (int i = lane; i < a.d; i += 32) mine[i] = 0.f;
    __syncwarp();
    const int64_t rows = a.tokens * heads, step = (int64_t)gridDim.x * kWarps;
    for (int64_t row = (int64_t)blockIdx.x * kWarps + warp; row < rows; row += step) {
      const int64_t t = row / heads;
      const int h = (int)(row - t * heads);
      const T* x = a.norm ? static_cast<const T*>(xr.p) + t * xr.st + h * xr.sh : nullptr;
      const T* dy = static_cast<const T*>(gr.p) + t * gr.st + h * gr.sh;
      const int64_t pos = a.positions[t];
      const bool known = pos >= 0 && pos < a.max_pos;
      const float* turn = a.rope + (known ? pos : 0) * a.r;
      auto value = [&](int u, int& ia, int& ib, float& ga, float& gb) {
        pair_of(u, a.d, a.r, a.interleaved, ia, ib);
        ga = Pack<T>::to_f(dy[ia]);
        gb = ib >= 0 ? Pack<T>::to_f(dy[ib]) : 0.f;
        if (u < a.r / 2) {
          const float c = known ? turn[u] : quiet_nan(), s = known ? turn[a.r / 2 + u] : quiet_nan();
          const float p = ga * c + gb * s;
          gb = gb * c - ga * s;
          ga = p;
        }
      };
      float inv = 1.f, k = 0.f;
      if (a.norm) {
        float ss = 0.f, sg = 0.f;
        for (int u = lane; u < pairs; u += 32) {
          int ia, ib;
          float ga, gb;
          value(u, ia, ib, ga, gb);
          const float xa = Pack<T>::to_f(x[ia]), xb = ib >= 0 ? Pack<T>::to_f(x[ib]) : 0.f;
          const float wa = Pack<T>::to_f(w[ia]), wb = ib >= 0 ? Pack<T>::to_f(w[ib]) : 0.f;
          ss = fmaf(xa, xa, fmaf(xb, xb, ss));
          sg = fmaf(ga * wa, xa, fmaf(gb * wb, xb, sg));
        }
        ss = warp_allreduce_sum(ss);
        sg = warp_allreduce_sum(sg);
        inv = rsqrtf(ss / (float)a.d + a.eps);
        k = inv * inv * inv * (sg / (float)a.d);
      }
      T* y = dx + row * a.d;
      for (int u = lane; u < pairs; u += 32) {
        int ia, ib;
        float ga, gb;
        value(u, ia, ib, ga, gb);
        if (!a.norm) {
          y[ia] = Pack<T>::from_f(ga);
          if (ib >= 0) y[ib] = Pack<T>::from_f(gb);
          continue;
        }
        const float xa = Pack<T>::to_f(x[ia]);
        y[ia] = Pack<T>::from_f(inv * ga * Pack<T>::to_f(w[ia]) - xa * k);
        mine[ia] += ga * xa * inv;
        if (ib >= 0) {
          const float xb = Pack<T>::to_f(x[ib]);
          y[ib] = Pack<T>::from_f(inv * gb * Pack<T>::to_f(w[ib]) - xb * k);
          mine[ib] += gb * xb * inv;
        }
      }
    }
    if (!a.norm) continue;
    __syncthreads();
    for (int i = tid; i < a.d; i += kBlock) {
      float s = 0.f;
      for (int v = 0; v < kWarps; ++v) s += dw[v * a.d + i];
      a.ws[((int64_t)blockIdx.x * 2 + part) * a.d + i] = s;
    }
    __syncthreads();
  }
}

// ---- 16-byte vectors: a head's row in the registers of a group of lanes ------------
//
// A lane holds one unit, two 16-byte vectors of the row chosen so that the turn stays
// inside the lane: elements [8 j, 8 j + 8) and their partners half a rotary_dim on
// (neighbouring vectors where pairs are interleaved or not turned). head_dim 128 in
// bf16 takes 8 lanes, so a warp works on 4 rows at once; cosines, sines and weights stay
// in registers over the rows of a token. Bound by HBM: each row is read once and written
// once; the next row's vectors are in flight while a row is computed.
template <typename T>
struct UnitOf {
  int ea, eb;            // first elements of the two vectors
  bool on, turned;
  __device__ __forceinline__ UnitOf(int j, int d, int r, int interleaved) {
    constexpr int E = Pack<T>::kE;
    on = j * 2 * E < d;
    turned = j * 2 * E < r;
    if (interleaved || !turned) {
      ea = j * 2 * E;
      eb = ea + E;
    } else {
      ea = j * E;
      eb = ea + r / 2;
    }
  }
};

// Cosines and sines of a unit: table columns [j E, j E + E) and rotary_dim / 2 on, in
// either pairing.
template <typename T>
struct Turn {
  static constexpr int E = Pack<T>::kE;
  float c[E], s[E];
  __device__ __forceinline__ void load(const float* rope, int64_t pos, int64_t max_pos, int r, int j) {
    const bool known = pos >= 0 && pos < max_pos;
    const float4* row = reinterpret_cast<const float4*>(rope + (known ? pos : 0) * r + j * E);
    const float4* row2 = reinterpret_cast<const float4*>(rope + (known ? pos : 0) * r + r / 2 + j * E);
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {
      const float4 a = __ldg(row + i), b = __ldg(row2 + i);
      c[4 * i] = a.x, c[4 * i + 1] = a.y, c[4 * i + 2] = a.z, c[4 * i + 3] = a.w;
      s[4 * i] = b.x, s[4 * i + 1] = b.y, s[4 * i + 2] = b.z, s[4 * i + 3] = b.w;
    }
    if (!known)
#pragma unroll
      for (int i = 0; i < E; ++i) c[i] = s[i] = quiet_nan();
  }
  // (a, b) turned by the angle (back: by its negative).
  template <bool kBack>
  __device__ __forceinline__ void apply(float (&a)[E], float (&b)[E], int interleaved) const {
    if (!interleaved) {
#pragma unroll
      for (int i = 0; i < E; ++i) pair<kBack>(a[i], b[i], c[i], s[i]);
    } else {
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        pair<kBack>(a[2 * i], a[2 * i + 1], c[i], s[i]);
        pair<kBack>(b[2 * i], b[2 * i + 1], c[E / 2 + i], s[E / 2 + i]);
      }
    }
  }
  template <bool kBack>
  static __device__ __forceinline__ void pair(float& a, float& b, float c, float s) {
    const float x = kBack ? a * c + b * s : a * c - b * s;
    b = kBack ? b * c - a * s : a * s + b * c;
    a = x;
  }
};

template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
template <int L>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  return v;
}

// Rows are numbered over tokens, then heads (q, k, v); a warp takes `run` groups of
// 32 / L neighbouring rows.
template <typename T, int L, bool kWrite>
__global__ void __launch_bounds__(kBlock) qk_rope_kernel(const __grid_constant__ QkArgs a, int run) {
  constexpr int E = Pack<T>::kE, kRows = 32 / L;
  ptx::grid_dep_wait();
  ptx::grid_dep_launch_dependents();
  const int tid = thread_here(), lane = tid & 31, j = lane % L;
  const UnitOf<T> u(j, a.d, a.r, a.interleaved);
  const int heads = a.hq + a.hk + (kWrite ? a.hk : 0);
  const int64_t rows = a.tokens * heads;
  int64_t row = ((int64_t)blockIdx.x * kWarps + (tid >> 5)) * run * kRows + lane / L;
  int64_t t = (unsigned)row / (unsigned)heads;   // at most 2^31 rows and a CTA's more
  int h = (int)(row - t * heads);
  uint4 wq[2] = {}, wk[2] = {};
  if (a.norm && u.on) {
    wq[0] = ptx::ld_cached_v4(static_cast<const T*>(a.qw) + u.ea);
    wq[1] = ptx::ld_cached_v4(static_cast<const T*>(a.qw) + u.eb);
    wk[0] = ptx::ld_cached_v4(static_cast<const T*>(a.kw) + u.ea);
    wk[1] = ptx::ld_cached_v4(static_cast<const T*>(a.kw) + u.eb);
  }
  auto fetch = [&](int64_t t, int h, bool live, uint4 (&x)[2]) {
    if (!live || !u.on) {
      x[0] = x[1] = make_uint4(0u, 0u, 0u, 0u);
      return;
    }
    const T* p;
    if (h < a.hq) p = static_cast<const T*>(a.q.p) + t * a.q.st + h * a.q.sh;
    else if (!kWrite || h < a.hq + a.hk) p = static_cast<const T*>(a.k.p) + t * a.k.st + (h - a.hq) * a.k.sh;
    else p = static_cast<const T*>(a.v.p) + t * a.v.st + (h - a.hq - a.hk) * a.v.sh;
    x[0] = ptx::ld_stream_v4(p + u.ea);
    x[1] = ptx::ld_stream_v4(p + u.eb);
  };
  Turn<T> turn;
  int64_t turn_of = -1, slot = -1;
  uint4 next[2];
  fetch(t, h, row < rows, next);
#pragma unroll 1
  for (int i = 0; i < run; ++i) {
    const bool live = row < rows;
    if (!__any_sync(0xFFFFFFFFu, live)) break;
    if (live && t != turn_of) {
      turn_of = t;
      const int64_t pos = a.positions[t];
      if (kWrite) slot = a.slots[t];
      if (u.turned) turn.load(a.rope, pos, a.max_pos, a.r, j);
    }
    const uint4 x[2] = {next[0], next[1]};
    const int64_t t_now = t;
    const int h_now = h;
    row += kRows;
    h += kRows;
    while (h >= heads) {
      h -= heads;
      ++t;
    }
    if (i + 1 < run) fetch(t, h, row < rows, next);

    const bool is_q = h_now < a.hq, is_v = kWrite && h_now >= a.hq + a.hk;
    float ya[E], yb[E];
    Pack<T>::unpack(x[0], ya);
    Pack<T>::unpack(x[1], yb);
    if (a.norm) {
      float sa = 0.f, sb = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        sa = fmaf(ya[e], ya[e], sa);
        sb = fmaf(yb[e], yb[e], sb);
      }
      const float inv = rsqrtf(lanes_sum<L>(sa + sb) / (float)a.d + a.eps);
      if (!is_v) {
        float wa[E], wb[E];
        Pack<T>::unpack(is_q ? wq[0] : wk[0], wa);
        Pack<T>::unpack(is_q ? wq[1] : wk[1], wb);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          ya[e] = (ya[e] * inv) * wa[e];
          yb[e] = (yb[e] * inv) * wb[e];
        }
      }
    }
    if (u.turned && !is_v) turn.template apply<false>(ya, yb, a.interleaved);
    if (!kWrite || is_q) {
      if (live && u.on) {
        T* y = is_q ? static_cast<T*>(a.qo.p) + t_now * a.qo.st + h_now * a.qo.sh
                    : static_cast<T*>(a.ko.p) + t_now * a.ko.st + (h_now - a.hq) * a.ko.sh;
        ptx::st_v4(y + u.ea, Pack<T>::pack(ya));
        ptx::st_v4(y + u.eb, Pack<T>::pack(yb));
      }
      if (!kWrite) continue;
    }
    if constexpr (kWrite) {
      const bool keep = live && !is_q && slot >= 0 && slot < a.num_slots;
      const int64_t at = keep ? cache_row(slot, is_v ? h_now - a.hq - a.hk : h_now - a.hq, a) : 0;
      void* cache = is_v ? a.vc : a.kc;
      if (!a.e4m3) {
        if (keep && u.on) {
          T* y = static_cast<T*>(cache) + at * a.d;
          ptx::st_v4(y + u.ea, Pack<T>::pack(ya));
          ptx::st_v4(y + u.eb, Pack<T>::pack(yb));
        }
        continue;
      }
      if (!__any_sync(0xFFFFFFFFu, keep)) continue;
      float most = kE4M3Floor;
#pragma unroll
      for (int e = 0; e < E; ++e) most = fmaxf(most, fmaxf(fabsf(ya[e]), fabsf(yb[e])));
      most = lanes_max<L>(most);
      if (keep && u.on) {
        const float to = kE4M3Max / most;
        unsigned char* y = static_cast<unsigned char*>(cache) + at * a.d;
        uint32_t ca[E / 4], cb[E / 4];
#pragma unroll
        for (int e = 0; e < E / 4; ++e) {
          ca[e] = e4m3x2_of(ya[4 * e] * to, ya[4 * e + 1] * to) |
                  (uint32_t)e4m3x2_of(ya[4 * e + 2] * to, ya[4 * e + 3] * to) << 16;
          cb[e] = e4m3x2_of(yb[4 * e] * to, yb[4 * e + 1] * to) |
                  (uint32_t)e4m3x2_of(yb[4 * e + 2] * to, yb[4 * e + 3] * to) << 16;
        }
        if constexpr (E == 8) {
          *reinterpret_cast<uint2*>(y + u.ea) = make_uint2(ca[0], ca[1]);
          *reinterpret_cast<uint2*>(y + u.eb) = make_uint2(cb[0], cb[1]);
        } else {
          *reinterpret_cast<uint32_t*>(y + u.ea) = ca[0];
          *reinterpret_cast<uint32_t*>(y + u.eb) = cb[0];
        }
        if (j == 0) (is_v ? a.vs : a.ks)[at] = most / kE4M3Max;
      }
    }
  }
}

// The backward: g and x in registers, dw summed per lane over the CTA's rows (a run of
// each operand's rows for each warp), then over the warp's row groups and the warps in a
// fixed order.
template <typename T, int L>
__global__ void __launch_bounds__(kBlock, 2)
qk_rope_backward_kernel(const __grid_constant__ QkBackArgs a) {
  constexpr int E = Pack<T>::kE, kRows = 32 / L;
  extern __shared__ float dw[];     // [kWarps][d]
  ptx::grid_dep_wait();
  ptx::grid_dep_launch_dependents();
  const int tid = thread_here(), lane = tid & 31, warp = tid >> 5, j = lane % L;
  const UnitOf<T> u(j, a.d, a.r, a.interleaved);
  const int64_t workers = (int64_t)gridDim.x * kWarps, me = (int64_t)blockIdx.x * kWarps + warp;
  const float rd = 1.f / (float)a.d;
#pragma unroll 1
  for (int part = 0; part < 2; ++part) {
    const int heads = part == 0 ? a.hq : a.hk;
    const Rows xr = part == 0 ? a.q : a.k, gr = part == 0 ? a.dqo : a.dko;
    T* dx = static_cast<T*>(part == 0 ? a.dq : a.dk);
    float wa[E] = {}, wb[E] = {}, da[E] = {}, db[E] = {};
    if (a.norm && u.on) {
      const T* w = static_cast<const T*>(part == 0 ? a.qw : a.kw);
      Pack<T>::unpack(ptx::ld_cached_v4(w + u.ea), wa);
      Pack<T>::unpack(ptx::ld_cached_v4(w + u.eb), wb);
    }
    const int64_t rows = a.tokens * heads, groups = (rows + kRows - 1) / kRows;
    const int64_t first = groups * me / workers, end = groups * (me + 1) / workers;
    int64_t row = first * kRows + lane / L;
    int64_t t = row / heads;
    int h = (int)(row - t * heads);
    Turn<T> turn;
    int64_t turn_of = -1;
    uint4 x[2], g[2];
    auto fetch = [&]() {
      x[0] = x[1] = g[0] = g[1] = make_uint4(0u, 0u, 0u, 0u);
      if (row >= rows || !u.on) return;
      const T* p = static_cast<const T*>(gr.p) + t * gr.st + h * gr.sh;
      g[0] = ptx::ld_stream_v4(p + u.ea);
      g[1] = ptx::ld_stream_v4(p + u.eb);
      if (a.norm) {
        p = static_cast<const T*>(xr.p) + t * xr.st + h * xr.sh;
        x[0] = ptx::ld_stream_v4(p + u.ea);
        x[1] = ptx::ld_stream_v4(p + u.eb);
      }
    };
    if (first < end) fetch();
#pragma unroll 1
    for (int64_t i = first; i < end; ++i) {
      const bool live = row < rows;
      if (live && t != turn_of) {
        turn_of = t;
        if (u.turned) turn.load(a.rope, a.positions[t], a.max_pos, a.r, j);
      }
      float xa[E], xb[E], ga[E], gb[E];
      Pack<T>::unpack(x[0], xa);
      Pack<T>::unpack(x[1], xb);
      Pack<T>::unpack(g[0], ga);
      Pack<T>::unpack(g[1], gb);
      T* y = dx + row * a.d;
      row += kRows;
      h += kRows;
      while (h >= heads) {
        h -= heads;
        ++t;
      }
      if (i + 1 < end) fetch();
      if (u.turned && live) turn.template apply<true>(ga, gb, a.interleaved);
      if (a.norm) {
        float ss = 0.f, sg = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          ss = fmaf(xa[e], xa[e], fmaf(xb[e], xb[e], ss));
          sg = fmaf(ga[e] * wa[e], xa[e], fmaf(gb[e] * wb[e], xb[e], sg));
        }
        ss = lanes_sum<L>(ss);
        sg = lanes_sum<L>(sg);
        const float inv = rsqrtf(ss * rd + a.eps);
        const float k = inv * inv * inv * (sg * rd);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float na = ga[e] * inv, nb = gb[e] * inv;
          da[e] = fmaf(na, xa[e], da[e]);
          db[e] = fmaf(nb, xb[e], db[e]);
          ga[e] = na * wa[e] - xa[e] * k;
          gb[e] = nb * wb[e] - xb[e] * k;
        }
      }
      if (live && u.on) {
        ptx::st_v4(y + u.ea, Pack<T>::pack(ga));
        ptx::st_v4(y + u.eb, Pack<T>::pack(gb));
      }
    }
    if (!a.norm) continue;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int o = L; o < 32; o <<= 1) {
        da[e] += __shfl_xor_sync(0xFFFFFFFFu, da[e], o);
        db[e] += __shfl_xor_sync(0xFFFFFFFFu, db[e], o);
      }
    if (lane < L && u.on) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        dw[warp * a.d + u.ea + e] = da[e];
        dw[warp * a.d + u.eb + e] = db[e];
      }
    }
    __syncthreads();
    for (int i = tid; i < a.d; i += kBlock) {
      float s = 0.f;
      for (int v = 0; v < kWarps; ++v) s += dw[v * a.d + i];
      a.ws[((int64_t)blockIdx.x * 2 + part) * a.d + i] = s;
    }
    __syncthreads();
  }
}

// dw of both weights from the CTAs' partials ([parts][2 d]): a CTA has 32 columns, its warps
// the parts w, w + 32, ..., added in that order and then in warp order.
constexpr int kDwWarps = 32;

template <typename T>
__global__ void __launch_bounds__(kDwWarps * 32)
qk_rope_dw_kernel(const float* ws, int parts, int d, T* dqw, T* dkw) {
  __shared__ float s_sum[kDwWarps][32];
  ptx::grid_dep_wait();
  ptx::grid_dep_launch_dependents();
  const int tid = thread_here(), lane = tid & 31, warp = tid >> 5;
  const int col = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (col < 2 * d) {
#pragma unroll 10
    for (int i = warp; i < parts; i += kDwWarps) s += ws[(int64_t)i * 2 * d + col];
  }
  s_sum[warp][lane] = s;
  __syncthreads();
  if (warp != 0 || col >= 2 * d) return;
  s = 0.f;
#pragma unroll
  for (int w = 0; w < kDwWarps; ++w) s += s_sum[w][lane];
  (col < d ? dqw + col : dkw + (col - d))[0] = Pack<T>::from_f(s);
}

// Lanes of a row where the vector kernels take it, else 0 (the kernels for any row):
// units of two whole vectors on both sides of rotary_dim, at most 32 of them, and every
// address a multiple of 16 bytes.
int lanes_of(int d, int r, int eb, uintptr_t addresses, int64_t strides) {
  const int unit = 32 / eb;   // elements
  if (d % unit || r % unit || d / unit > 32) return 0;
  if ((addresses & 15u) || (strides * eb) % 16) return 0;
  const int n = d / unit;
  return n <= 4 ? 4 : n <= 8 ? 8 : n <= 16 ? 16 : 32;
}
uintptr_t bits_of(const void* p) { return reinterpret_cast<uintptr_t>(p); }

template <typename T, bool kWrite>
const void* forward_fn(int lanes) {
  switch (lanes) {
    case 4:
      return reinterpret_cast<const void*>(qk_rope_kernel<T, 4, kWrite>);
    case 8:
      return reinterpret_cast<const void*>(qk_rope_kernel<T, 8, kWrite>);
    case 16:
      return reinterpret_cast<const void*>(qk_rope_kernel<T, 16, kWrite>);
    case 32:
      return reinterpret_cast<const void*>(qk_rope_kernel<T, 32, kWrite>);
    default:
      return reinterpret_cast<const void*>(qk_rope_any_kernel<T, kWrite>);
  }
}
template <typename T>
const void* backward_fn(int lanes) {
  switch (lanes) {
    case 4:
      return reinterpret_cast<const void*>(qk_rope_backward_kernel<T, 4>);
    case 8:
      return reinterpret_cast<const void*>(qk_rope_backward_kernel<T, 8>);
    case 16:
      return reinterpret_cast<const void*>(qk_rope_backward_kernel<T, 16>);
    case 32:
      return reinterpret_cast<const void*>(qk_rope_backward_kernel<T, 32>);
    default:
      return reinterpret_cast<const void*>(qk_rope_backward_any_kernel<T>);
  }
}

// ---- host ----------------------------------------------------------------------

int check_common(const char* who, int64_t tokens, int hq, int hk, int d, int r, int dtype,
                 int64_t max_pos) {
  if (dtype != RMSNORM_TP_F32 && dtype != RMSNORM_TP_BF16 && dtype != RMSNORM_TP_F16)
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: unknown dtype %d", who, dtype);
  if (hq < 1 || hk < 1 || hq > 65536 || hk > 65536)
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: q_heads %d or kv_heads %d outside [1, 65536]", who, hq,
                  hk);
  if (d < 2 || d > RMSNORM_HEAD_DIM_MAX)
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: head_dim %d outside [2, %d]", who, d,
                  RMSNORM_HEAD_DIM_MAX);
  if (r < 2 || r > d || r % 2)
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: rotary_dim %d must be even and in [2, head_dim %d]", who,
                  r, d);
  if (max_pos < 1) return refuse(RMSNORM_TP_ERR_INVALID, "%s: an empty rope table", who);
  if (tokens < 0 || tokens > (int64_t(1) << 31) / (hq + 2 * hk))
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: %lld tokens of %d heads: at most 2^31 rows", who,
                  (long long)tokens, hq + 2 * hk);
  return RMSNORM_TP_OK;
}

int check_forward(const char* who, const rmsnorm_qk_rope_args* a, bool write) {
  if (!a) return refuse(RMSNORM_TP_ERR_INVALID, "%s: NULL arguments", who);
  int rc = check_common(who, a->tokens, a->q_heads, a->kv_heads, a->head_dim, a->rotary_dim, a->dtype,
                        a->max_positions);
  if (rc != RMSNORM_TP_OK) return rc;
  if ((a->q_weight == nullptr) != (a->k_weight == nullptr))
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: one of q_weight and k_weight is NULL", who);
  if (write) {
    rc = check_cache(who, a->cache);
    if (rc != RMSNORM_TP_OK) return rc;
    const rmsnorm_kv_cache* c = a->cache;
    if (c->kv_heads != a->kv_heads || c->head_dim != a->head_dim)
      return refuse(RMSNORM_TP_ERR_INVALID, "%s: a cache of %d heads of %d for %d heads of %d", who,
                    c->kv_heads, c->head_dim, a->kv_heads, a->head_dim);
    if (c->dtype != RMSNORM_KV_E4M3 && c->dtype != a->dtype)
      return refuse(RMSNORM_TP_ERR_INVALID, "%s: a cache of dtype %d for inputs of dtype %d", who,
                    c->dtype, a->dtype);
  }
  if (a->tokens == 0) return RMSNORM_TP_OK;
  if (!a->q || !a->k || !a->q_out || !a->rope || !a->positions || (write ? !a->v || !a->slots : !a->k_out))
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: NULL tensor pointer", who);
  const int eb = elem_bytes(a->dtype);
  const View q = view_of(a->q, a->tokens, a->q_heads, a->head_dim, a->q_strides, eb);
  const View k = view_of(a->k, a->tokens, a->kv_heads, a->head_dim, a->k_strides, eb);
  const View qo = view_of(a->q_out, a->tokens, a->q_heads, a->head_dim, a->q_out_strides, eb);
  const View in[3] = {q, k, view_of(a->v, a->tokens, a->kv_heads, a->head_dim, a->v_strides, eb)};
  for (const View& v : in)
    if (v.base && (v.s0 < 0 || v.s1 < 0))
      return refuse(RMSNORM_TP_ERR_INVALID, "%s: negative stride", who);
  View outs[2] = {qo, view_of(a->k_out, a->tokens, a->kv_heads, a->head_dim, a->k_out_strides, eb)};
  for (int i = 0; i < (write ? 1 : 2); ++i) {
    if (outs[i].s0 < 0 || outs[i].s1 < 0 || !view_apart(outs[i]))
      return refuse(RMSNORM_TP_ERR_INVALID, "%s: rows of %s overlap one another", who,
                    i ? "k_out" : "q_out");
    for (int j = 0; j < (write ? 3 : 2); ++j)
      if (!(i == j && views_same(outs[i], in[j])) && views_overlap(outs[i], in[j]))
        return refuse(RMSNORM_TP_ERR_INVALID, "%s: %s overlaps an input", who, i ? "k_out" : "q_out");
  }
  if (!write && views_overlap(outs[0], outs[1]))
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: q_out overlaps k_out", who);
  return RMSNORM_TP_OK;
}

template <bool kWrite>
int run_forward(const char* who, const rmsnorm_qk_rope_args* in, void* stream) {
  const int rc = check_forward(who, in, kWrite);
  if (rc != RMSNORM_TP_OK || in->tokens == 0) return rc;
  QkArgs a = {};
  a.q = Rows{in->q, in->q_strides[0], in->q_strides[1]};
  a.k = Rows{in->k, in->k_strides[0], in->k_strides[1]};
  a.qo = OutRows{in->q_out, in->q_out_strides[0], in->q_out_strides[1]};
  a.qw = in->q_weight;
  a.kw = in->k_weight;
  a.rope = in->rope;
  a.positions = in->positions;
  a.tokens = in->tokens;
  a.max_pos = in->max_positions;
  a.hq = in->q_heads;
  a.hk = in->kv_heads;
  a.d = in->head_dim;
  a.r = in->rotary_dim;
  a.interleaved = in->interleaved != 0;
  a.norm = in->q_weight != nullptr;
  a.eps = in->eps;
  if (kWrite) {
    const rmsnorm_kv_cache* c = in->cache;
    a.v = Rows{in->v, in->v_strides[0], in->v_strides[1]};
    a.slots = in->slots;
    a.kc = c->k;
    a.vc = c->v;
    a.ks = c->k_scale;
    a.vs = c->v_scale;
    a.page = c->page_size;
    a.num_slots = c->num_pages * c->page_size;
    a.e4m3 = c->dtype == RMSNORM_KV_E4M3;
  } else {
    a.ko = OutRows{in->k_out, in->k_out_strides[0], in->k_out_strides[1]};
  }
  OnDevice on(in->device);
  if (on.err != cudaSuccess) return launch_failed(on.err, who);
  const int64_t rows = a.tokens * (a.hq + a.hk * (kWrite ? 2 : 1));
  uintptr_t bits = bits_of(a.q.p) | bits_of(a.k.p) | bits_of(a.v.p) | bits_of(a.qo.p) | bits_of(a.ko.p) |
                   bits_of(a.qw) | bits_of(a.kw) | bits_of(a.rope);
  int64_t strides = a.q.st | a.q.sh | a.k.st | a.k.sh | a.v.st | a.v.sh | a.qo.st | a.qo.sh | a.ko.st | a.ko.sh;
  const int lanes = lanes_of(a.d, a.r, elem_bytes(in->dtype), bits, strides);
  const void* fn = in->dtype == RMSNORM_TP_F32    ? forward_fn<float, kWrite>(lanes)
                   : in->dtype == RMSNORM_TP_BF16 ? forward_fn<__nv_bfloat16, kWrite>(lanes)
                                                  : forward_fn<__half, kWrite>(lanes);
  // groups of rows for each warp: as many as leave every SM 32 warps, at most 8
  const int64_t groups = lanes ? (rows * lanes + 31) / 32 : rows;
  int run = 1;
  if (lanes) {
    const int64_t full = 32ll * sm_count(in->device);
    run = (int)(groups / (full > 0 ? full : 1));
    run = run < 1 ? 1 : run > 8 ? 8 : run;
  }
  const int64_t blocks = (groups + (int64_t)run * kWarps - 1) / ((int64_t)run * kWarps);
  void* args[] = {&a, &run};
  const cudaError_t e = launch_dependent(fn, dim3((unsigned)blocks), dim3(kBlock), 0, args,
                                         reinterpret_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? RMSNORM_TP_OK : launch_failed(e, who);
}

}  // namespace
}  // namespace rtp

extern "C" {

int rmsnorm_qk_rope_forward(const rmsnorm_qk_rope_args* args, void* stream) {
  return rtp::run_forward<false>("qk_rope_forward", args, stream);
}

int rmsnorm_qk_rope_write(const rmsnorm_qk_rope_args* args, void* stream) {
  return rtp::run_forward<true>("qk_rope_write", args, stream);
}

size_t rmsnorm_qk_rope_backward_workspace_bytes(int32_t head_dim) {
  if (head_dim < 2 || head_dim > RMSNORM_HEAD_DIM_MAX) return 0;
  return (size_t)rtp::kBackwardMaxGrid * 2u * (size_t)head_dim * sizeof(float);
}

int rmsnorm_qk_rope_backward(const rmsnorm_qk_rope_backward_args* in, void* stream) {
  using namespace rtp;
  const char* who = "qk_rope_backward";
  if (!in) return refuse(RMSNORM_TP_ERR_INVALID, "%s: NULL arguments", who);
  int rc = check_common(who, in->tokens, in->q_heads, in->kv_heads, in->head_dim, in->rotary_dim,
                        in->dtype, in->max_positions);
  if (rc != RMSNORM_TP_OK) return rc;
  const bool norm = in->q_weight != nullptr;
  if (norm != (in->k_weight != nullptr))
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: one of q_weight and k_weight is NULL", who);
  if (norm && (!in->dq_weight || !in->dk_weight || !in->workspace ||
               in->workspace_bytes < (int64_t)rmsnorm_qk_rope_backward_workspace_bytes(in->head_dim)))
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: NULL dq_weight or dk_weight, or a workspace of %lld bytes < %zu", who,
                  (long long)in->workspace_bytes,
                  rmsnorm_qk_rope_backward_workspace_bytes(in->head_dim));
  const int eb = elem_bytes(in->dtype);
  if (in->tokens > 0) {
    if (!in->dq_out || !in->dk_out || !in->dq || !in->dk || !in->rope || !in->positions ||
        (norm && (!in->q || !in->k)))
      return refuse(RMSNORM_TP_ERR_INVALID, "%s: NULL tensor pointer", who);
    const int64_t sq[2] = {(int64_t)in->q_heads * in->head_dim, in->head_dim};
    const int64_t sk[2] = {(int64_t)in->kv_heads * in->head_dim, in->head_dim};
    const View dst[2] = {view_of(in->dq, in->tokens, in->q_heads, in->head_dim, sq, eb),
                         view_of(in->dk, in->tokens, in->kv_heads, in->head_dim, sk, eb)};
    const View src[4] = {
        view_of(in->dq_out, in->tokens, in->q_heads, in->head_dim, in->dq_out_strides, eb),
        view_of(in->dk_out, in->tokens, in->kv_heads, in->head_dim, in->dk_out_strides, eb),
        view_of(in->q, in->tokens, in->q_heads, in->head_dim, in->q_strides, eb),
        view_of(in->k, in->tokens, in->kv_heads, in->head_dim, in->k_strides, eb)};
    for (int j = 0; j < (norm ? 4 : 2); ++j) {
      if (src[j].s0 < 0 || src[j].s1 < 0)
        return refuse(RMSNORM_TP_ERR_INVALID, "%s: negative stride", who);
      for (int i = 0; i < 2; ++i)
        if (views_overlap(dst[i], src[j]))
          return refuse(RMSNORM_TP_ERR_INVALID, "%s: %s overlaps an input", who, i ? "dk" : "dq");
    }
    if (views_overlap(dst[0], dst[1]))
      return refuse(RMSNORM_TP_ERR_INVALID, "%s: dq overlaps dk", who);
  }
  OnDevice on(in->device);
  if (on.err != cudaSuccess) return launch_failed(on.err, who);
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int grid = 0;
  if (in->tokens > 0) {
    QkBackArgs a = {};
    a.dqo = Rows{in->dq_out, in->dq_out_strides[0], in->dq_out_strides[1]};
    a.dko = Rows{in->dk_out, in->dk_out_strides[0], in->dk_out_strides[1]};
    a.q = Rows{in->q, in->q_strides[0], in->q_strides[1]};
    a.k = Rows{in->k, in->k_strides[0], in->k_strides[1]};
    a.dq = in->dq;
    a.dk = in->dk;
    a.qw = in->q_weight;
    a.kw = in->k_weight;
    a.rope = in->rope;
    a.positions = in->positions;
    a.ws = static_cast<float*>(in->workspace);
    a.tokens = in->tokens;
    a.max_pos = in->max_positions;
    a.hq = in->q_heads;
    a.hk = in->kv_heads;
    a.d = in->head_dim;
    a.r = in->rotary_dim;
    a.interleaved = in->interleaved != 0;
    a.norm = norm;
    a.eps = in->eps;
    const uintptr_t bits = bits_of(a.dqo.p) | bits_of(a.dko.p) | (norm ? bits_of(a.q.p) | bits_of(a.k.p) : 0) |
                           bits_of(a.dq) | bits_of(a.dk) | bits_of(a.qw) | bits_of(a.kw) | bits_of(a.rope);
    const int64_t strides = a.dqo.st | a.dqo.sh | a.dko.st | a.dko.sh |
                            (norm ? a.q.st | a.q.sh | a.k.st | a.k.sh : 0);
    const int lanes = lanes_of(a.d, a.r, eb, bits, strides);
    const int64_t groups = lanes ? (a.tokens * a.hq * lanes + 31) / 32 : a.tokens * a.hq;
    const int64_t want = (groups + kWarps - 1) / kWarps;
    grid = (int)(want < kBackwardMaxGrid ? want : kBackwardMaxGrid);
    const void* fn = in->dtype == RMSNORM_TP_F32    ? backward_fn<float>(lanes)
                     : in->dtype == RMSNORM_TP_BF16 ? backward_fn<__nv_bfloat16>(lanes)
                                                    : backward_fn<__half>(lanes);
    void* args[] = {&a};
    const size_t smem = norm ? (size_t)kWarps * a.d * sizeof(float) : 0;
    const cudaError_t e = launch_dependent(fn, dim3((unsigned)grid), dim3(kBlock), smem, args, st);
    if (e != cudaSuccess) return launch_failed(e, who);
  }
  if (norm) {   // no tokens: zeros
    const float* ws = static_cast<const float*>(in->workspace);
    int d = in->head_dim;
    void* dqw = in->dq_weight;
    void* dkw = in->dk_weight;
    void* args[] = {&ws, &grid, &d, &dqw, &dkw};
    const void* fn = in->dtype == RMSNORM_TP_F32    ? reinterpret_cast<const void*>(qk_rope_dw_kernel<float>)
                     : in->dtype == RMSNORM_TP_BF16 ? reinterpret_cast<const void*>(qk_rope_dw_kernel<__nv_bfloat16>)
                                                    : reinterpret_cast<const void*>(qk_rope_dw_kernel<__half>);
    const cudaError_t e = launch_dependent(fn, dim3((2 * d + 31) / 32), dim3(kDwWarps * 32), 0, args, st);
    if (e != cudaSuccess) return launch_failed(e, who);
  }
  return RMSNORM_TP_OK;
}

}  // extern "C"
