// Norms of query and key heads with the position rotation in the same pass,
// the same pass written into a paged cache, and the backward pass.
//
//   forward   y = R(p) (x inv w),  inv = rsqrt(mean_D(x^2) + eps)
//   backward  g = R(p)^T dy;  dx = inv g w - x inv^3 mean_D(g w x);
//             dw = sum over tokens and heads of g x inv
//   cache     a row's amax gives its scale, its codes are e4m3(y * 448 / amax)
#include <atomic>

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
  float* ws;             // [grid][d] fp32 partials of dw: the queries' CTAs, then the keys';
                         // NULL: the grid is one cluster and sums dw itself
  void* dqw;
  void* dkw;
  int64_t tokens, max_pos;
  int hq, hk, d, r;
  int interleaved, norm;
  float eps;
};

constexpr int kMaxParts = 1024;        // most CTAs of a backward call: the workspace's rows
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
// then its elements), the second time from L1. Scalar loads bound it: where both
// could run, 8192 tokens of 40 heads of 128 (bf16) take 118 us here and 29.7 in the
// vector kernel, the backward 472 and 53.4. Sizes that only this takes: 8192 tokens of 40
// heads of 80, 40 of them turned (bf16), 142 us and 450 for the backward, 8.8 and 19 times
// their bytes.
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

// All CTAs of the cluster, shared-memory writes before it visible after it.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// *p in the shared memory of CTA `rank` of the cluster.
__device__ __forceinline__ float cluster_load(const float* p, unsigned rank) {
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(ptx::smem_addr(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

// The end of a backward kernel of kW warps: dw[warp][d] added over the CTA's warps and left
// in the workspace for the second kernel, or, where the grid is one cluster, added over the
// CTAs of the operand by its first CTA, in their order, from their shared memory.
template <typename T, int kW>
__device__ __forceinline__ void leave_dw(const QkBackArgs& a, float* dw, int tid, bool is_q, int block, int blocks) {
  for (int i = tid; i < a.d; i += kW * 32) {
    float s = 0.f;
    for (int v = 0; v < kW; ++v) s += dw[v * a.d + i];
    if (a.ws) a.ws[(int64_t)blockIdx.x * a.d + i] = s;
    else dw[i] = s;                      // only this thread reads column i of every warp
  }
  if (a.ws) return;
  cluster_sync();
  if (block == 0)
    for (int i = tid; i < a.d; i += kW * 32) {
      float s = 0.f;
      for (int c = 0; c < blocks; ++c) s += cluster_load(dw + i, blockIdx.x + c);
      static_cast<T*>(is_q ? a.dqw : a.dkw)[i] = Pack<T>::from_f(s);
    }
  cluster_sync();                        // the others' shared memory has been read
}

// CTAs [0, q_blocks) share the queries' rows, the others the keys'; every lane adds its
// pairs' dw into its warp's own slice of shared memory, the warps' slices are added in
// warp order.
template <typename T>
__global__ void __launch_bounds__(kBlock)
qk_rope_backward_any_kernel(const __grid_constant__ QkBackArgs a, int q_blocks) {
  extern __shared__ float dw[];     // [kWarps][d]
  ptx::grid_dep_wait();
  const int tid = thread_here(), lane = tid & 31, warp = tid >> 5;
  const int pairs = a.r / 2 + (a.d - a.r + 1) / 2;
  const bool is_q = (int)blockIdx.x < q_blocks;
  const int blocks = is_q ? q_blocks : gridDim.x - q_blocks, block = is_q ? blockIdx.x : blockIdx.x - q_blocks;
  float* mine = dw + warp * a.d;
  const int heads = is_q ? a.hq : a.hk;
  const Rows& xr = is_q ? a.q : a.k;
  const Rows& gr = is_q ? a.dqo : a.dko;
  T* dx = static_cast<T*>(is_q ? a.dq : a.dk);
  const T* w = static_cast<const T*>(is_q ? a.qw : a.kw);
  if (a.norm)
    for (int i = lane; i < a.d; i += 32) mine[i] = 0.f;
  __syncwarp();
  const int64_t rows = a.tokens * heads, step = (int64_t)blocks * kWarps;
  for (int64_t row = (int64_t)block * kWarps + warp; row < rows; row += step) {
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
      k = (sg / (float)a.d * inv) * inv * inv;   // in this order: inv^3 alone leaves fp32's range
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
  if (!a.norm) return;
  __syncthreads();
  leave_dw<T, kWarps>(a, dw, tid, is_q, block, blocks);
}

// ---- 16-byte vectors: a head's row in the registers of a group of lanes ------------
//
// A lane holds one unit, two 16-byte vectors of the row chosen so that the turn stays
// inside the lane: elements [8 j, 8 j + 8) and their partners half a rotary_dim on
// (neighbouring vectors where pairs are interleaved or not turned). head_dim 128 in
// bf16 takes 8 lanes, so a warp works on 4 rows at once; cosines, sines and weights stay
// in registers over the rows of a token. Each row is read once and written once; rows
// ahead are on their way while a row is computed. 8192 tokens of 32 + 8 heads of 128
// (bf16, 168.9 MB): 29.7 us, 5.7 TB/s, 87 % of a copy; about as much by instruction issue
// (58 % of the cycles at 21 warps an SM: six CTAs of four warps, 80 registers; five CTAs
// 31.5 us, seven spill and take 30.5). With K and V written as e4m3 36.8 us, 5.0 TB/s: the
// row's maximum, the scaling and the conversion are what is added.
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

// Two fp32 in one register pair: sm_100 multiplies and adds them in one instruction.
using f2 = unsigned long long;
__device__ __forceinline__ f2 f2_of(float lo, float hi) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void f2_to(f2 v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float f2_sum(f2 v) {
  float a, b;
  f2_to(v, a, b);
  return a + b;
}

// 16 bytes of T as pairs of fp32.
template <typename T>
struct Vec {
  static constexpr int E = Pack<T>::kE, N = E / 2;
  f2 v[N];
  __device__ __forceinline__ void from(const uint4& x) {
    float f[E];
    Pack<T>::unpack(x, f);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = f2_of(f[2 * i], f[2 * i + 1]);
  }
  __device__ __forceinline__ uint4 to() const {
    float f[E];
    floats(f);
    return Pack<T>::pack(f);
  }
  __device__ __forceinline__ void floats(float (&f)[E]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) f2_to(v[i], f[2 * i], f[2 * i + 1]);
  }
};

// Cosines and sines of a unit: table columns [j E, j E + E) and rotary_dim / 2 on, in
// either pairing (neighbours: (sine, -sine) and (cosine, cosine) of one pair in a pair).
template <typename T>
struct Turn {
  static constexpr int E = Pack<T>::kE, N = E / 2;
  f2 c[N], s[N];
  __device__ __forceinline__ void load(const float* rope, int64_t pos, int64_t max_pos, int r, int j) {
    const bool known = pos >= 0 && pos < max_pos;
    const float* row = rope + (known ? pos : 0) * r + j * E;
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(row) + i);
      const float4 b = __ldg(reinterpret_cast<const float4*>(row + r / 2) + i);
      c[2 * i] = f2_of(a.x, a.y), c[2 * i + 1] = f2_of(a.z, a.w);
      s[2 * i] = f2_of(b.x, b.y), s[2 * i + 1] = f2_of(b.z, b.w);
    }
    if (!known)
#pragma unroll
      for (int i = 0; i < N; ++i) c[i] = s[i] = f2_of(quiet_nan(), quiet_nan());
  }
  // (a, b) turned by the angle (back: by its negative).
  template <bool kBack>
  __device__ __forceinline__ void apply(Vec<T>& a, Vec<T>& b, int interleaved) const {
    const f2 sign = kBack ? f2_of(1.f, -1.f) : f2_of(-1.f, 1.f);
    if (!interleaved) {
      const f2 minus = f2_of(-1.f, -1.f);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const f2 as = mul2(a.v[i], s[i]), bs = mul2(b.v[i], s[i]);
        a.v[i] = fma2(a.v[i], c[i], kBack ? bs : mul2(bs, minus));
        b.v[i] = fma2(b.v[i], c[i], kBack ? mul2(as, minus) : as);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        neighbours(a.v[i], i, sign);
        neighbours(b.v[i], N + i, sign);
      }
    }
  }
  // pair k of the unit, whose cosine and sine are half of c[k / 2] and s[k / 2]
  __device__ __forceinline__ void neighbours(f2& v, int k, f2 sign) const {
    float c0, c1, s0, s1, x, y;
    f2_to(c[k / 2], c0, c1);
    f2_to(s[k / 2], s0, s1);
    f2_to(v, x, y);
    const float cc = k & 1 ? c1 : c0, ss = k & 1 ? s1 : s0;
    // (x c -+ y s, y c +- x s)
    v = fma2(f2_of(y, x), mul2(f2_of(ss, ss), sign), mul2(v, f2_of(cc, cc)));
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

// What becomes of an operand's rows.
enum Out { kRowsOut, kCacheOut };

// A lane's rows on their way: kStages stages of kVecs 16-byte vectors in shared memory, each
// written by the lane's own asynchronous copies and read by the lane alone, so that deep
// loads cost no registers and no barrier.
template <int kVecs, int kStages>
struct Ring {
  static constexpr int kDeep = kStages, kWarpBytes = kStages * kVecs * 512;
  uint32_t base;                         // of this lane
  __device__ __forceinline__ Ring(void* smem, int warp, int lane)
      : base(ptx::smem_addr(smem) + warp * kWarpBytes + lane * 16) {}
  __device__ __forceinline__ uint32_t at(int stage, int vec) const { return base + (stage * kVecs + vec) * 512; }
  __device__ __forceinline__ static int after(int stage) { return stage + 1 == kStages ? 0 : stage + 1; }
  // In place of a copy that is not made.
  __device__ __forceinline__ void zero(int stage) const {
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
      asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(at(stage, i)), "r"(0) : "memory");
  }
  __device__ __forceinline__ uint4 get(int stage, int vec) const {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(at(stage, vec))
                 : "memory");
    return v;
  }
};

using RopeRing = Ring<2, 4>;             // x
using BackRing = Ring<4, 2>;             // dy and x

// `run` groups of 32 / L rows of one operand. kTurned: normed and turned (else as they are:
// the values on their way to the cache).
template <typename T, int L, bool kTurned, int kOut>
__device__ __forceinline__ void qk_rope_rows(const QkArgs& a, const Rows& in, const OutRows& out, const void* w,
                                             void* cache, float* scales, unsigned heads, unsigned warp, int lane,
                                             int run, const RopeRing& ring) {
  constexpr int E = Pack<T>::kE, N = E / 2, kRows = 32 / L, kDeep = RopeRing::kDeep;
  const int j = lane % L;
  const UnitOf<T> u(j, a.d, a.r, a.interleaved);
  const unsigned rows = (unsigned)a.tokens * heads;   // at most 2^31
  const unsigned first = warp * (unsigned)run * kRows + lane / L;
  if (first - lane / L >= rows) return;
  run = min(run, (int)((rows - (first - lane / L) + kRows - 1) / kRows));   // groups with a row
  const int64_t in_step = kRows * in.sh;
  const int across = u.eb - u.ea;
  // the lane walks down its rows ([tokens, heads] numbered token by token) by a pointer that
  // is made anew where the token changes
  unsigned ahead = first, ahead_end = 0;
  const T* from = nullptr;
  auto fetch = [&](int stage) {
    if (ahead < rows && u.on) {
      if (ahead >= ahead_end) {
        const unsigned t = ahead / heads, h = ahead - t * heads;
        ahead_end = ahead - h + heads;
        from = static_cast<const T*>(in.p) + t * in.st + (int64_t)h * in.sh + u.ea;
      }
      cp_async16(ring.at(stage, 0), from);
      cp_async16(ring.at(stage, 1), from + across);
      from += in_step;
    } else {
      ring.zero(stage);
    }
    cp_commit();
    ahead += kRows;
  };
#pragma unroll
  for (int i = 0; i < kDeep; ++i) {
    if (i < run) fetch(i);
    else cp_commit();
  }
  Vec<T> wa, wb;
  Turn<T> turn;
  if (kTurned && a.norm && u.on) {
    wa.from(ptx::ld_cached_v4(static_cast<const T*>(w) + u.ea));
    wb.from(ptx::ld_cached_v4(static_cast<const T*>(w) + u.eb));
  }
  const float rd = 1.f / (float)a.d;
  unsigned row = first, end = 0;
  int stage = 0;
  T* to = nullptr;
  int64_t at = 0;                        // cache row
  bool keep = kOut == kRowsOut;
  const int64_t to_step = kOut == kRowsOut ? kRows * out.sh : (int64_t)kRows * a.page * a.d;
#pragma unroll 1
  for (int i = 0; i < run; ++i) {
    const bool live = row < rows;
    cp_wait<kDeep - 1>();
    Vec<T> ya, yb;
    ya.from(ring.get(stage, 0));
    yb.from(ring.get(stage, 1));
    if (i + kDeep < run) fetch(stage);
    else cp_commit();
    stage = ring.after(stage);
    if (row >= end && live) {
      const unsigned t = row / heads, h = row - t * heads;
      end = row - h + heads;
      if (kTurned && u.turned) turn.load(a.rope, a.positions[t], a.max_pos, a.r, j);
      if constexpr (kOut == kRowsOut) {
        to = static_cast<T*>(out.p) + t * out.st + (int64_t)h * out.sh + u.ea;
      } else {
        const int64_t slot = a.slots[t];
        keep = slot >= 0 && slot < a.num_slots;
        at = keep ? cache_row(slot, h, a) : 0;
        to = static_cast<T*>(cache) + at * a.d + u.ea;
      }
    }
    if (kTurned && a.norm) {
      f2 sa = mul2(ya.v[0], ya.v[0]), sb = mul2(yb.v[0], yb.v[0]);
#pragma unroll
      for (int e = 1; e < N; ++e) {
        sa = fma2(ya.v[e], ya.v[e], sa);
        sb = fma2(yb.v[e], yb.v[e], sb);
      }
      const float inv = rsqrtf(lanes_sum<L>(f2_sum(sa) + f2_sum(sb)) * rd + a.eps);
      const f2 inv2 = f2_of(inv, inv);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        ya.v[e] = mul2(mul2(ya.v[e], inv2), wa.v[e]);
        yb.v[e] = mul2(mul2(yb.v[e], inv2), wb.v[e]);
      }
    }
    if (kTurned && u.turned) turn.template apply<false>(ya, yb, a.interleaved);
    if (kOut == kRowsOut || !a.e4m3) {
      if (live && keep && u.on) {
        ptx::st_v4(to, ya.to());
        ptx::st_v4(to + across, yb.to());
      }
    } else {
      float fa[E], fb[E];
      ya.floats(fa);
      yb.floats(fb);
      float most = kE4M3Floor;
#pragma unroll
      for (int e = 0; e < E; ++e) most = fmaxf(most, fmaxf(fabsf(fa[e]), fabsf(fb[e])));
      most = lanes_max<L>(most);
      if (live && keep && u.on) {
        const float up = kE4M3Max / most;
        unsigned char* y = static_cast<unsigned char*>(cache) + at * a.d + u.ea;
        uint32_t ca[E / 4], cb[E / 4];
#pragma unroll
        for (int e = 0; e < E / 4; ++e) {
          ca[e] = e4m3x2_of(fa[4 * e] * up, fa[4 * e + 1] * up) |
                  (uint32_t)e4m3x2_of(fa[4 * e + 2] * up, fa[4 * e + 3] * up) << 16;
          cb[e] = e4m3x2_of(fb[4 * e] * up, fb[4 * e + 1] * up) |
                  (uint32_t)e4m3x2_of(fb[4 * e + 2] * up, fb[4 * e + 3] * up) << 16;
        }
        if constexpr (E == 8) {
          *reinterpret_cast<uint2*>(y) = make_uint2(ca[0], ca[1]);
          *reinterpret_cast<uint2*>(y + across) = make_uint2(cb[0], cb[1]);
        } else {
          *reinterpret_cast<uint32_t*>(y) = ca[0];
          *reinterpret_cast<uint32_t*>(y + across) = cb[0];
        }
        if (j == 0) scales[at] = most / kE4M3Max;
      }
      at += (int64_t)kRows * a.page;
    }
    to += to_step;
    row += kRows;
  }
  cp_wait<0>();
}

// CTAs [0, q_blocks) have the queries' rows, the next ones the keys', then the values'.
constexpr int kRopeBlock = 128;
constexpr int kRopeWarps = kRopeBlock / 32;

struct Split {
  int q_blocks, k_blocks, q_run, k_run;   // CTAs, and groups of rows of a warp
};

template <typename T, int L, bool kWrite>
__global__ void __launch_bounds__(kRopeBlock, 6)
qk_rope_kernel(const __grid_constant__ QkArgs a, const __grid_constant__ Split sp) {
  ptx::grid_dep_wait();
  __shared__ uint4 smem[kRopeWarps * RopeRing::kWarpBytes / 16];
  const int tid = thread_here(), lane = tid & 31;
  const RopeRing ring(smem, tid >> 5, lane);
  int block = blockIdx.x;
  if (block < sp.q_blocks) {
    qk_rope_rows<T, L, true, kRowsOut>(a, a.q, a.qo, a.qw, nullptr, nullptr, a.hq, block * kRopeWarps + (tid >> 5),
                                       lane, sp.q_run, ring);
    return;
  }
  block -= sp.q_blocks;
  if (!kWrite || block < sp.k_blocks) {
    qk_rope_rows<T, L, true, kWrite ? kCacheOut : kRowsOut>(a, a.k, a.ko, a.kw, a.kc, a.ks, a.hk,
                                                            block * kRopeWarps + (tid >> 5), lane, sp.k_run, ring);
    return;
  }
  block -= sp.k_blocks;
  if constexpr (kWrite)
    qk_rope_rows<T, L, false, kCacheOut>(a, a.v, a.ko, nullptr, a.vc, a.vs, a.hk, block * kRopeWarps + (tid >> 5),
                                         lane, sp.k_run, ring);
}

// The backward: g and x in registers, dw summed per lane over the lane's rows, then over
// the warp's row groups and the CTA's warps in a fixed order. CTAs [0, q_blocks) share the
// queries' rows equally, the others the keys'. 8192 tokens of 32 + 8 heads of 128 (bf16,
// 253.8 MB): 53.4 us, 4.75 TB/s, 73 % of a copy (fp32 88 us, 88 %); cosines, weights, dw, g and x fill 128
// registers, and 16 warps an SM do not hide a row's chain of products and lane sums (issue
// 51 % of the cycles; at 96 registers the spills cost more: 66 us).
constexpr int kBackCtas = 4;               // resident on an SM (128 registers a thread)

template <typename T, int L>
__global__ void __launch_bounds__(kRopeBlock, kBackCtas)
qk_rope_backward_kernel(const __grid_constant__ QkBackArgs a, int q_blocks) {
  constexpr int E = Pack<T>::kE, N = E / 2, kRows = 32 / L, kDeep = BackRing::kDeep;
  extern __shared__ __align__(16) float dw[];   // the rings, then [kRopeWarps][d]
  ptx::grid_dep_wait();
  const int tid = thread_here(), lane = tid & 31, warp = tid >> 5, j = lane % L;
  const BackRing ring(dw, warp, lane);
  const UnitOf<T> u(j, a.d, a.r, a.interleaved);
  const int across = u.eb - u.ea;
  const bool is_q = (int)blockIdx.x < q_blocks;
  const unsigned blocks = is_q ? q_blocks : gridDim.x - q_blocks, block = is_q ? blockIdx.x : blockIdx.x - q_blocks;
  const unsigned heads = is_q ? a.hq : a.hk;
  const Rows xr = is_q ? a.q : a.k, gr = is_q ? a.dqo : a.dko;
  Vec<T> wa = {}, wb = {}, da = {}, db = {};
  if (a.norm && u.on) {
    const T* w = static_cast<const T*>(is_q ? a.qw : a.kw);
    wa.from(ptx::ld_cached_v4(w + u.ea));
    wb.from(ptx::ld_cached_v4(w + u.eb));
  }
  const unsigned rows = (unsigned)a.tokens * heads, groups = (rows + kRows - 1) / kRows;
  const unsigned workers = blocks * kRopeWarps, me = block * kRopeWarps + warp;
  const unsigned first = (unsigned)((uint64_t)groups * me / workers);
  const unsigned n = (unsigned)((uint64_t)groups * (me + 1) / workers) - first;
  unsigned row = first * kRows + lane / L, end = 0;
  T* y = static_cast<T*>(is_q ? a.dq : a.dk) + (int64_t)row * a.d + u.ea;
  unsigned ahead = row, ahead_end = 0;
  const T* gp = nullptr;
  const T* xp = nullptr;
  const int64_t g_step = kRows * gr.sh, x_step = kRows * xr.sh;
  auto fetch = [&](int stage) {
    if (ahead < rows && u.on) {
      if (ahead >= ahead_end) {
        const unsigned t = ahead / heads, h = ahead - t * heads;
        ahead_end = ahead - h + heads;
        gp = static_cast<const T*>(gr.p) + t * gr.st + (int64_t)h * gr.sh + u.ea;
        xp = static_cast<const T*>(xr.p) + t * xr.st + (int64_t)h * xr.sh + u.ea;
      }
      cp_async16(ring.at(stage, 0), gp);
      cp_async16(ring.at(stage, 1), gp + across);
      gp += g_step;
      if (a.norm) {
        cp_async16(ring.at(stage, 2), xp);
        cp_async16(ring.at(stage, 3), xp + across);
        xp += x_step;
      }
    } else {
      ring.zero(stage);
    }
    cp_commit();
    ahead += kRows;
  };
#pragma unroll
  for (int i = 0; i < kDeep; ++i) {
    if (i < (int)n) fetch(i);
    else cp_commit();
  }
  const float rd = 1.f / (float)a.d;
  Turn<T> turn;
  int stage = 0;
#pragma unroll 1
  for (unsigned i = 0; i < n; ++i) {
    const bool live = row < rows;
    if (live && row >= end) {
      const unsigned t = row / heads;
      end = (t + 1) * heads;
      if (u.turned) turn.load(a.rope, a.positions[t], a.max_pos, a.r, j);
    }
    cp_wait<kDeep - 1>();
    Vec<T> xa, xb, ga, gb;              // zeros behind the last row
    ga.from(ring.get(stage, 0));
    gb.from(ring.get(stage, 1));
    if (u.turned && live) turn.template apply<true>(ga, gb, a.interleaved);
    if (a.norm) {
      xa.from(ring.get(stage, 2));
      xb.from(ring.get(stage, 3));
    }
    if (i + kDeep < n) fetch(stage);
    else cp_commit();
    stage = ring.after(stage);
    if (a.norm) {
      f2 ss = 0ull, sg = 0ull;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        ss = fma2(xa.v[e], xa.v[e], fma2(xb.v[e], xb.v[e], ss));
        sg = fma2(mul2(ga.v[e], wa.v[e]), xa.v[e], fma2(mul2(gb.v[e], wb.v[e]), xb.v[e], sg));
      }
      const float sum = lanes_sum<L>(f2_sum(ss)), dot = lanes_sum<L>(f2_sum(sg));
      // behind the last row nothing: the root of an eps of 0 would make 0 * inf of it in dw
      const float inv = live ? rsqrtf(sum * rd + a.eps) : 0.f;
      const float k = -(dot * rd * inv) * inv * inv;   // in this order: inv^3 alone leaves fp32's range
      const f2 inv2 = f2_of(inv, inv), k2 = f2_of(k, k);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        ga.v[e] = mul2(ga.v[e], inv2);
        gb.v[e] = mul2(gb.v[e], inv2);
        da.v[e] = fma2(ga.v[e], xa.v[e], da.v[e]);
        db.v[e] = fma2(gb.v[e], xb.v[e], db.v[e]);
        ga.v[e] = fma2(ga.v[e], wa.v[e], mul2(xa.v[e], k2));
        gb.v[e] = fma2(gb.v[e], wb.v[e], mul2(xb.v[e], k2));
      }
    }
    if (live && u.on) {
      ptx::st_v4(y, ga.to());
      ptx::st_v4(y + across, gb.to());
    }
    row += kRows;
    y += kRows * a.d;
  }
  cp_wait<0>();
  if (!a.norm) return;
  ptx::grid_dep_launch_dependents();   // the sum of dw may come to the SMs (and waits)
  __syncthreads();                  // every warp is done with its ring
  float fa[E], fb[E];
  da.floats(fa);
  db.floats(fb);
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int o = L; o < 32; o <<= 1) {
      fa[e] += __shfl_xor_sync(0xFFFFFFFFu, fa[e], o);
      fb[e] += __shfl_xor_sync(0xFFFFFFFFu, fb[e], o);
    }
  if (lane < L && u.on) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      dw[warp * a.d + u.ea + e] = fa[e];
      dw[warp * a.d + u.eb + e] = fb[e];
    }
  }
  __syncthreads();
  leave_dw<T, kRopeWarps>(a, dw, tid, is_q, block, blocks);
}

// dw of both weights from the CTAs' partials: a CTA has 32 columns of one of them, its warps
// the parts w, w + 32, ..., added in that order and then in warp order. Two L2 round trips.
constexpr int kDwWarps = 32;

template <typename T>
__global__ void __launch_bounds__(kDwWarps * 32)
qk_rope_dw_kernel(const float* ws, int q_parts, int parts, int d, T* dqw, T* dkw) {
  __shared__ float s_sum[kDwWarps][32];
  ptx::grid_dep_wait();
  const int tid = thread_here(), lane = tid & 31, warp = tid >> 5;
  const bool is_q = blockIdx.y == 0;
  const int col = blockIdx.x * 32 + lane, first = is_q ? 0 : q_parts, end = is_q ? q_parts : parts;
  float s = 0.f;
  if (col < d) {
#pragma unroll 12
    for (int i = first + warp; i < end; i += kDwWarps) s += ws[(int64_t)i * d + col];
  }
  s_sum[warp][lane] = s;
  __syncthreads();
  if (warp != 0 || col >= d) return;
  s = 0.f;
#pragma unroll
  for (int w = 0; w < kDwWarps; ++w) s += s_sum[w][lane];
  (is_q ? dqw : dkw)[col] = Pack<T>::from_f(s);
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

// Whether a backward call runs as one cluster of 16 CTAs, which adds up dw through shared
// memory (no second kernel, no workspace): rows for the vector kernel, at most 8 groups of
// them for each warp. A decision by the sizes, so that the caller knows what the workspace
// has to hold; on odd addresses the kernel for any row runs as that cluster. 333 tokens of 9
// heads of 64 (fp16): 9.2 us on the device against 4.6 in two kernels, but 15.9 against 20.7
// a call, as the host issues them (a captured call has the device time: what it loses there is
// the price). 16 CTAs are past the portable cluster size: a whole B200 has room for them, a
// part of one may refuse the launch.
constexpr int kCluster = 16;
bool one_cluster(int64_t tokens, int hq, int hk, int d, int r, int dtype) {
  const int lanes = lanes_of(d, r, elem_bytes(dtype), 0, 0);
  return lanes && tokens * (hq + hk) * lanes / 32 <= 8 * kCluster * kRopeWarps;
}

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
  if (write) {
    // rows of the cache that one warp writes must not be rows that another reads
    const rmsnorm_kv_cache* c = a->cache;
    const uint64_t rows = (uint64_t)c->num_pages * c->kv_heads * c->page_size;   // (sizes of no memory may wrap)
    const int ceb = c->dtype == RMSNORM_KV_E4M3 ? 1 : eb, seb = c->dtype == RMSNORM_KV_E4M3 ? 4 : 0;
    const View held[4] = {span_of(c->k, rows * c->head_dim * ceb), span_of(c->v, rows * c->head_dim * ceb),
                          span_of(c->k_scale, rows * seb), span_of(c->v_scale, rows * seb)};
    if (views_overlap(held[0], held[1]))
      return refuse(RMSNORM_TP_ERR_INVALID, "%s: the cache's k overlaps its v", who);
    for (const View& h : held)
      if (views_overlap(h, in[0]) || views_overlap(h, in[1]) || views_overlap(h, in[2]) || views_overlap(h, outs[0]))
        return refuse(RMSNORM_TP_ERR_INVALID, "%s: q, k, v or q_out overlaps the cache", who);
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
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (lanes) {
    // groups of rows for each warp: as many as leave every SM 32 warps, at most 8; whole
    // tokens where that is a few more
    const int per = 32 / lanes, sms = sm_count(in->device);
    auto runs = [&](int64_t groups, int heads) {
      int64_t run = groups / (32ll * (sms > 0 ? sms : 1));
      run = run < 1 ? 1 : run > 8 ? 8 : run;
      const int64_t token = heads % per == 0 ? heads / per : 1;
      return (int)((run + token - 1) / token * token <= 2 * run ? (run + token - 1) / token * token : run);
    };
    auto blocks = [&](int64_t groups, int run) {
      return (int)((groups + (int64_t)run * kRopeWarps - 1) / ((int64_t)run * kRopeWarps));
    };
    const int64_t gq = (a.tokens * a.hq + per - 1) / per, gk = (a.tokens * a.hk + per - 1) / per;
    Split sp;
    sp.q_run = runs(gq, a.hq);
    sp.k_run = runs(gk, a.hk);
    sp.q_blocks = blocks(gq, sp.q_run);
    sp.k_blocks = blocks(gk, sp.k_run);
    void* args[] = {&a, &sp};
    e = launch_dependent(fn, dim3((unsigned)sp.q_blocks + (kWrite ? 2u : 1u) * (unsigned)sp.k_blocks),
                         dim3(kRopeBlock), 0, args, st);
  } else {
    void* args[] = {&a};
    e = launch_dependent(fn, dim3((unsigned)((rows + kWarps - 1) / kWarps)), dim3(kBlock), 0, args, st);
  }
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

size_t rmsnorm_qk_rope_backward_workspace_bytes(int64_t tokens, int32_t q_heads, int32_t kv_heads,
                                                int32_t head_dim, int32_t rotary_dim, int32_t dtype) {
  using namespace rtp;
  if (check_common("qk_rope_backward_workspace_bytes", tokens, q_heads, kv_heads, head_dim, rotary_dim, dtype,
                   1) != RMSNORM_TP_OK ||
      one_cluster(tokens, q_heads, kv_heads, head_dim, rotary_dim, dtype))
    return 0;
  return (size_t)kMaxParts * (size_t)head_dim * sizeof(float);
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
  const bool cluster = norm && in->tokens > 0 &&
                       one_cluster(in->tokens, in->q_heads, in->kv_heads, in->head_dim, in->rotary_dim, in->dtype);
  const int64_t need = !norm || cluster || in->tokens == 0 ? 0 : (int64_t)kMaxParts * in->head_dim * 4;
  if (norm && (!in->dq_weight || !in->dk_weight || (need && !in->workspace) || in->workspace_bytes < need))
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: NULL dq_weight or dk_weight, or a workspace of %lld bytes < %lld",
                  who, (long long)in->workspace_bytes, (long long)need);
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
  int grid = 0, q_blocks = 0;
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
    a.ws = cluster ? nullptr : static_cast<float*>(in->workspace);
    a.dqw = in->dq_weight;
    a.dkw = in->dk_weight;
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
    // one resident wave of CTAs, shared by q and k as their rows are
    const int sms = sm_count(in->device), warps = lanes ? kRopeWarps : kWarps;
    const int most = min(kMaxParts, lanes ? sms * kBackCtas : 2 * sms);
    if (most < 2) return refuse(RMSNORM_TP_ERR_CUDA, "%s: no device %d", who, in->device);
    const int64_t rows_of_cta = (int64_t)warps * (lanes ? 32 / lanes : 1);
    const int64_t wq = (a.tokens * a.hq + rows_of_cta - 1) / rows_of_cta;
    const int64_t wk = (a.tokens * a.hk + rows_of_cta - 1) / rows_of_cta;
    if (cluster) {
      grid = kCluster;
      q_blocks = (a.hq * kCluster + (a.hq + a.hk) / 2) / (a.hq + a.hk);
      q_blocks = q_blocks < 1 ? 1 : q_blocks >= grid ? grid - 1 : q_blocks;
    } else if (wq + wk <= most) {
      q_blocks = (int)wq;
      grid = (int)(wq + wk);
    } else {
      grid = most;
      q_blocks = (int)((wq * grid + (wq + wk) / 2) / (wq + wk));
      q_blocks = q_blocks < 1 ? 1 : q_blocks >= grid ? grid - 1 : q_blocks;
    }
    const void* fn = in->dtype == RMSNORM_TP_F32    ? backward_fn<float>(lanes)
                     : in->dtype == RMSNORM_TP_BF16 ? backward_fn<__nv_bfloat16>(lanes)
                                                    : backward_fn<__half>(lanes);
    void* args[] = {&a, &q_blocks};
    // the vector kernels' rings (at most 8 KB of dw lies over them)
    const size_t sums = norm ? (size_t)warps * a.d * sizeof(float) : 0;
    const size_t smem = lanes ? (size_t)warps * BackRing::kWarpBytes : sums;
    cudaError_t e = cudaSuccess;
    if (cluster) {                     // over 8 CTAs: the kernel has to say so, once on a device
      static std::atomic<bool> said[64][3][6];
      std::atomic<bool>* known = in->device < 64 ? &said[in->device][in->dtype][lanes ? __builtin_ctz(lanes) : 0] : nullptr;
      if (!known || !known->load()) {
        e = cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (known && e == cudaSuccess) known->store(true);
      }
    }
    if (e == cudaSuccess)
      e = launch_dependent(fn, dim3((unsigned)grid), dim3(warps * 32), smem, args, st, cluster ? kCluster : 0);
    if (e != cudaSuccess) return launch_failed(e, who);
  }
  if (norm && !cluster) {   // no tokens: zeros
    const float* ws = static_cast<const float*>(in->workspace);
    int d = in->head_dim;
    void* dqw = in->dq_weight;
    void* dkw = in->dk_weight;
    void* args[] = {&ws, &q_blocks, &grid, &d, &dqw, &dkw};
    const void* fn = in->dtype == RMSNORM_TP_F32    ? reinterpret_cast<const void*>(qk_rope_dw_kernel<float>)
                     : in->dtype == RMSNORM_TP_BF16 ? reinterpret_cast<const void*>(qk_rope_dw_kernel<__nv_bfloat16>)
                                                    : reinterpret_cast<const void*>(qk_rope_dw_kernel<__half>);
    const cudaError_t e = launch_dependent(fn, dim3((d + 31) / 32, 2), dim3(kDwWarps * 32), 0, args, st);
    if (e != cudaSuccess) return launch_failed(e, who);
  }
  return RMSNORM_TP_OK;
}

}  // extern "C"
