// Attention of one new token of each sequence over a paged cache.
//
//   s_j = scale q . k_j;  m = max s;  l = sum exp(s_j - m);  o = sum exp(s_j - m) v_j / l
//
// A sequence's tokens are divided over several CTAs ("splits"); each leaves its
// m, l and o (relative to its own m) in the workspace, and a second kernel joins
// them: o = sum_i exp(m_i - m) o_i / sum_i exp(m_i - m) l_i.
#include <atomic>

#include "heads_common.cuh"

namespace rtp {
namespace {

struct AttnArgs {
  const void* q;
  void* out;
  float* lse;
  const void* k;
  const void* v;
  const float* ks;
  const float* vs;
  const int32_t* table;
  const int32_t* lens;
  float* part;          // per (sequence, head, split): m, l, o[d]
  int64_t qst, qsh, table_stride, num_pages, max_tokens, batch;
  int hq, hk, page, d, splits;
  int row_groups;       // groups of 16 query heads that share a kv head
  int segments;         // kv heads * row_groups
  int q_pairs;          // the queries' elements can be read two at a time
  float scale_log2;     // scale * log2(e): scores in base 2
};

constexpr float kLn2 = 0.69314718055994531f;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ int64_t length_of(const AttnArgs& a, int64_t b) {
  const int64_t n = a.lens[b];
  return n < 0 ? 0 : n > a.max_tokens ? a.max_tokens : n;
}

// ---- any type and head_dim --------------------------------------------------------
// One CTA per (query head, sequence, split): a thread per token for the scores, a
// thread per element for the values. Reads the keys' rows uncoalesced and the
// cache once for each query head.
constexpr int kAnyBlock = 128;

template <typename TQ, typename TC>
__global__ void __launch_bounds__(kAnyBlock) attention_any_kernel(const __grid_constant__ AttnArgs a) {
  constexpr bool kE4M3 = sizeof(TC) == 1;
  __shared__ float q[256];
  __shared__ float p[kAnyBlock];
  __shared__ int64_t at[kAnyBlock];
  __shared__ float red[kAnyBlock / 32];
  ptx::grid_dep_wait();
  const int h = blockIdx.x, tid = thread_here();
  const int64_t b = blockIdx.y, split = blockIdx.z;
  const int kvh = h / (a.hq / a.hk);
  const TQ* qg = static_cast<const TQ*>(a.q) + b * a.qst + h * a.qsh;
  for (int i = tid; i < a.d; i += kAnyBlock) q[i] = Pack<TQ>::to_f(qg[i]);
  const int64_t len = length_of(a, b);
  const int64_t per = (len + a.splits - 1) / a.splits;
  const int64_t t0 = split * per, t1 = t0 + per < len ? t0 + per : len;
  float m = -INFINITY, l = 0.f, o[2] = {0.f, 0.f};
  for (int64_t base = t0; base < t1; base += kAnyBlock) {
    __syncthreads();
    const int64_t t = base + tid;
    float s = -INFINITY;
    int64_t row = -1;
    if (t < t1) {
      const int64_t pg = a.table[b * a.table_stride + t / a.page];
      if (pg >= 0 && pg < a.num_pages) {
        row = (pg * a.hk + kvh) * a.page + t % a.page;
        const TC* k = static_cast<const TC*>(a.k) + row * a.d;
        float acc = 0.f;
        for (int i = 0; i < a.d; ++i) {
          if constexpr (kE4M3)
            acc = fmaf(q[i], e4m3_to(reinterpret_cast<const unsigned char*>(k)[i]), acc);
          else
            acc = fmaf(q[i], Pack<TC>::to_f(k[i]), acc);
        }
        s = acc * (kE4M3 ? a.ks[row] : 1.f) * a.scale_log2;
      }
    }
    float top = s;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
    if ((tid & 31) == 0) red[tid >> 5] = top;
    at[tid] = row;
    __syncthreads();
    float mn = m;
    for (int w = 0; w < kAnyBlock / 32; ++w) mn = fmaxf(mn, red[w]);
    const float ref = mn == -INFINITY ? 0.f : mn;
    const float e = row >= 0 ? exp2f(s - ref) : 0.f;
    p[tid] = e;
    const float sum = warp_allreduce_sum(e);
    __syncthreads();
    if ((tid & 31) == 0) red[tid >> 5] = sum;
    __syncthreads();
    const float alpha = exp2f(m - ref);
    l *= alpha;
    for (int w = 0; w < kAnyBlock / 32; ++w) l += red[w];
    m = mn;
    const int n = (int)(t1 - base < kAnyBlock ? t1 - base : kAnyBlock);
    for (int c = 0; c < 2; ++c) {
      const int i = tid + c * kAnyBlock;
      if (i >= a.d) continue;
      float acc = o[c] * alpha;
      for (int j = 0; j < n; ++j) {
        if (at[j] < 0) continue;
        const TC* v = static_cast<const TC*>(a.v) + at[j] * a.d;
        if constexpr (kE4M3)
          acc = fmaf(p[j] * a.vs[at[j]], e4m3_to(reinterpret_cast<const unsigned char*>(v)[i]), acc);
        else
          acc = fmaf(p[j], Pack<TC>::to_f(v[i]), acc);
      }
      o[c] = acc;
    }
  }
  float* w = a.part + ((b * a.hq + h) * a.splits + split) * (a.d + 2);
  if (tid == 0) {
    w[0] = m;
    w[1] = l;
  }
  for (int c = 0; c < 2; ++c)
    if (tid + c * kAnyBlock < a.d) w[2 + tid + c * kAnyBlock] = o[c];
}

// Joins a head's splits: one CTA per (sequence, query head).
template <typename TQ>
__global__ void __launch_bounds__(kAnyBlock) attention_join_any_kernel(const __grid_constant__ AttnArgs a) {
  ptx::grid_dep_wait();
  const int tid = thread_here();
  const int64_t row = blockIdx.x;
  const float* w = a.part + row * a.splits * (a.d + 2);
  float m = -INFINITY, l = 0.f;
  for (int s = 0; s < a.splits; ++s) m = fmaxf(m, w[s * (a.d + 2)]);
  const float ref = m == -INFINITY ? 0.f : m;
  for (int s = 0; s < a.splits; ++s) l += exp2f(w[s * (a.d + 2)] - ref) * w[s * (a.d + 2) + 1];
  for (int i = tid; i < a.d; i += kAnyBlock) {
    float o = 0.f;
    for (int s = 0; s < a.splits; ++s)
      o = fmaf(exp2f(w[s * (a.d + 2)] - ref), w[s * (a.d + 2) + 2 + i], o);
    static_cast<TQ*>(a.out)[row * a.d + i] = Pack<TQ>::from_f(l == 0.f ? 0.f : o / l);
  }
  if (a.lse && tid == 0) a.lse[row] = kLn2 * (ref + log2f(l));
}

// ---- tensor cores: 16-bit queries, head_dim 64, 96, 128, 192 or 256 ----------------
//
// The bound is HBM: a token's K and V rows are read once for its whole group of query
// heads, and the products need (at 16 padded heads) 4 * 16 * head_dim flops for them, a
// tenth of what warp-level mma.sync gives at that rate of bytes; tcgen05's 128-row tiles
// would be 1/16 used at a group of 8. A CTA of 4 warps takes tiles of 64 tokens, 16 for
// each warp, which runs its own softmax and its own cp.async ring (no CTA barrier in
// the loop; the loads run ahead over the borders of sequences), and the warps' results
// are joined at a sequence's end.
//
// All (sequence, kv head, 16 query heads) are laid behind one another in tiles, and each
// CTA takes an equal run of tiles, from the lengths on the device: ragged batches
// balance to a tile and nothing on the host knows a length. A run that ends inside a
// sequence leaves m, l and o in the workspace (at most two for each CTA), and the join
// kernel adds them in CTA order.
constexpr int kWarps = 4;
constexpr int kBlock = 32 * kWarps;
constexpr int kTile = 16 * kWarps;      // tokens of a CTA's tile
constexpr int kRows = 16;               // query heads of a tile

struct alignas(16) Meta {               // what a CTA's last segment leaves to the join
  int32_t open, b, hs, last;            // open: it goes on in the CTAs up to `last`
};

template <int D, bool kE4M3>
struct Shape {
  static constexpr int kChunks = D * (kE4M3 ? 1 : 2) / 16;   // 16-byte chunks of a row
  // rows of 8 k chunks are swizzled (chunk ^ (row & 7)), others padded to an odd number:
  // either way 8 rows of one chunk fall into 8 different bank groups
  static constexpr bool kSwizzle = kChunks % 8 == 0;
  static constexpr int kPitch = (kSwizzle ? kChunks : (kChunks | 1)) * 16;
  static constexpr int kOperand = 16 * kPitch;               // one warp's K (or V) tile
  static constexpr int kSide = kE4M3 ? 128 + 16 : 16;        // its scales and its mask
  static constexpr int kStage = 2 * kOperand + kSide;
  static constexpr int kJoin = kWarps * 8 * (D / 2 + 8) * 4;
  // two CTAs of at most 110 KB on an SM where at least three stages fit, else one
  static constexpr int kTwo = (110 * 1024 - kJoin) / (kWarps * kStage);
  static constexpr int kOne = (220 * 1024 - kJoin) / (kWarps * kStage);
  static constexpr int kCtas = kTwo >= 3 ? 2 : 1;
  static constexpr int kStages = kCtas == 2 ? (kTwo > 6 ? 6 : kTwo) : (kOne > 6 ? 6 : kOne);
  static constexpr int kSmem = kJoin + kWarps * kStages * kStage;
  static_assert(kStages >= 3, "the ring needs three stages");
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
  const int n = live ? 16 : 0;          // 0: zeros, nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool live) {
  const int n = live ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
template <bool kBf16>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (kBf16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
                 "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
                 "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 2^x and log2(x) to 2 ulp, results under 2^-126 as 0.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t e4m3x2_f16x2(uint32_t two) {
  uint32_t r;
  asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(r) : "r"(two));
  return r;
}
template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (kBf16) return bf16x2_pack(lo, hi);
  else return f16x2_pack(lo, hi);
}
template <bool kBf16>
__device__ __forceinline__ void unpack2(uint32_t u, float& lo, float& hi) {
  if constexpr (kBf16) bf16x2_unpack(u, lo, hi);
  else f16x2_unpack(u, lo, hi);
}
// Two 16-bit parts of numerators x, y >= 0, together exact to 2^-16 of them: the value cut
// off, and what is left. Neither is negative, and the second never 0 beside a first that is
// not, so that a numerator meets an infinity in V as one positive number would.
template <bool kBf16>
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  constexpr float kLeast = kBf16 ? 1.17549435e-38f : 5.9604644775390625e-8f;   // 2^-126, 2^-24
  float hx, hy;
  if constexpr (kBf16) hi = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
  else asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(y), "f"(x));
  unpack2<kBf16>(hi, hx, hy);
  lo = pack2<kBf16>(fmaxf(x - hx, kLeast), fmaxf(y - hy, kLeast));
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xFFFFFFFFu, v, 1);
  return v + __shfl_xor_sync(0xFFFFFFFFu, v, 2);
}
// The reference of exponentials: 0 where nothing has been seen (their value is 0 then).
__device__ __forceinline__ float ref_of(float m) { return m == -INFINITY ? 0.f : m; }

// Place in the row of tiles: tile `tile` of the `tiles` of segment (b, hs).
struct Place {
  int b, hs, tile, tiles;
  int64_t len;
};

__device__ __forceinline__ int tiles_of(int64_t len) { return (int)((len + kTile - 1) / kTile); }

// To the next tile; the caller knows that there is one.
__device__ __forceinline__ void advance(const AttnArgs& a, Place& p) {
  if (++p.tile < p.tiles) return;
  p.tile = 0;
  if (++p.hs < a.segments) return;
  p.hs = 0;
  do {
    ++p.b;
    p.len = length_of(a, p.b);
  } while (p.len == 0);
  p.tiles = tiles_of(p.len);
}

template <typename TQ, bool kE4M3, int D>
__global__ void __launch_bounds__(kBlock, Shape<D, kE4M3>::kCtas)
attention_kernel(const __grid_constant__ AttnArgs a) {
  using S = Shape<D, kE4M3>;
  constexpr bool kBf16 = !kE4M3 && sizeof(TQ) == 2 && !__is_same(TQ, __half);   // of the products
  // the numerators as two 16-bit parts where their rounding to one would be of the output's
  // own size; one fp16 part (2^-11) beside a bf16 output (2^-8)
  constexpr bool kTwoParts = !kE4M3 || __is_same(TQ, __half);
  // fp16 numerators run up to 2^15 instead of 1, so that fp16's smallest number, 2^-24, is
  // 2^-39 of the largest
  constexpr float kLift = kBf16 || kE4M3 ? 1.f : 32768.f;
  constexpr float kLiftLog2 = kBf16 || kE4M3 ? 0.f : 15.f;
  constexpr int kEb = kE4M3 ? 1 : 2;
  constexpr int NT = D / 8, KS = D / 16;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ float s_m[kWarps][kRows], s_l[kWarps][kRows], s_v[kWarps][kRows];
  __shared__ int64_t s_scan[kWarps];
  __shared__ int64_t s_rest;
  __shared__ int s_b;
  ptx::grid_dep_wait();
  ptx::grid_dep_launch_dependents();
  const int tid = thread_here(), lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, qd = lane & 3;

  // this CTA's run of tiles [t0, t1): every thread sums the tiles of a run of sequences
  const int64_t per = (a.batch + kBlock - 1) / kBlock;
  int64_t mine = 0;
  for (int64_t b = tid * per; b < (tid + 1) * per && b < a.batch; ++b)
    mine += (int64_t)tiles_of(length_of(a, b)) * a.segments;
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) s_scan[warp] = upto;
  __syncthreads();
  int64_t total = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) upto += s_scan[w];
    total += s_scan[w];
  }
  const int64_t workers = total < gridDim.x ? total : gridDim.x;
  const int64_t me = blockIdx.x;
  Meta* meta = reinterpret_cast<Meta*>(a.part);
  if (me >= workers) {
    if (tid == 0) meta[me] = Meta{0, 0, 0, 0};
    return;
  }
  const int64_t t0 = total * me / workers, t1 = total * (me + 1) / workers;
  if (upto - mine <= t0 && t0 < upto) {
    int64_t rest = t0 - (upto - mine);
    int64_t b = tid * per;
    for (;; ++b) {
      const int64_t n = (int64_t)tiles_of(length_of(a, b)) * a.segments;
      if (rest < n) break;
      rest -= n;
    }
    s_b = (int)b;
    s_rest = rest;
  }
  __syncthreads();
  Place at;
  at.b = s_b;
  at.len = length_of(a, at.b);
  at.tiles = tiles_of(at.len);
  at.hs = (int)(s_rest / at.tiles);
  at.tile = (int)(s_rest - (int64_t)at.hs * at.tiles);
  const int n = (int)(t1 - t0);

  float* join = reinterpret_cast<float*>(smem);
  const uint32_t ring = ptx::smem_addr(smem) + S::kJoin + warp * S::kStages * S::kStage;
  unsigned char* ring_p = smem + S::kJoin + warp * S::kStages * S::kStage;

  // ---- loads: lane l < 16 knows the row of token l of the warp's next tile ----
  Place ahead = at;
  int sent = 0;
  int32_t page_id = -1;               // of this lane's token, read one tile early
  auto look_up = [&]() {
    const int64_t t = (int64_t)ahead.tile * kTile + warp * 16 + (lane & 15);
    page_id = t < ahead.len ? a.table[ahead.b * a.table_stride + (unsigned)t / (unsigned)a.page] : -1;
  };
  look_up();
  auto send = [&]() {
    if (sent < n) {
      const int stage = sent % S::kStages;
      const uint32_t dst = ring + stage * S::kStage;
      const int64_t t = (int64_t)ahead.tile * kTile + warp * 16 + (lane & 15);
      const bool live = page_id >= 0 && page_id < a.num_pages;
      const unsigned mask = __ballot_sync(0xFFFFFFFFu, live) & 0xFFFFu;
      const int kvh = ahead.hs / a.row_groups;
      const int64_t row = live ? ((int64_t)page_id * a.hk + kvh) * a.page + (unsigned)t % (unsigned)a.page : 0;
      if (lane == 0)
        *reinterpret_cast<unsigned*>(ring_p + stage * S::kStage + 2 * S::kOperand + (kE4M3 ? 128 : 0)) = mask;
      if constexpr (kE4M3)            // lanes 0-15 K's scales, 16-31 V's
        cp_async4(dst + 2 * S::kOperand + lane * 4, (lane < 16 ? a.ks : a.vs) + row, live);
      const unsigned char* kp = static_cast<const unsigned char*>(a.k);
      const unsigned char* vp = static_cast<const unsigned char*>(a.v);
#pragma unroll
      for (int i = 0; i < (16 * S::kChunks + 31) / 32; ++i) {
        const int u = i * 32 + lane;
        const int r = u / S::kChunks, c = u - r * S::kChunks;
        const int64_t from = __shfl_sync(0xFFFFFFFFu, row, r & 15) * (D * kEb) + c * 16;
        const bool on = (mask >> (r & 15)) & 1u;
        if (16 * S::kChunks % 32 == 0 || u < 16 * S::kChunks) {
          const uint32_t to = dst + r * S::kPitch + (S::kSwizzle ? c ^ (r & 7) : c) * 16;
          cp_async16(to, kp + from, on);
          cp_async16(to + S::kOperand, vp + from, on);
        }
      }
      if (++sent < n) {
        advance(a, ahead);
        look_up();
      }
    }
    cp_commit();
  };
#pragma unroll 1
  for (int i = 0; i < S::kStages - 1; ++i) send();

  uint32_t q[KS][4];
  float o[NT][4];
  float m[2], l[2], mv[2];            // rows g and g + 8; mv: maximum of the V-weighted scores
  float unit[2];                      // factor of the raw scores
  int rows = 0;

  const uint32_t k_lane = kE4M3 ? ((lane >> 3) & 1) * 8 + (lane & 7) : (lane >> 4) * 8 + (lane & 7);
  const uint32_t k_chunk = kE4M3 ? lane >> 4 : (lane >> 3) & 1;
  const uint32_t v_lane = ((lane >> 3) & 1) * 8 + (lane & 7);
  const uint32_t v_chunk = lane >> 4;
  const uint32_t k_row = k_lane * S::kPitch, v_row = S::kOperand + v_lane * S::kPitch;

  bool fresh = true, whole = false;
#pragma unroll 1
  for (int i = 0; i < n; ++i) {
    if (fresh) {
      fresh = false;
      whole = at.tile == 0;
      const int group = a.hq / a.hk;
      const int kvh = at.hs / a.row_groups, first = (at.hs - kvh * a.row_groups) * kRows;
      rows = min(kRows, group - first);
      const TQ* qg = static_cast<const TQ*>(a.q) + at.b * a.qst + (int64_t)(kvh * group + first) * a.qsh;
      const unsigned short* qu = reinterpret_cast<const unsigned short*>(qg);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = g + (j & 1) * 8;
          // e4m3: a thread's four K codes are neighbours, so its k index runs 4 qd .. 4 qd + 3
          const int e = ks * 16 + (kE4M3 ? 4 * qd + (j >> 1) * 2 : 2 * qd + (j >> 1) * 8);
          uint32_t v = 0;
          if (r < rows) {
            const unsigned short* p = qu + r * a.qsh + e;
            v = a.q_pairs ? *reinterpret_cast<const uint32_t*>(p) : p[0] | (uint32_t)p[1] << 16;
          }
          q[ks][j] = v;
        }
      unit[0] = unit[1] = a.scale_log2;
      if constexpr (kE4M3) {
        // fp16 beside the fp16 that the codes become: each head scaled by a power of two so
        // that its largest element lies in [2^14, 2^15), exact down to 2^-28 of it
        float most[2] = {0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float x, y;
            unpack2<__is_same(TQ, __nv_bfloat16)>(q[ks][j], x, y);
            most[j & 1] = fmaxf(most[j & 1], fmaxf(fabsf(x), fabsf(y)));
          }
        float up[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          int e = (int)(__float_as_uint(quad_max(most[r])) >> 23);   // biased exponent
          e = e < 40 ? 40 : e == 255 ? 141 : e;
          up[r] = __uint_as_float((unsigned)(127 + 141 - e) << 23);
          unit[r] *= __uint_as_float((unsigned)(127 - 141 + e) << 23);
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float x, y;
            unpack2<__is_same(TQ, __nv_bfloat16)>(q[ks][j], x, y);
            q[ks][j] = f16x2_pack(x * up[j & 1], y * up[j & 1]);
          }
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
      m[0] = m[1] = mv[0] = mv[1] = -INFINITY;
      l[0] = l[1] = 0.f;
    }
    cp_wait<S::kStages - 2>();
    __syncwarp();
    send();                           // into the stage that every lane left in the last turn
    const int stage = i % S::kStages;
    const uint32_t base = ring + stage * S::kStage;
    const unsigned char* side = ring_p + stage * S::kStage + 2 * S::kOperand;
    const unsigned mask = *reinterpret_cast<const unsigned*>(side + (kE4M3 ? 128 : 0));
    if (mask != 0u) {
      float s[2][4] = {};
#pragma unroll
      for (int ks = 0; ks < KS; ks += kE4M3 ? 2 : 1) {
        uint32_t r[4];
        const uint32_t c = (kE4M3 ? ks : 2 * ks) + k_chunk;
        ldsm4(r, base + k_row + (S::kSwizzle ? c ^ (k_lane & 7) : c) * 16);
        if constexpr (kE4M3) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int t = 0; t < 2; ++t)
              mma<false>(s[t], q[ks + h], e4m3x2_f16x2(r[2 * h + t]), e4m3x2_f16x2(r[2 * h + t] >> 16));
        } else {
          mma<kBf16>(s[0], q[ks], r[0], r[1]);
          mma<kBf16>(s[1], q[ks], r[2], r[3]);
        }
      }
      float w[2][4];                  // numerators as V meets them
      float grow = 0.f;               // > 0: a maximum rose
      float top[2] = {-INFINITY, -INFINITY}, topv[2] = {-INFINITY, -INFINITY};
      float lv[2][2];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int tok = t * 8 + 2 * qd + j;
          float f = 1.f;
          if constexpr (kE4M3) {
            f = reinterpret_cast<const float*>(side)[tok];
            lv[t][j] = lg2(reinterpret_cast<const float*>(side)[16 + tok]);
          }
          const bool on = (mask >> tok) & 1u;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float& x = s[t][2 * r + j];
            x = on ? x * (kE4M3 ? unit[r] * f : unit[r]) : -INFINITY;
            top[r] = fmaxf(top[r], x);
            if constexpr (kE4M3) topv[r] = fmaxf(topv[r], on ? x + lv[t][j] : -INFINITY);
          }
        }
      float ref[2], refv[2], keep[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float now = fmaxf(m[r], quad_max(top[r]));
        ref[r] = ref_of(now);
        const float fade = ex2(m[r] - ref[r]);
        if (now > m[r]) grow = 1.f;
        m[r] = now;
        l[r] *= fade;
        keep[r] = fade;
        if constexpr (kE4M3) {
          const float nowv = fmaxf(mv[r], quad_max(topv[r]));
          refv[r] = ref_of(nowv);
          keep[r] = ex2(mv[r] - refv[r]);
          if (nowv > mv[r]) grow = 1.f;
          mv[r] = nowv;
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float x = s[t][2 * r + j];
            const float p = ex2(x - ref[r]);
            l[r] += p;
            if constexpr (kE4M3) {
              const bool on = (mask >> (t * 8 + 2 * qd + j)) & 1u;
              w[t][2 * r + j] = on ? ex2(x + lv[t][j] - refv[r]) : 0.f;
            } else {
              w[t][2 * r + j] = p * kLift;
            }
          }
      if (__any_sync(0xFFFFFFFFu, grow > 0.f)) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          o[j][0] *= keep[0];
          o[j][1] *= keep[0];
          o[j][2] *= keep[1];
          o[j][3] *= keep[1];
        }
      }
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float x = w[j >> 1][(j & 1) * 2], y = w[j >> 1][(j & 1) * 2 + 1];
        if constexpr (kTwoParts) split2<kBf16>(x, y, hi[j], lo[j]);
        else hi[j] = pack2<kBf16>(x, y);
      }
#pragma unroll
      for (int j = 0; j < NT / 2; j += kE4M3 ? 2 : 1) {
        uint32_t r[4];
        const uint32_t c = (kE4M3 ? j : 2 * j) + v_chunk;
        ldsm4t(r, base + v_row + (S::kSwizzle ? c ^ (v_lane & 7) : c) * 16);
        if constexpr (kE4M3) {
          // r[2 h], r[2 h + 1]: tokens 0-7 and 8-15 of chunk j + h; its bytes are
          // (token 2 qd: elements 2 g, 2 g + 1), (token 2 qd + 1: the same)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t x = __byte_perm(r[2 * h], 0, 0x3120), y = __byte_perm(r[2 * h + 1], 0, 0x3120);
            float (&even)[4] = o[2 * (j + h)];
            float (&odd)[4] = o[2 * (j + h) + 1];
            const uint32_t e0 = e4m3x2_f16x2(x), e1 = e4m3x2_f16x2(y);
            const uint32_t d0 = e4m3x2_f16x2(x >> 16), d1 = e4m3x2_f16x2(y >> 16);
            mma<false>(even, hi, e0, e1);
            mma<false>(odd, hi, d0, d1);
            if constexpr (kTwoParts) {
              mma<false>(even, lo, e0, e1);
              mma<false>(odd, lo, d0, d1);
            }
          }
        } else {
          mma<kBf16>(o[2 * j], hi, r[0], r[1]);
          mma<kBf16>(o[2 * j + 1], hi, r[2], r[3]);
          mma<kBf16>(o[2 * j], lo, r[0], r[1]);
          mma<kBf16>(o[2 * j + 1], lo, r[2], r[3]);
        }
      }
    }

    const bool last = at.tile + 1 == at.tiles;
    if (last || i + 1 == n) {
      // ---- the warps' results of the segment, joined: half a head's elements of 8 rows at a time
      if constexpr (!kE4M3) {
        mv[0] = m[0] - kLiftLog2;
        mv[1] = m[1] - kLiftLog2;
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float sum = quad_sum(l[r]);
        if (qd == 0) {
          s_m[warp][g + 8 * r] = m[r];
          s_v[warp][g + 8 * r] = mv[r];
          s_l[warp][g + 8 * r] = sum;
        }
      }
      whole = whole && last;
      const int kvh = at.hs / a.row_groups, first = (at.hs - kvh * a.row_groups) * kRows;
      const int64_t out_row = (int64_t)at.b * a.hq + kvh * (a.hq / a.hk) + first;
      // the slot of a segment that began here, or of one that began before
      const bool began = i + 1 - (at.tile + 1) >= 0;
      const int64_t slot = 2 * me + (began ? 1 : 0);
      float* pm = reinterpret_cast<float*>(meta + gridDim.x) + slot * kRows * 2;
      float* po = reinterpret_cast<float*>(meta + gridDim.x) + 2ll * gridDim.x * kRows * 2 + slot * kRows * D;
      if (i + 1 == n && tid == 0) {
        // tile of the whole row where the segment ends -> the CTA that has it
        const int64_t end = t1 + (at.tiles - at.tile - 1) - 1;
        const bool open = began && !last;
        meta[me] = Meta{open ? 1 : 0, at.b, at.hs, open ? (int)(((end + 1) * workers - 1) / total) : 0};
      }
      constexpr int kHalf = D / 2, kStride = kHalf + 8;
      for (int rh = 0; rh * 8 < rows; ++rh)
#pragma unroll
        for (int dh = 0; dh < 2; ++dh) {
          float* to = join + (warp * 8 + g) * kStride;
#pragma unroll
          for (int j = 0; j < NT / 2; j += kE4M3 ? 2 : 1) {
            const int k = dh * (NT / 2) + j;
            const float x0 = rh ? o[k][2] : o[k][0], x1 = rh ? o[k][3] : o[k][1];
            if constexpr (kE4M3) {
              const float y0 = rh ? o[k + 1][2] : o[k + 1][0], y1 = rh ? o[k + 1][3] : o[k + 1][1];
              *reinterpret_cast<float4*>(to + j * 8 + 4 * qd) = make_float4(x0, y0, x1, y1);
            } else {
              *reinterpret_cast<float2*>(to + j * 8 + 2 * qd) = make_float2(x0, x1);
            }
          }
          __syncthreads();
          for (int u = tid; u < 8 * (kHalf / 4); u += kBlock) {
            const int r8 = u / (kHalf / 4), e = (u - r8 * (kHalf / 4)) * 4, r = rh * 8 + r8;
            if (r >= rows) continue;
            float mm = -INFINITY, ll = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, s_m[w][r]);
            const float base2 = ref_of(mm);
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
              ll += s_l[w][r] * ex2(s_m[w][r] - base2);
              const float f = s_v[w][r] == -INFINITY ? 0.f : ex2(s_v[w][r] - base2);
              const float4 y = *reinterpret_cast<const float4*>(join + (w * 8 + r8) * kStride + e);
              x.x = fmaf(f, y.x, x.x);
              x.y = fmaf(f, y.y, x.y);
              x.z = fmaf(f, y.z, x.z);
              x.w = fmaf(f, y.w, x.w);
            }
            const int at_e = dh * kHalf + e;
            if (whole) {
              if (ll == 0.f) x = make_float4(0.f, 0.f, 0.f, 0.f);
              const float d = ll == 0.f ? 1.f : ll;
              uint2 y;
              y.x = pack2<__is_same(TQ, __nv_bfloat16)>(x.x / d, x.y / d);
              y.y = pack2<__is_same(TQ, __nv_bfloat16)>(x.z / d, x.w / d);
              *reinterpret_cast<uint2*>(static_cast<TQ*>(a.out) + (out_row + r) * D + at_e) = y;
              if (a.lse && at_e == 0) a.lse[out_row + r] = kLn2 * (base2 + log2f(ll));
            } else {
              *reinterpret_cast<float4*>(po + r * D + at_e) = x;
              if (at_e == 0) {
                pm[2 * r] = mm;
                pm[2 * r + 1] = ll;
              }
            }
          }
          __syncthreads();
        }
      fresh = true;
    }
    if (i + 1 < n) advance(a, at);
  }
  cp_wait<0>();
}

// Joins what the CTAs left of one segment: block (CTA, row) with the parts
// of that row, the CTA's own and those behind it, warp w every eighth part.
constexpr int kJoinWarps = 8;

template <typename TQ, int D>
__global__ void __launch_bounds__(kJoinWarps * 32) attention_join_kernel(const __grid_constant__ AttnArgs a) {
  __shared__ float s_o[kJoinWarps][D];
  __shared__ float s_x[kJoinWarps];
  ptx::grid_dep_wait();
  ptx::grid_dep_launch_dependents();
  const int tid = thread_here(), lane = tid & 31, warp = tid >> 5;
  // sequences without tokens have no tile: their zeros are written here
  const int64_t blocks = (int64_t)gridDim.x * gridDim.y;
  for (int64_t b = (int64_t)blockIdx.y * gridDim.x + blockIdx.x; b < a.batch; b += blocks) {
    if (length_of(a, b) != 0) continue;
    for (int i = tid; i < a.hq * D; i += kJoinWarps * 32)
      static_cast<TQ*>(a.out)[b * a.hq * D + i] = Pack<TQ>::from_f(0.f);
    if (a.lse)
      for (int i = tid; i < a.hq; i += kJoinWarps * 32) a.lse[b * a.hq + i] = -INFINITY;
  }
  const int64_t workers = gridDim.x, me = blockIdx.x;
  const Meta* meta = reinterpret_cast<const Meta*>(a.part);
  const Meta seg = meta[me];
  if (!seg.open) return;
  const int group = a.hq / a.hk;
  const int kvh = seg.hs / a.row_groups, first = (seg.hs - kvh * a.row_groups) * kRows;
  const int r = blockIdx.y;
  if (r >= min(kRows, group - first)) return;
  const float* pm = reinterpret_cast<const float*>(meta + workers);
  const float* po = pm + 2 * workers * kRows * 2;
  const int parts = seg.last - (int)me + 1;
  auto slot = [&](int i) { return i == 0 ? 2 * me + 1 : 2 * (me + i); };
  float top = -INFINITY;
  for (int i = tid; i < parts; i += kJoinWarps * 32) top = fmaxf(top, pm[(slot(i) * kRows + r) * 2]);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
  if (lane == 0) s_x[warp] = top;
  __syncthreads();
  for (int w = 0; w < kJoinWarps; ++w) top = fmaxf(top, s_x[w]);
  const float ref = ref_of(top);
  float o[D / 32], l = 0.f;
#pragma unroll
  for (int j = 0; j < D / 32; ++j) o[j] = 0.f;
#pragma unroll 4
  for (int i = warp; i < parts; i += kJoinWarps) {
    const float2 ml = *reinterpret_cast<const float2*>(pm + (slot(i) * kRows + r) * 2);
    const float f = ex2(ml.x - ref);
    l = fmaf(f, ml.y, l);
    const float* p = po + (slot(i) * kRows + r) * D;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) o[j] = fmaf(f, p[j * 32 + lane], o[j]);
  }
#pragma unroll
  for (int j = 0; j < D / 32; ++j) s_o[warp][j * 32 + lane] = o[j];
  __syncthreads();
  if (lane == 0) s_x[warp] = l;
  __syncthreads();
  l = 0.f;
  for (int w = 0; w < kJoinWarps; ++w) l += s_x[w];
  const int64_t row = (int64_t)seg.b * a.hq + kvh * group + first + r;
  for (int e = tid; e < D; e += kJoinWarps * 32) {
    float x = 0.f;
    for (int w = 0; w < kJoinWarps; ++w) x += s_o[w][e];
    static_cast<TQ*>(a.out)[row * D + e] = Pack<TQ>::from_f(l == 0.f ? 0.f : x / l);
  }
  if (a.lse && tid == 0) a.lse[row] = kLn2 * (ref + log2f(l));
}

// ---- which kernel, and its launch ---------------------------------------------------
struct Kernels {
  const void* main;
  const void* join;
  int smem, ctas;
  std::atomic<bool>* ready;      // per device: the shared-memory limit has been raised
};
constexpr int kMaxDevices = 64;

template <typename TQ, bool kE4M3, int D>
Kernels kernels() {
  static std::atomic<bool> ready[kMaxDevices];
  return Kernels{reinterpret_cast<const void*>(attention_kernel<TQ, kE4M3, D>),
                 reinterpret_cast<const void*>(attention_join_kernel<TQ, D>), Shape<D, kE4M3>::kSmem,
                 Shape<D, kE4M3>::kCtas, ready};
}
template <typename TQ, bool kE4M3>
Kernels kernels_of(int d) {
  switch (d) {
    case 64:
      return kernels<TQ, kE4M3, 64>();
    case 96:
      return kernels<TQ, kE4M3, 96>();
    case 128:
      return kernels<TQ, kE4M3, 128>();
    case 192:
      return kernels<TQ, kE4M3, 192>();
    case 256:
      return kernels<TQ, kE4M3, 256>();
    default:
      return Kernels{nullptr, nullptr, 0, 0, nullptr};
  }
}
// main == nullptr: the sizes or the type take the plain kernel.
Kernels find_kernels(int dtype, int cache_dtype, int d) {
  const bool e4m3 = cache_dtype == RMSNORM_KV_E4M3;
  if (dtype == RMSNORM_TP_BF16)
    return e4m3 ? kernels_of<__nv_bfloat16, true>(d) : kernels_of<__nv_bfloat16, false>(d);
  if (dtype == RMSNORM_TP_F16) return e4m3 ? kernels_of<__half, true>(d) : kernels_of<__half, false>(d);
  return Kernels{nullptr, nullptr, 0, 0, nullptr};
}

int row_groups_of(const rmsnorm_paged_attention_args* a) {
  return (a->q_heads / a->cache->kv_heads + kRows - 1) / kRows;
}
// CTAs of the main kernel: one resident wave, or a tile each of the longest lengths.
int64_t worker_count(const rmsnorm_paged_attention_args* a, const Kernels& k, int sms) {
  const int64_t tiles = (a->max_pages * a->cache->page_size + kTile - 1) / kTile;
  const int64_t most = tiles * a->batch * a->cache->kv_heads * row_groups_of(a);
  const int64_t wave = (int64_t)sms * k.ctas;
  return most < 1 ? 1 : most < wave ? most : wave;
}

template <typename TQ>
const void* any_fn(bool e4m3) {
  return e4m3 ? reinterpret_cast<const void*>(attention_any_kernel<TQ, unsigned char>)
              : reinterpret_cast<const void*>(attention_any_kernel<TQ, TQ>);
}

// Splits of the longest possible sequence: enough CTAs for two waves.
int any_splits(const rmsnorm_paged_attention_args* a, int sms) {
  const int64_t rows = a->batch * a->q_heads, most = a->max_pages * a->cache->page_size;
  int64_t s = (2 * sms * 4 + rows - 1) / (rows > 0 ? rows : 1);
  const int64_t by_len = (most + 2 * kAnyBlock - 1) / (2 * kAnyBlock);
  if (s > by_len) s = by_len;
  return (int)(s < 1 ? 1 : s > 256 ? 256 : s);
}

int check_attention(const char* who, const rmsnorm_paged_attention_args* a) {
  if (!a) return refuse(RMSNORM_TP_ERR_INVALID, "%s: NULL arguments", who);
  const int rc = check_cache(who, a->cache);
  if (rc != RMSNORM_TP_OK) return rc;
  const rmsnorm_kv_cache* c = a->cache;
  if (a->dtype != RMSNORM_TP_F32 && a->dtype != RMSNORM_TP_BF16 && a->dtype != RMSNORM_TP_F16)
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: unknown dtype %d", who, a->dtype);
  if (c->dtype != RMSNORM_KV_E4M3 && c->dtype != a->dtype)
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: a cache of dtype %d for queries of dtype %d", who,
                  c->dtype, a->dtype);
  if (a->q_heads < 1 || a->q_heads > 65536 || a->q_heads % c->kv_heads)
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: q_heads %d must be a multiple of kv_heads %d", who,
                  a->q_heads, c->kv_heads);
  if (a->batch < 0 || a->batch > 65535)
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: batch %lld outside [0, 65535]", who, (long long)a->batch);
  if (a->max_pages < 0 || a->max_pages * (int64_t)c->page_size > (int64_t(1) << 31) - 1)
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: %lld pages of %d tokens: a sequence holds under 2^31 tokens",
                  who, (long long)a->max_pages, c->page_size);
  if (a->device < 0) return refuse(RMSNORM_TP_ERR_INVALID, "%s: device %d", who, a->device);
  return RMSNORM_TP_OK;
}

}  // namespace
}  // namespace rtp

extern "C" {

size_t rmsnorm_paged_attention_workspace_bytes(const rmsnorm_paged_attention_args* a) {
  using namespace rtp;
  if (check_attention("paged_attention_workspace_bytes", a) != RMSNORM_TP_OK) return 0;
  const int sms = sm_count(a->device);
  if (sms < 1) {
    refuse(RMSNORM_TP_ERR_CUDA, "paged_attention_workspace_bytes: no device %d", a->device);
    return 0;
  }
  const Kernels k = find_kernels(a->dtype, a->cache->dtype, a->cache->head_dim);
  if (k.main != nullptr)
    return (size_t)worker_count(a, k, sms) *
           (sizeof(Meta) + 2 * kRows * (size_t)(a->cache->head_dim + 2) * sizeof(float));
  return (size_t)a->batch * a->q_heads * any_splits(a, sms) * (a->cache->head_dim + 2) * sizeof(float);
}

int rmsnorm_paged_attention(const rmsnorm_paged_attention_args* in, void* stream) {
  using namespace rtp;
  const char* who = "paged_attention";
  const int rc = check_attention(who, in);
  if (rc != RMSNORM_TP_OK || in->batch == 0) return rc;
  const rmsnorm_kv_cache* c = in->cache;
  if (!in->q || !in->out || !in->seq_lens || (in->max_pages > 0 && !in->page_table))
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: NULL tensor pointer", who);
  const int eb = elem_bytes(in->dtype);
  const int64_t so[2] = {(int64_t)in->q_heads * c->head_dim, c->head_dim};
  const View q = view_of(in->q, in->batch, in->q_heads, c->head_dim, in->q_strides, eb);
  if (q.s0 < 0 || q.s1 < 0) return refuse(RMSNORM_TP_ERR_INVALID, "%s: negative stride", who);
  if (views_overlap(view_of(in->out, in->batch, in->q_heads, c->head_dim, so, eb), q))
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: out overlaps q", who);
  const int sms = sm_count(in->device);
  if (sms < 1) return refuse(RMSNORM_TP_ERR_CUDA, "%s: no device %d", who, in->device);
  const size_t need = rmsnorm_paged_attention_workspace_bytes(in);
  if (!in->workspace || in->workspace_bytes < (int64_t)need)
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: workspace of %lld bytes < %zu", who,
                  (long long)in->workspace_bytes, need);
  AttnArgs a = {};
  a.q = in->q;
  a.out = in->out;
  a.lse = in->lse;
  a.k = c->k;
  a.v = c->v;
  a.ks = c->k_scale;
  a.vs = c->v_scale;
  a.table = in->page_table;
  a.lens = in->seq_lens;
  a.part = static_cast<float*>(in->workspace);
  a.qst = in->q_strides[0];
  a.qsh = in->q_strides[1];
  a.table_stride = in->page_table_stride;
  a.num_pages = c->num_pages;
  a.max_tokens = in->max_pages * c->page_size;
  a.batch = in->batch;
  a.hq = in->q_heads;
  a.hk = c->kv_heads;
  a.page = c->page_size;
  a.d = c->head_dim;
  a.scale_log2 = in->scale * kLog2e;
  a.row_groups = row_groups_of(in);
  a.segments = a.hk * a.row_groups;
  a.q_pairs = ((reinterpret_cast<uintptr_t>(in->q) & 3u) | (uintptr_t)((a.qst | a.qsh) & 1)) == 0;
  OnDevice on(in->device);
  if (on.err != cudaSuccess) return launch_failed(on.err, who);
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  void* args[] = {&a};
  const Kernels k = find_kernels(in->dtype, c->dtype, a.d);
  if (k.main != nullptr) {
    if (in->device >= kMaxDevices || !k.ready[in->device]) {
      const cudaError_t e =
          cudaFuncSetAttribute(k.main, cudaFuncAttributeMaxDynamicSharedMemorySize, k.smem);
      if (e != cudaSuccess) return launch_failed(e, who);
      if (in->device < kMaxDevices) k.ready[in->device] = true;
    }
    const unsigned n = (unsigned)worker_count(in, k, sms);
    cudaError_t e = launch_dependent(k.main, dim3(n), dim3(kBlock), k.smem, args, st);
    const int group = a.hq / a.hk;
    if (e == cudaSuccess)
      e = launch_dependent(k.join, dim3(n, group < kRows ? group : kRows), dim3(kJoinWarps * 32), 0, args, st);
    return e == cudaSuccess ? RMSNORM_TP_OK : launch_failed(e, who);
  }
  a.splits = any_splits(in, sms);
  const bool e4m3 = c->dtype == RMSNORM_KV_E4M3;
  const void* fn = in->dtype == RMSNORM_TP_F32    ? any_fn<float>(e4m3)
                   : in->dtype == RMSNORM_TP_BF16 ? any_fn<__nv_bfloat16>(e4m3)
                                                  : any_fn<__half>(e4m3);
  const void* join = in->dtype == RMSNORM_TP_F32
                         ? reinterpret_cast<const void*>(attention_join_any_kernel<float>)
                     : in->dtype == RMSNORM_TP_BF16
                         ? reinterpret_cast<const void*>(attention_join_any_kernel<__nv_bfloat16>)
                         : reinterpret_cast<const void*>(attention_join_any_kernel<__half>);
  cudaError_t e = launch_dependent(fn, dim3((unsigned)a.hq, (unsigned)a.batch, (unsigned)a.splits),
                                   dim3(kAnyBlock), 0, args, st);
  if (e == cudaSuccess)
    e = launch_dependent(join, dim3((unsigned)(a.batch * a.hq)), dim3(kAnyBlock), 0, args, st);
  return e == cudaSuccess ? RMSNORM_TP_OK : launch_failed(e, who);
}

}  // extern "C"
