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
  int row_groups;       // groups of 8 (16) query heads that share a kv head
  int segments;         // kv heads * row_groups
  int q_pairs;          // the queries' elements can be read two at a time
  int whole_pages;      // pages hold whole tiles of a warp
  int undivided;        // a CTA for each segment, which no other shares
  FastDiv page_div;
  float scale_log2;     // scale * log2(e): scores in base 2
};

constexpr int64_t kMostTiles = int64_t(1) << 36;   // of all heads: a CTA's share of them is an int
constexpr int64_t kMostTokens = (int64_t(1) << 31) - 128;   // a tile's last token is an int
constexpr float kLn2 = 0.69314718055994531f;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ int64_t length_of(const AttnArgs& a, int64_t b) {
  const int64_t n = a.lens[b];
  return n < 0 ? 0 : n > a.max_tokens ? a.max_tokens : n;
}

// ---- any type and head_dim --------------------------------------------------------
// (fp32, and the multiples of 16 that the tensor-core kernel has no shape for.) One CTA per
// (query head, sequence, split): a thread per token for the scores, a thread per element for
// the values. Reads the keys' rows uncoalesced and the cache once for each query head: one
// sequence of 262144 tokens, 8 heads of 128 over one (bf16), 1133 us against 30 there.
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
// heads. The products are K Q^T and V^T P with the tokens (then the elements) as the 16
// rows of mma.sync and 8 query heads as its columns, so a group of up to 8 pads nothing
// but itself, and over 16-bit caches mma.sync keeps up with the bytes (0.74 to 1.0 of a copy
// for groups of up to 16). tcgen05, with the tokens as its 128 rows and the heads as its
// columns, has not been tried; where the products are the larger part (the figures below) it
// may be worth it. A CTA of 4 warps takes tiles of 64 tokens, 16 for each warp, which runs its
// own softmax and its own cp.async ring (no CTA barrier in the loop; the loads run ahead over
// the borders of sequences); the warps' results are joined at a sequence's end.
//
// All (sequence, kv head, 8 or 16 query heads) are laid behind one another in tiles, each
// with one share more for its begin and end, and each CTA takes an equal run of shares, from
// the lengths on the device: ragged batches balance to a tile and nothing on the host knows
// a length. A run that ends inside a
// sequence leaves its reference, sum and o in the workspace (at most two such parts for
// each CTA), and the join kernel adds them in CTA order.
//
// The softmax's reference is a score seen, not the maximum: it moves only when a score
// passes it by more than 2^8, so most tiles need no maximum over the warp and no
// rescaling. Exponentials are taken of what is left over reference + 8, so they are at most
// 1 and a weighted V element is no larger than the element.
//
// Measured (device): 64 sequences of up to 16384 tokens, 32 + 8 heads of 128, e4m3 (1085 MB)
// 170 us, 6.4 TB/s; one sequence of 262144 tokens, 8 + 1 heads of 128, bf16 (134 MB) 30 us:
// 21 of streaming at 6.2 TB/s, 4 before the first tiles arrive (lengths, place, pages, rows:
// four memory round trips), 4.6 of the join; 48 of up to 2011, 16 + 16 heads of 64, fp16
// (185 MB) 38 us. Short of a copy (64 sequences of 4096, 4 kv heads): e4m3 with up to 8 query
// heads a kv head at head_dim 64 and 96 (0.56 to 0.62), with 9 to 16 (0.39, 0.45, 0.59, 0.65,
// 0.61 at 64, 96, 128, 192, 256) and, past 16 heads, all of them, as K and V are read once for
// each 16 (32 heads: 16-bit 0.42 to 0.49, e4m3 0.22 to 0.36). There 8 or 12 warps an SM issue
// in half of the cycles (46 to 54 %): a warp's turn is one chain of products, softmax and
// products, and too few warps hide it.
constexpr int kWarps = 4;
constexpr int kBlock = 32 * kWarps;
constexpr float kSlack = 8.f;           // how far scores may pass the reference (log2)
constexpr int kJoinBlock = 256;         // threads of the join kernel
constexpr int kSegment = 1;             // cost of a segment's begin and end, in tiles

// One CTA's share in the join of a segment (query heads of one kv head of one sequence)
// whose tiles `parts` CTAs from `owner` on have: units (4 elements) [u0, u1) of its rows
// from `row` on, 2^lg threads for each. parts == 0: none.
struct alignas(16) Share {
  int64_t row;
  int32_t owner, parts, u0, u1, lg, pad;
};

template <int D, bool kE4M3, int NG>
struct Shape {
  static constexpr int kRowBytes = D * (kE4M3 ? 1 : 2);
  static constexpr int kChunks = kRowBytes / 16;             // 16-byte chunks of a row
  // rows of 8 k chunks are swizzled (chunk ^ (row & 7)), others padded to an odd number:
  // either way 8 rows of one chunk fall into 8 different bank groups
  static constexpr bool kSwizzle = kChunks % 8 == 0;
  static constexpr int kPitch = (kSwizzle ? kChunks : (kChunks | 1)) * 16;
  // tokens of a warp's tile, in blocks of 16: two where a row is short (e4m3) and the
  // registers allow it, so that the loop's own work is shared by more of them. 64 sequences
  // of 4096 tokens and 4 kv heads, one and two blocks: head_dim 64 42 and 36 us, 128 55 and
  // 53, 256 115 and 96; but 96 56 and 60, 192 83 and 93 (fewer CTAs fit), which keep one.
  static constexpr int kBlocks = kE4M3 && NG == 1 && D != 96 && D != 192 ? 2 : 1;
  static constexpr int kTok = 16 * kBlocks;
  static constexpr int kTile = kTok * kWarps;                // of a CTA's tile
  static constexpr int kOperand = kTok * kPitch;             // one warp's K (or V) tile
  static constexpr int kScales = kE4M3 ? 8 * kTok : 0;       // bytes of its scales
  static constexpr int kSide = kScales + 16;                 // they and its mask, behind the rings
  static constexpr int kTiles = 2 * kOperand;
  static constexpr int kStage = kTiles + kSide;
  // lanes that load one row, and rows of one load instruction
  static constexpr int kLanes = kChunks % 8 == 0 ? 8 : kChunks % 4 == 0 ? 4 : 2;
  static constexpr int kRowsAtOnce = 32 / kLanes;
  // a segment's join goes through the stage that each warp has just left: 8 heads of fp32 at
  // once where they fit it, else half their elements
  static constexpr int kHalves = 8 * (D + 4) * 4 <= kTiles ? 1 : 2;
  static constexpr int kJoinPitch = D / kHalves + 4;         // 8 heads' rows on all banks
  static_assert(8 * kJoinPitch * 4 <= kTiles, "the join fits a stage");
  // three CTAs of at most 74 KB on an SM (and 168 registers a thread: NG = 1) where at
  // least three stages fit, else two of 111 KB, else one
  static constexpr int kThree = NG == 1 ? 74 * 1024 / (kWarps * kStage) : 0;
  static constexpr int kTwo = 111 * 1024 / (kWarps * kStage);
  static constexpr int kOne = 222 * 1024 / (kWarps * kStage);
  static constexpr int kCtas = kThree >= 3 ? 3 : kTwo >= 3 ? 2 : 1;
  static constexpr int kFit = kCtas == 3 ? kThree : kCtas == 2 ? kTwo : kOne;
  static constexpr int kStages = kFit > 6 ? 6 : kFit;
  static constexpr int kSmem = kWarps * kStages * kStage;
  static_assert(kStages >= 3, "the ring needs three stages");
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
// 8 x 8 matrix of 16-bit elements transposed over the warp.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
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
// Two 16-bit parts of numerators x, y >= 0, together exact to 2^-16 of them (fp16 to 2^-20,
// or 2^-25 where that is more): the value cut off, and what is left. Neither is negative,
// and the second never 0 beside a first that is not, so that a numerator meets an infinity
// in V as one positive number would. fp16's smallest number 2^-24 is not far below the
// numerators, so there the second part is not raised to it, which would add it to every
// token behind a long sequence's few that count: instead the first is cut from a value
// that is less than x by 2^-24 and 2^-20 of it, or is 0, and the second is rounded to
// nearest; a weight under 2^-32 of the heaviest is then 0 in both, and makes NaN of an infinity.
template <bool kBf16>
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  float hx, hy;
  if constexpr (kBf16) {
    constexpr float kLeast = 1.17549435e-38f;   // 2^-126
    hi = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
    unpack2<kBf16>(hi, hx, hy);
    lo = pack2<kBf16>(fmaxf(x - hx, kLeast), fmaxf(y - hy, kLeast));
  } else {
    constexpr float kLess = 1.f - 9.5367431640625e-7f, kLeast = 5.9604644775390625e-8f;   // 1 - 2^-20, 2^-24
    asm("cvt.rz.relu.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(fmaf(y, kLess, -kLeast)), "f"(fmaf(x, kLess, -kLeast)));
    unpack2<kBf16>(hi, hx, hy);
    lo = pack2<kBf16>(x - hx, y - hy);
  }
}
// Over the lanes that hold one head (lane / 4 differs).
__device__ __forceinline__ float head_max(float v) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  return v;
}
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
// The reference of exponentials: 0 where nothing has been seen (their value is 0 then).
__device__ __forceinline__ float ref_of(float m) { return m == -INFINITY ? 0.f : m; }

// Place in the row of tiles: tile `tile` of the `tiles` of segment (sequence b, kv head,
// group of its query heads).
// `rem`: what is left of the CTA's run, from this tile on.
struct Place {
  int b, kvh, rg, tile, tiles, len, rem;
};

// a / b of non-negative numbers, in 32 bits where they fit (a 64-bit division takes some
// hundred instructions, and a CTA cannot load before its first).
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return (unsigned)a / (unsigned)b;
  return a / b;
}

template <int kTile>
__device__ __forceinline__ int tiles_of(int64_t len) { return (int)((len + kTile - 1) / kTile); }

// Shares of a sequence's segment: its tiles, and kSegment for its queries and its join.
template <int kTile>
__device__ __forceinline__ int64_t shares_of(int64_t len) { return len == 0 ? 0 : tiles_of<kTile>(len) + kSegment; }

// To the next tile, if rem says that there is one.
template <int kTile>
__device__ __forceinline__ void advance(const AttnArgs& a, Place& p) {
  --p.rem;
  if (++p.tile < p.tiles) return;
  p.rem -= kSegment;
  if (p.rem <= 0) return;
  p.tile = 0;
  if (++p.rg < a.row_groups) return;
  p.rg = 0;
  if (++p.kvh < a.hk) return;
  p.kvh = 0;
  do {
    ++p.b;
    p.len = (int)length_of(a, p.b);
  } while (p.len == 0);
  p.tiles = tiles_of<kTile>(p.len);
}

// NG: groups of 8 query heads that one CTA holds.
template <typename TQ, bool kE4M3, int D, int NG>
__global__ void __launch_bounds__(kBlock, Shape<D, kE4M3, NG>::kCtas)
attention_kernel(const __grid_constant__ AttnArgs a) {
  using S = Shape<D, kE4M3, NG>;
  constexpr bool kQBf16 = __is_same(TQ, __nv_bfloat16);
  constexpr bool kBf16 = !kE4M3 && kQBf16;   // of the products: e4m3 codes become fp16
  // the numerators as two 16-bit parts where their rounding to one would be of the output's
  // own size; one fp16 part (2^-11) beside a bf16 output (2^-8)
  constexpr bool kTwoParts = !kE4M3 || !kQBf16;
  // fp16 numerators (e4m3: times V's scale) run up to 2^15, so that fp16's smallest number is
  // 2^-31 of the reference's: an element that is 0 in the tokens of weight is made of the others
  constexpr float kLiftLog2 = kBf16 ? 0.f : 15.f, kLift = kBf16 ? 1.f : 32768.f;
  constexpr int KS = D / 16, MB = S::kBlocks, kTok = S::kTok, kTile = S::kTile;
  constexpr unsigned kAll = kTok == 32 ? ~0u : 0xFFFFu;
  constexpr int kRows = 8 * NG;
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ float s_m[kWarps][kRows], s_l[kWarps][kRows], s_v[kWarps][kRows];
  __shared__ int64_t s_scan[kWarps];
  __shared__ int64_t s_rest;
  __shared__ int s_b;
  // No early launch of the next kernel: its CTAs took registers on some SMs while this
  // one's wave was being placed, so that these SMs ran one CTA fewer (2048 segments of 1024
  // tokens, head_dim 64: 109 us a call back to back, 79 without).
  ptx::grid_dep_wait();
  const int tid = thread_here(), lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, qd = lane & 3;

  // this CTA's run of shares [t0, t1): every thread sums those of a run of sequences
  int64_t each = 0, more = 0, t0 = 0, t1 = 0;
  const int64_t me = blockIdx.x;
  Share* meta = reinterpret_cast<Share*>(a.part) + 2 * me;   // divided: of the segment that began before, of one left open
  Place at;
  int hs;
  if (a.undivided) {
    at.b = (int)((unsigned)blockIdx.x / (unsigned)a.segments);
    hs = (int)((unsigned)blockIdx.x - (unsigned)at.b * a.segments);
    at.len = (int)length_of(a, at.b);
    at.tiles = tiles_of<kTile>(at.len);
    at.tile = 0;
    at.rem = at.tiles;
  } else {
    const int64_t per = (a.batch + kBlock - 1) / kBlock;
    int64_t mine = 0;
    for (int64_t b = tid * per; b < (tid + 1) * per && b < a.batch; ++b)
      mine += shares_of<kTile>(length_of(a, b)) * a.segments;
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
    if (tid < 2) meta[tid].parts = 0;
    if (me >= workers) return;
    // the first `more` CTAs have one share more than the others
    each = quotient(total, workers);
    more = total - each * workers;
    t0 = me * each + (me < more ? me : more);
    t1 = t0 + each + (me < more ? 1 : 0);
    if (upto - mine <= t0 && t0 < upto) {
      int64_t rest = t0 - (upto - mine);
      int64_t b = tid * per;
      for (;; ++b) {
        const int64_t n = shares_of<kTile>(length_of(a, b)) * a.segments;
        if (rest < n) break;
        rest -= n;
      }
      s_b = (int)b;
      s_rest = rest;
    }
    __syncthreads();
    at.b = s_b;
    at.len = (int)length_of(a, at.b);
    at.tiles = tiles_of<kTile>(at.len);
    hs = (int)quotient(s_rest, at.tiles + kSegment);
    const int into_segment = (int)(s_rest - (int64_t)hs * (at.tiles + kSegment)) - kSegment;
    at.tile = into_segment > 0 ? into_segment : 0;
    at.rem = (int)(t1 - t0) + (into_segment < 0 ? into_segment : 0);   // under 2^31: kMostTiles
    if (at.rem <= 0) return;            // a run of nothing but a segment's extra share
  }
  at.kvh = hs / a.row_groups;
  at.rg = hs - at.kvh * a.row_groups;
  auto worker_of = [&](int64_t share) {
    const int64_t line = more * (each + 1);
    return (int)(share < line ? quotient(share, each + 1) : more + quotient(share - line, each));
  };
  const int group = a.hq / a.hk;
  auto row_of = [&](const Place& p) { return (int64_t)p.b * a.hq + p.kvh * group + p.rg * kRows; };
  // this CTA's share in a segment whose first tile lies in share `from` of the run
  auto share_of = [&](const Place& p, int64_t from) {
    const int owner = worker_of(from), parts = worker_of(from + p.tiles - 1) - owner + 1, i = (int)me - owner;
    const int units = min(kRows, group - p.rg * kRows) * (D / 4);
    const int u0 = units * i / parts, u1 = units * (i + 1) / parts;
    // a power of two of threads for a unit, no more than half of them idle
    int lg = 0;
    while ((2 << lg) * (u1 - u0) <= kJoinBlock && (1 << lg) < parts) ++lg;
    return Share{row_of(p), owner, parts, u0, u1, lg, 0};
  };
  if (tid == 0 && at.tile > 0) meta[0] = share_of(at, t0 - at.tile);
  if (at.rem == 0) {                    // undivided, and the sequence has no tokens
    const int rows = min(kRows, group - at.rg * kRows);
    for (int i = tid; i < rows * D; i += kBlock)
      static_cast<TQ*>(a.out)[row_of(at) * D + i] = Pack<TQ>::from_f(0.f);
    if (a.lse && tid < rows) a.lse[row_of(at) + tid] = -INFINITY;
    return;
  }

  static_assert(!S::kSwizzle || S::kPitch % 128 == 0, "the swizzle's address bits are those of a chunk in 128 bytes");
  constexpr int kRing = S::kStages * S::kTiles;   // of a warp
  const uint32_t ring = ptx::smem_addr(smem) + warp * kRing;
  unsigned char* sides = smem + kWarps * kRing + warp * S::kStages * S::kSide;

  // ---- loads ----
  const int lr = lane / S::kLanes, lc = lane % S::kLanes;
  const unsigned char* kp = static_cast<const unsigned char*>(a.k) + lc * 16;
  const unsigned char* vp = static_cast<const unsigned char*>(a.v) + lc * 16;
  // this lane's chunk of its row in the tile, for rows lr and lr + 4 of 8
  const uint32_t to0 = lr * S::kPitch + (S::kSwizzle ? lc ^ (lr & 7) : lc) * 16;
  const uint32_t to1 = lr * S::kPitch + (S::kSwizzle ? lc ^ ((lr + S::kRowsAtOnce) & 7) : lc) * 16;
  const int lane_tok = warp * kTok + (a.whole_pages ? 0 : lane & (kTok - 1));
  Place ahead = at;
  uint32_t into = 0;                  // stage that the next tile goes to
  int32_t page_id = -1, page_off = 0; // read one tile early
  int table_of = -1;
  const int32_t* table = nullptr;     // of sequence table_of
  // whole pages of tiles: the warp's tokens lie in one page, one row behind another; else
  // lane l (for 16 tokens also l + 16) knows the row of token l
  auto look_up = [&]() {
    const int t = ahead.tile * kTile + lane_tok;
    const unsigned pg = a.page_div.quotient(t);
    page_off = t - (int)pg * a.page;
    if (table_of != ahead.b) {
      table_of = ahead.b;
      table = a.table + table_of * a.table_stride;
    }
    page_id = t < ahead.len ? table[pg] : -1;
  };
  look_up();
  auto send = [&]() {
    if (ahead.rem > 0) {
      const uint32_t dst = ring + into * S::kTiles;
      unsigned char* side = sides + into * S::kSide;
      const bool live = (unsigned)page_id < (unsigned)a.num_pages;
      const int64_t row = live ? ((int64_t)page_id * a.hk + ahead.kvh) * a.page + page_off : 0;
      const int rest = ahead.len - (ahead.tile * kTile + lane_tok);
      unsigned mask;
      if (a.whole_pages) mask = !live ? 0u : rest >= kTok ? kAll : (1u << rest) - 1u;
      else mask = __ballot_sync(0xFFFFFFFFu, live) & kAll;
      if (lane == 0) *reinterpret_cast<unsigned*>(side + S::kScales) = mask;
      if constexpr (kE4M3) {          // K's scales, then V's: for 16 tokens half the lanes each
        const int64_t r = a.whole_pages ? row + (lane & (kTok - 1)) : row;
        const bool on = (mask >> (lane & (kTok - 1))) & 1u;
        cp_async4_if(ptx::smem_addr(side) + lane * 4, (lane < kTok ? a.ks : a.vs) + (on ? r : 0), on);
        if (kTok == 32) cp_async4_if(ptx::smem_addr(side) + 128 + lane * 4, a.vs + (on ? r : 0), on);
      }
      if (a.whole_pages && mask == kAll) {
        const int64_t from = (row + lr) * S::kRowBytes;
        const unsigned char* kf = kp + from;
        const unsigned char* vf = vp + from;
#pragma unroll
        for (int i = 0; i < kTok / S::kRowsAtOnce; ++i)
#pragma unroll
          for (int k = 0; k < S::kChunks / S::kLanes; ++k) {
            const uint32_t to = dst + (i & 1 ? to1 : to0) + i * S::kRowsAtOnce * S::kPitch + k * S::kLanes * 16;
            const int at = i * S::kRowsAtOnce * S::kRowBytes + k * S::kLanes * 16;
            cp_async16(to, kf + at);
            cp_async16(to + S::kOperand, vf + at);
          }
      } else {
#pragma unroll
        for (int i = 0; i < kTok / S::kRowsAtOnce; ++i) {
          const int r = i * S::kRowsAtOnce + lr;
          const int64_t from = (a.whole_pages ? row + r : __shfl_sync(0xFFFFFFFFu, row, r)) * S::kRowBytes;
          const bool on = (mask >> r) & 1u;
          const int64_t safe = on ? from : 0;
          const uint32_t to = dst + (i & 1 ? to1 : to0) + i * S::kRowsAtOnce * S::kPitch;
#pragma unroll
          for (int k = 0; k < S::kChunks / S::kLanes; ++k) {
            cp_async16_if(to + k * S::kLanes * 16, kp + safe + k * S::kLanes * 16, on);
            cp_async16_if(to + S::kOperand + k * S::kLanes * 16, vp + safe + k * S::kLanes * 16, on);
          }
        }
      }
      into = into + 1 == S::kStages ? 0 : into + 1;
      advance<kTile>(a, ahead);
      if (ahead.rem > 0) look_up();
    }
    cp_commit();
  };
#pragma unroll 1
  for (int i = 0; i < S::kStages - 1; ++i) send();

  uint32_t q[NG][KS][2];
  float o[NG][KS][4];                 // [16 elements][head 2 qd, 2 qd + 1] of each group of 8
  float m[NG][2], l[NG][2], mv[NG][2];   // references of the scores and (e4m3) of the V-weighted ones
  float unit[NG][2];                  // factor of the raw scores
  uint32_t stage = 0;

  // K as 16 tokens x 16 elements: matrices (tokens 0-7, 8-15) x (chunk, next chunk)
  const uint32_t k_tok = ((lane >> 3) & 1) * 8 + (lane & 7), k_chunk = lane >> 4;
  // V^T: 16-bit (chunk, next chunk) x (tokens 0-7, 8-15), e4m3 as K
  const uint32_t v_tok = kE4M3 ? k_tok : (lane >> 4) * 8 + (lane & 7);
  const uint32_t v_chunk = kE4M3 ? k_chunk : (lane >> 3) & 1;
  const uint32_t k_lane = k_tok * S::kPitch + (S::kSwizzle ? k_chunk ^ (k_tok & 7) : k_chunk) * 16;
  const uint32_t v_lane = S::kOperand + v_tok * S::kPitch + (S::kSwizzle ? v_chunk ^ (v_tok & 7) : v_chunk) * 16;
  auto chunk = [](uint32_t at, uint32_t c) {
    return S::kSwizzle ? (at ^ ((c & 7u) * 16)) + (c & ~7u) * 16 : at + c * 16;
  };

  auto load_q = [&](const Place& p) {
    const int first = p.rg * kRows, rows = min(kRows, group - first);
    const unsigned short* qu = static_cast<const unsigned short*>(a.q) + p.b * a.qst +
                               (int64_t)(p.kvh * group + first) * a.qsh;
#pragma unroll
    for (int x = 0; x < NG; ++x)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int r = 8 * x + g;
          // e4m3: a thread's four K codes are neighbours, so its k index runs 4 qd .. 4 qd + 3
          const int e = ks * 16 + (kE4M3 ? 4 * qd + 2 * j : 2 * qd + 8 * j);
          uint32_t v = 0;
          if (r < rows) {
            const unsigned short* at = qu + r * a.qsh + e;
            v = a.q_pairs ? *reinterpret_cast<const uint32_t*>(at) : at[0] | (uint32_t)at[1] << 16;
          }
          q[x][ks][j] = v;
        }
  };
  load_q(at);
#pragma unroll 1
  while (at.rem > 0) {
    // ---- a segment, or what this CTA has of it ----
    const bool began = at.tile == 0;
    const int rows = min(kRows, group - at.rg * kRows);
    const int end = min(at.tiles - at.tile, at.rem) + at.tile;
    {
#pragma unroll
      for (int x = 0; x < NG; ++x) {
        unit[x][0] = unit[x][1] = a.scale_log2;
        if constexpr (kE4M3) {
          // fp16 beside the fp16 that the codes become: each head scaled by a power of two so
          // that its largest element lies in [2^14, 2^15), exact down to 2^-28 of it
          float most = 0.f;
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float lo, hi;
              unpack2<kQBf16>(q[x][ks][j], lo, hi);
              most = fmaxf(most, fmaxf(fabsf(lo), fabsf(hi)));
            }
          most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 1));
          most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 2));
          int e = (int)(__float_as_uint(most) >> 23);   // biased exponent
          e = e < 40 ? 40 : e == 255 ? 141 : e;
          const float up = __uint_as_float((unsigned)(127 + 141 - e) << 23);
          const float down = __uint_as_float((unsigned)(127 - 141 + e) << 23);
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float lo, hi;
              unpack2<kQBf16>(q[x][ks][j], lo, hi);
              q[x][ks][j] = f16x2_pack(lo * up, hi * up);
            }
          // lane 4 g' holds head g's factor; this lane's scores are those of heads 2 qd, 2 qd + 1
          unit[x][0] *= __shfl_sync(0xFFFFFFFFu, down, 8 * qd);
          unit[x][1] *= __shfl_sync(0xFFFFFFFFu, down, 8 * qd + 4);
        }
#pragma unroll
        for (int j = 0; j < KS; ++j) o[x][j][0] = o[x][j][1] = o[x][j][2] = o[x][j][3] = 0.f;
        m[x][0] = m[x][1] = mv[x][0] = mv[x][1] = -INFINITY;
        l[x][0] = l[x][1] = 0.f;
      }
    }
#pragma unroll 1
    for (int tile = at.tile; tile < end; ++tile) {
      cp_wait<S::kStages - 2>();
      __syncwarp();
      send();                           // into the stage that every lane left in the last turn
      // swizzled: chunk c + k_chunk (c even) of row k_tok lies at the address of chunk k_chunk
      // with the low bits of c flipped
      const uint32_t k_at = ring + stage * S::kTiles + k_lane, v_at = ring + stage * S::kTiles + v_lane;
      const unsigned char* side = sides + stage * S::kSide;
      stage = stage + 1 == S::kStages ? 0 : stage + 1;
      const unsigned mask = *reinterpret_cast<const unsigned*>(side + S::kScales);
      if (mask != 0u) {
        // (token g, heads 2 qd, 2 qd + 1), (token g + 8, the same) of each block
        float s[MB][NG][4];
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          float s2[NG][4];              // the odd steps' sums: two chains instead of one
#pragma unroll
          for (int x = 0; x < NG; ++x)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[mb][x][j] = s2[x][j] = 0.f;
#pragma unroll
          for (int ks = 0; ks < KS; ks += 2) {
            uint32_t r[4], r2[4];
            const uint32_t from = k_at + mb * 16 * S::kPitch;
            if constexpr (kE4M3) {
              uint32_t w[4];
              ldsm4(w, chunk(from, ks));
              r[0] = e4m3x2_f16x2(w[0]), r[2] = e4m3x2_f16x2(w[0] >> 16);
              r[1] = e4m3x2_f16x2(w[1]), r[3] = e4m3x2_f16x2(w[1] >> 16);
              r2[0] = e4m3x2_f16x2(w[2]), r2[2] = e4m3x2_f16x2(w[2] >> 16);
              r2[1] = e4m3x2_f16x2(w[3]), r2[3] = e4m3x2_f16x2(w[3] >> 16);
            } else {
              ldsm4(r, chunk(from, 2 * ks));
              ldsm4(r2, chunk(from, 2 * ks + 2));
            }
#pragma unroll
            for (int x = 0; x < NG; ++x) {
              mma<kBf16>(s[mb][x], r, q[x][ks][0], q[x][ks][1]);
              mma<kBf16>(s2[x], r2, q[x][ks + 1][0], q[x][ks + 1][1]);
            }
          }
#pragma unroll
          for (int x = 0; x < NG; ++x)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[mb][x][j] += s2[x][j];
        }
        // tokens g + 8 t of all blocks
        bool on[2 * MB];
        float lv[2 * MB];
        bool rise = false;
#pragma unroll
        for (int t = 0; t < 2 * MB; ++t) {
          on[t] = (mask >> (g + 8 * t)) & 1u;
          float ksc = 1.f;
          lv[t] = 0.f;
          if constexpr (kE4M3) {
            ksc = reinterpret_cast<const float*>(side)[8 * t + g];
            lv[t] = lg2(reinterpret_cast<const float*>(side)[kTok + 8 * t + g]);
          }
#pragma unroll
          for (int x = 0; x < NG; ++x)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float& v = s[t >> 1][x][2 * (t & 1) + h];
              v = on[t] ? v * (kE4M3 ? unit[x][h] * ksc : unit[x][h]) : -INFINITY;
              rise |= v > m[x][h] + kSlack;
              if constexpr (kE4M3) rise |= on[t] && v + lv[t] > mv[x][h] + kSlack;
            }
        }
        if (__any_sync(0xFFFFFFFFu, rise)) {
#pragma unroll
          for (int x = 0; x < NG; ++x)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float top = -INFINITY, topv = -INFINITY;
#pragma unroll
              for (int t = 0; t < 2 * MB; ++t) {
                const float v = s[t >> 1][x][2 * (t & 1) + h];
                top = fmaxf(top, v);
                if (on[t]) topv = fmaxf(topv, v + lv[t]);
              }
              const float now = fmaxf(m[x][h], head_max(top));
              float keep = ex2(m[x][h] - ref_of(now));
              l[x][h] *= keep;
              m[x][h] = now;
              if constexpr (kE4M3) {
                const float nowv = fmaxf(mv[x][h], head_max(topv));
                keep = ex2(mv[x][h] - ref_of(nowv));
                mv[x][h] = nowv;
              }
#pragma unroll
              for (int j = 0; j < KS; ++j) {
                o[x][j][h] *= keep;
                o[x][j][2 + h] *= keep;
              }
            }
        }
        uint32_t hi[MB][NG][2], lo[MB][NG][2];   // P as 16 tokens x 8 heads
#pragma unroll
        for (int x = 0; x < NG; ++x) {
          const float ref[2] = {ref_of(m[x][0]) + kSlack, ref_of(m[x][1]) + kSlack};
          const float refv[2] = {ref_of(mv[x][0]) + (kSlack - kLiftLog2), ref_of(mv[x][1]) + (kSlack - kLiftLog2)};
#pragma unroll
          for (int t = 0; t < 2 * MB; ++t) {
            uint32_t& to_hi = hi[t >> 1][x][t & 1];
            uint32_t& to_lo = lo[t >> 1][x][t & 1];
            float w[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float v = s[t >> 1][x][2 * (t & 1) + h], p = ex2(v - ref[h]);
              l[x][h] += p;
              w[h] = kE4M3 ? (on[t] ? ex2(v + lv[t] - refv[h]) : 0.f) : p * kLift;
            }
            if constexpr (kTwoParts) {
              split2<kBf16>(w[0], w[1], to_hi, to_lo);
              to_lo = transposed(to_lo);
            } else {
              to_hi = pack2<kBf16>(w[0], w[1]);
            }
            to_hi = transposed(to_hi);
          }
        }
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
          for (int j = 0; j < KS; j += kE4M3 ? 2 : 1) {
            uint32_t r[4], r2[4];
            const uint32_t from = chunk(v_at + mb * 16 * S::kPitch, kE4M3 ? j : 2 * j);
            if constexpr (kE4M3) {
              // bytes of w: (token 2 qd: elements 2 g, 2 g + 1), (token 2 qd + 1: the same), so row
              // g of the product is element 2 g and row g + 8 element 2 g + 1
              uint32_t w[4];
              ldsm4t(w, from);
#pragma unroll
              for (int t = 0; t < 4; ++t) w[t] = __byte_perm(w[t], 0, 0x3120);
              r[0] = e4m3x2_f16x2(w[0]), r[1] = e4m3x2_f16x2(w[0] >> 16);
              r[2] = e4m3x2_f16x2(w[1]), r[3] = e4m3x2_f16x2(w[1] >> 16);
              r2[0] = e4m3x2_f16x2(w[2]), r2[1] = e4m3x2_f16x2(w[2] >> 16);
              r2[2] = e4m3x2_f16x2(w[3]), r2[3] = e4m3x2_f16x2(w[3] >> 16);
            } else {
              ldsm4t(r, from);
            }
#pragma unroll
            for (int x = 0; x < NG; ++x) {
              mma<kBf16>(o[x][j], r, hi[mb][x][0], hi[mb][x][1]);
              if constexpr (kTwoParts) mma<kBf16>(o[x][j], r, lo[mb][x][0], lo[mb][x][1]);
              if constexpr (kE4M3) {
                mma<kBf16>(o[x][j + 1], r2, hi[mb][x][0], hi[mb][x][1]);
                if constexpr (kTwoParts) mma<kBf16>(o[x][j + 1], r2, lo[mb][x][0], lo[mb][x][1]);
              }
            }
          }
      }
    }

    const bool last = end == at.tiles, whole = began && last;
    // the next segment's queries, asked for before the join
    Place next = at;
    next.tile = end - 1;
    next.rem = at.rem - (end - 1 - at.tile);
    advance<kTile>(a, next);
    if (next.rem > 0) load_q(next);
    {
      // ---- the warps' results of the segment, joined through the stages just left (the next
      // copies into them are sent behind the last barrier)
      unsigned char* left = smem + (stage == 0 ? S::kStages - 1 : stage - 1) * S::kTiles;
#pragma unroll
      for (int x = 0; x < NG; ++x)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float sum = head_sum(l[x][h]);
          if (g == 0) {
            // what the sums are relative to (-inf: nothing seen)
            s_m[warp][8 * x + 2 * qd + h] = m[x][h] + kSlack;
            s_v[warp][8 * x + 2 * qd + h] = (kE4M3 ? mv[x][h] : m[x][h]) + kSlack;
            s_l[warp][8 * x + 2 * qd + h] = sum;
          }
        }
      const int64_t out_row = row_of(at);
      // the part of a segment that began before, or of one left open
      const int64_t slot = 2 * me + (began ? 1 : 0);
      float* pm = reinterpret_cast<float*>(reinterpret_cast<Share*>(a.part) + 2 * gridDim.x) + slot * kRows * 2;
      float* po = reinterpret_cast<float*>(reinterpret_cast<Share*>(a.part) + 2 * gridDim.x) +
                  2ll * gridDim.x * kRows * 2 + slot * kRows * D;
      if (tid == 0 && began && !last)
        meta[1] = share_of(at, t1 - end);
      constexpr int kPart = D / S::kHalves;   // elements of a head at a time
#pragma unroll
      for (int x = 0; x < NG; ++x) {
        if (8 * x >= rows) break;
#pragma unroll
        for (int dh = 0; dh < S::kHalves; ++dh) {
          float* to = reinterpret_cast<float*>(left + warp * kRing) + 2 * qd * S::kJoinPitch;
#pragma unroll
          for (int j = 0; j < KS / S::kHalves; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float (&v)[4] = o[x][dh * (KS / S::kHalves) + j];
              float* p = to + h * S::kJoinPitch + 16 * j;
              if constexpr (kE4M3) {
                *reinterpret_cast<float2*>(p + 2 * g) = make_float2(v[h], v[2 + h]);
              } else {
                p[g] = v[h];
                p[g + 8] = v[2 + h];
              }
            }
          __syncthreads();
          for (int u = tid; u < 8 * (kPart / 4); u += kBlock) {
            const int r8 = u / (kPart / 4), e = (u - r8 * (kPart / 4)) * 4, r = 8 * x + r8;
            if (r >= rows) continue;
            float mm = -INFINITY, ll = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, s_m[w][r]);
            const float ref = ref_of(mm);
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
              ll += s_l[w][r] * ex2(s_m[w][r] - ref);
              const float f = s_v[w][r] == -INFINITY ? 0.f : ex2(s_v[w][r] - ref) * (1.f / kLift);
              const float4 z =
                  *reinterpret_cast<const float4*>(reinterpret_cast<float*>(left + w * kRing) + r8 * S::kJoinPitch + e);
              y.x = fmaf(f, z.x, y.x);
              y.y = fmaf(f, z.y, y.y);
              y.z = fmaf(f, z.z, y.z);
              y.w = fmaf(f, z.w, y.w);
            }
            const int at_e = dh * kPart + e;
            if (whole) {
              const float over = 1.f / (ll == 0.f ? 1.f : ll);   // no weight at all: o is 0
              uint2 out;
              out.x = pack2<kQBf16>(y.x * over, y.y * over);
              out.y = pack2<kQBf16>(y.z * over, y.w * over);
              *reinterpret_cast<uint2*>(static_cast<TQ*>(a.out) + (out_row + r) * D + at_e) = out;
              if (a.lse && at_e == 0) a.lse[out_row + r] = kLn2 * (ref + log2f(ll));
            } else {
              *reinterpret_cast<float4*>(po + r * D + at_e) = y;
              if (at_e == 0) {
                pm[2 * r] = mm;
                pm[2 * r + 1] = ll;
              }
            }
          }
          __syncthreads();
        }
      }
    }
    at = next;
  }
  cp_wait<0>();
}

// Joins what the CTAs left of a segment: every CTA that had a part of it takes an equal
// share of its elements over all parts (one CTA for all of one head took 16 us of one long
// sequence, this 4.6). A thread adds 4 elements of a head over some of the
// parts (neighbouring threads the others), then the threads and warps of these
// elements are added in a fixed order. Bound by latency (a few L2 round trips), so it is
// kept short rather than unrolled.

// Reference, sum and 4 elements of a softmax over some of the tokens.
struct Part {
  float m, v[5];
  __device__ __forceinline__ void to(float top) {
    const float f = ex2(m - ref_of(top));
    m = top;
#pragma unroll
    for (int j = 0; j < 5; ++j) v[j] *= f;
  }
  __device__ __forceinline__ void add(const Part& p) {
#pragma unroll
    for (int j = 0; j < 5; ++j) v[j] += p.v[j];
  }
};

template <typename TQ, int D, int NG>
__global__ void __launch_bounds__(kJoinBlock) attention_join_kernel(const __grid_constant__ AttnArgs a) {
  constexpr int kRows = 8 * NG, kUnits = D / 4;
  __shared__ Part s_part[kJoinBlock / 32];
  ptx::grid_dep_wait();
  const int tid = thread_here();
  const int64_t workers = gridDim.x, me = blockIdx.x;
  const Share* shares = reinterpret_cast<const Share*>(a.part);
  const float* pm = reinterpret_cast<const float*>(shares + 2 * workers);
  const float* po = pm + 2 * workers * kRows * 2;
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const Share sh = shares[2 * me + which];
    if (sh.parts == 0) continue;
    const int slices = 1 << sh.lg, lanes = min(slices, 32);
#pragma unroll 1
    for (int ub = sh.u0; ub < sh.u1; ub += kJoinBlock >> sh.lg) {
      const int u = ub + (tid >> sh.lg), r = u / kUnits, e = (u % kUnits) * 4;
      if (slices <= 32 && ub + ((tid & ~31) >> sh.lg) >= sh.u1) break;   // nothing for this warp
      Part mine{-INFINITY, {0.f, 0.f, 0.f, 0.f, 0.f}};
      int i = tid & (slices - 1);       // up to a power of two: parts may be fewer
      if (u < sh.u1 && i < sh.parts) {
        // the owner's part is that of a segment left open, the others' of one begun before
        const int first = (2 * sh.owner + (i == 0 ? 1 : 2 * i)) * kRows + r;   // under 2^15 rows
        const float* ml = pm + first * 2;
        const float4* y = reinterpret_cast<const float4*>(po + (int64_t)first * D + e);
        mine = Part{ml[0], {ml[1], y->x, y->y, y->z, y->w}};
#pragma unroll 1
        for (i += slices; i < sh.parts; i += slices) {
          const int at = (2 * (sh.owner + i)) * kRows + r;
          ml = pm + at * 2;
          y = reinterpret_cast<const float4*>(po + (int64_t)at * D + e);
          Part one{ml[0], {ml[1], y->x, y->y, y->z, y->w}};
          const float top = fmaxf(mine.m, one.m);
          mine.to(top);
          one.to(top);
          mine.add(one);
        }
      }
      float top = mine.m;
#pragma unroll 1
      for (int o = lanes >> 1; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
      mine.to(top);
#pragma unroll 1
      for (int o = lanes >> 1; o > 0; o >>= 1)
#pragma unroll
        for (int j = 0; j < 5; ++j) mine.v[j] += __shfl_xor_sync(0xFFFFFFFFu, mine.v[j], o);
      if (slices > 32) {              // several warps for one unit
        __syncthreads();
        if ((tid & 31) == 0) s_part[tid >> 5] = mine;
        __syncthreads();
        if ((tid & (slices - 1)) == 0) {
          const Part* others = s_part + (tid >> 5);
#pragma unroll 1
          for (int w = 1; w < slices / 32; ++w) top = fmaxf(top, others[w].m);
          mine.to(top);
#pragma unroll 1
          for (int w = 1; w < slices / 32; ++w) {
            Part other = others[w];
            other.to(top);
            mine.add(other);
          }
        }
      }
      if (u < sh.u1 && (tid & (slices - 1)) == 0) {
        const int64_t row = sh.row + r;
        const float over = 1.f / (mine.v[0] == 0.f ? 1.f : mine.v[0]);   // no weight at all: o is 0
        constexpr bool kQBf16 = __is_same(TQ, __nv_bfloat16);
        uint2 out;
        out.x = pack2<kQBf16>(mine.v[1] * over, mine.v[2] * over);
        out.y = pack2<kQBf16>(mine.v[3] * over, mine.v[4] * over);
        *reinterpret_cast<uint2*>(static_cast<TQ*>(a.out) + row * D + e) = out;
        if (a.lse && e == 0) a.lse[row] = kLn2 * (ref_of(top) + log2f(mine.v[0]));
      }
    }
  }
  // sequences without tokens have no tile: their zeros are written here
  for (int64_t b = me; b < a.batch; b += workers) {
    if (length_of(a, b) != 0) continue;
    for (int i = tid; i < a.hq * D; i += kJoinBlock)
      static_cast<TQ*>(a.out)[b * a.hq * D + i] = Pack<TQ>::from_f(0.f);
    if (a.lse)
      for (int i = tid; i < a.hq; i += kJoinBlock) a.lse[b * a.hq + i] = -INFINITY;
  }
}

// ---- which kernel, and its launch ---------------------------------------------------
struct Kernels {
  const void* main;
  const void* join;
  int smem, ctas, rows, warp_tokens;
  std::atomic<bool>* ready;   // per device: the shared-memory limit has been raised
};
constexpr int kMaxDevices = 64;

template <typename TQ, bool kE4M3, int D, int NG>
Kernels kernels() {
  static std::atomic<bool> ready[kMaxDevices];
  return Kernels{reinterpret_cast<const void*>(attention_kernel<TQ, kE4M3, D, NG>),
                 reinterpret_cast<const void*>(attention_join_kernel<TQ, D, NG>),
                 Shape<D, kE4M3, NG>::kSmem, Shape<D, kE4M3, NG>::kCtas, 8 * NG,
                 Shape<D, kE4M3, NG>::kTok, ready};
}
template <typename TQ, bool kE4M3, int NG>
Kernels kernels_of(int d) {
  switch (d) {
    case 64:
      return kernels<TQ, kE4M3, 64, NG>();
    case 96:
      return kernels<TQ, kE4M3, 96, NG>();
    case 128:
      return kernels<TQ, kE4M3, 128, NG>();
    case 192:
      return kernels<TQ, kE4M3, 192, NG>();
    case 256:
      return kernels<TQ, kE4M3, 256, NG>();
    default:
      return Kernels{};
  }
}
// main == nullptr: the sizes or the type take the plain kernel. Groups of more than 8 query
// heads take two of mma's 8 columns at once, so that K and V leave shared memory once.
Kernels find_kernels(const rmsnorm_paged_attention_args* a) {
  const bool e4m3 = a->cache->dtype == RMSNORM_KV_E4M3, bf16 = a->dtype == RMSNORM_TP_BF16;
  if (!bf16 && a->dtype != RMSNORM_TP_F16) return Kernels{};
  const int d = a->cache->head_dim;
  if (a->q_heads / a->cache->kv_heads <= 8) {
    if (bf16) return e4m3 ? kernels_of<__nv_bfloat16, true, 1>(d) : kernels_of<__nv_bfloat16, false, 1>(d);
    return e4m3 ? kernels_of<__half, true, 1>(d) : kernels_of<__half, false, 1>(d);
  }
  if (bf16) return e4m3 ? kernels_of<__nv_bfloat16, true, 2>(d) : kernels_of<__nv_bfloat16, false, 2>(d);
  return e4m3 ? kernels_of<__half, true, 2>(d) : kernels_of<__half, false, 2>(d);
}

int row_groups_of(const rmsnorm_paged_attention_args* a, const Kernels& k) {
  return (a->q_heads / a->cache->kv_heads + k.rows - 1) / k.rows;
}
// Whether each segment gets a CTA of its own and there is no join: up to 512 tokens of
// capacity. Divided and undivided, device time of 4 sequences of one kv head of
// 128: 7.9 and 5.9 us at 256 tokens, 8.4 and 10.5 at 512, 8.2 and 13.3 at 768, where the
// second launch and the workspace cost the host 4 us; 128 such segments: 9.9 and 7.9, 12.9
// and 10.7, 14.4 and 13.7.
bool undivided(const rmsnorm_paged_attention_args* a, const Kernels& k) {
  return a->max_pages * a->cache->page_size <= 512 &&
         a->batch * a->cache->kv_heads * row_groups_of(a, k) < (int64_t(1) << 30);
}
// CTAs of the main kernel: one resident wave, or a tile each of the longest lengths.
int64_t worker_count(const rmsnorm_paged_attention_args* a, const Kernels& k, int sms) {
  const int tile = k.warp_tokens * kWarps;
  const int64_t tiles = (a->max_pages * a->cache->page_size + tile - 1) / tile;
  const int64_t most = tiles * a->batch * a->cache->kv_heads * row_groups_of(a, k);
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
  if (a->max_pages < 0 || a->max_pages > kMostTokens / c->page_size)   // (no product that wraps)
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: %lld pages of %d tokens: a sequence holds at most 2^31 - 128",
                  who, (long long)a->max_pages, c->page_size);
  if ((a->max_pages * (int64_t)c->page_size / 64 + 2) * a->batch * a->q_heads > kMostTiles)
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: %lld sequences of %d heads and %lld tokens: too many", who,
                  (long long)a->batch, a->q_heads, (long long)(a->max_pages * (int64_t)c->page_size));
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
  const Kernels k = find_kernels(a);
  if (k.main != nullptr && undivided(a, k)) return 0;
  if (k.main != nullptr)
    return (size_t)worker_count(a, k, sms) * 2 *
           (sizeof(Share) + k.rows * (size_t)(a->cache->head_dim + 2) * sizeof(float));
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
  if ((reinterpret_cast<uintptr_t>(in->out) | reinterpret_cast<uintptr_t>(in->workspace)) & 15u)
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: out and the workspace must be 16-byte aligned", who);
  const int eb = elem_bytes(in->dtype);
  const int64_t so[2] = {(int64_t)in->q_heads * c->head_dim, c->head_dim};
  const View q = view_of(in->q, in->batch, in->q_heads, c->head_dim, in->q_strides, eb);
  if (q.s0 < 0 || q.s1 < 0) return refuse(RMSNORM_TP_ERR_INVALID, "%s: negative stride", who);
  if (views_overlap(view_of(in->out, in->batch, in->q_heads, c->head_dim, so, eb), q))
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: out overlaps q", who);
  const int sms = sm_count(in->device);
  if (sms < 1) return refuse(RMSNORM_TP_ERR_CUDA, "%s: no device %d", who, in->device);
  const size_t need = rmsnorm_paged_attention_workspace_bytes(in);
  if (need > 0 && (!in->workspace || in->workspace_bytes < (int64_t)need))
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
  a.q_pairs = ((reinterpret_cast<uintptr_t>(in->q) & 3u) | (uintptr_t)((a.qst | a.qsh) & 1)) == 0;
  OnDevice on(in->device);
  if (on.err != cudaSuccess) return launch_failed(on.err, who);
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  void* args[] = {&a};
  const Kernels k = find_kernels(in);
  if (k.main != nullptr) {
    a.row_groups = row_groups_of(in, k);
    a.segments = a.hk * a.row_groups;
    a.whole_pages = a.page % k.warp_tokens == 0;
    a.page_div = FastDiv::of(a.page);
    if (in->device >= kMaxDevices || !k.ready[in->device]) {
      const cudaError_t e =
          cudaFuncSetAttribute(k.main, cudaFuncAttributeMaxDynamicSharedMemorySize, k.smem);
      if (e != cudaSuccess) return launch_failed(e, who);
      if (in->device < kMaxDevices) k.ready[in->device] = true;
    }
    a.undivided = undivided(in, k);
    if (a.undivided) {
      const cudaError_t e =
          launch_dependent(k.main, dim3((unsigned)(a.batch * a.segments)), dim3(kBlock), k.smem, args, st);
      return e == cudaSuccess ? RMSNORM_TP_OK : launch_failed(e, who);
    }
    const unsigned n = (unsigned)worker_count(in, k, sms);
    cudaError_t e = launch_dependent(k.main, dim3(n), dim3(kBlock), k.smem, args, st);
    if (e == cudaSuccess) e = launch_dependent(k.join, dim3(n), dim3(kJoinBlock), 0, args, st);
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
