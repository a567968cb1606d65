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
__device__ __forceinline__ int64_t cache_row(int64_t slot, int head, int heads, int page) {
  const int64_t pg = slot / page;
  return (pg * heads + head) * page + (slot - pg * page);
}

// ---- any head_dim, alignment and stride: one warp per row ----------------------
// Lane l holds the pairs l, l + 32, ...; a row is read twice (its sum of squares,
// then its elements), the second time from L1.
template <typename T, bool kWrite>
__global__ void __launch_bounds__(kBlock) qk_rope_any_kernel(const __grid_constant__ QkArgs a) {
  ptx::grid_dep_wait();
  const int lane = threadIdx.x & 31;
  const int heads = a.hq + a.hk + (kWrite ? a.hk : 0);
  const int64_t row = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (row >= a.tokens * heads) return;
  const int64_t t = row / heads;
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
  const int64_t at = cache_row(slot, hh, a.hk, a.page);
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
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
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
    for (int i = threadIdx.x; i < a.d; i += kBlock) {
      float s = 0.f;
      for (int v = 0; v < kWarps; ++v) s += dw[v * a.d + i];
      a.ws[((int64_t)blockIdx.x * 2 + part) * a.d + i] = s;
    }
    __syncthreads();
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
  const void* fn = in->dtype == RMSNORM_TP_F32
                       ? reinterpret_cast<const void*>(qk_rope_any_kernel<float, kWrite>)
                   : in->dtype == RMSNORM_TP_BF16
                       ? reinterpret_cast<const void*>(qk_rope_any_kernel<__nv_bfloat16, kWrite>)
                       : reinterpret_cast<const void*>(qk_rope_any_kernel<__half, kWrite>);
  void* args[] = {&a};
  const cudaError_t e = launch_dependent(fn, dim3((unsigned)((rows + kWarps - 1) / kWarps)), dim3(kBlock),
                                         0, args, reinterpret_cast<cudaStream_t>(stream));
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
  if (norm && (!in->dweight || !in->workspace ||
               in->workspace_bytes < (int64_t)rmsnorm_qk_rope_backward_workspace_bytes(in->head_dim)))
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: NULL dweight or a workspace of %lld bytes < %zu", who,
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
    const int64_t want = (a.tokens * a.hq + kWarps - 1) / kWarps;
    grid = (int)(want < kBackwardMaxGrid ? want : kBackwardMaxGrid);
    const void* fn = in->dtype == RMSNORM_TP_F32
                         ? reinterpret_cast<const void*>(qk_rope_backward_any_kernel<float>)
                     : in->dtype == RMSNORM_TP_BF16
                         ? reinterpret_cast<const void*>(qk_rope_backward_any_kernel<__nv_bfloat16>)
                         : reinterpret_cast<const void*>(qk_rope_backward_any_kernel<__half>);
    void* args[] = {&a};
    const size_t smem = norm ? (size_t)kWarps * a.d * sizeof(float) : 0;
    const cudaError_t e = launch_dependent(fn, dim3((unsigned)grid), dim3(kBlock), smem, args, st);
    if (e != cudaSuccess) return launch_failed(e, who);
  }
  if (norm) {   // no tokens: zeros
    const cudaError_t e = launch_dw_reduce(static_cast<const float*>(in->workspace), grid,
                                           2 * (int64_t)in->head_dim, in->dweight, in->dtype, st);
    if (e != cudaSuccess) return launch_failed(e, who);
  }
  return RMSNORM_TP_OK;
}

}  // extern "C"
