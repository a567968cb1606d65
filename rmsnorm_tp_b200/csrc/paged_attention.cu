// Attention of one new token of each sequence over a paged cache.
//
//   s_j = scale q . k_j;  m = max s;  l = sum exp(s_j - m);  o = sum exp(s_j - m) v_j / l
//
// A sequence's tokens are divided over several CTAs ("splits"); each leaves its
// m, l and o (relative to its own m) in the workspace, and a second kernel joins
// them: o = sum_i exp(m_i - m) o_i / sum_i exp(m_i - m) l_i.
#include <float.h>

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
  int hq, hk, page, d, splits, max_pages;
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
  const int h = blockIdx.x, tid = threadIdx.x;
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
  const int64_t row = blockIdx.x;
  const float* w = a.part + row * a.splits * (a.d + 2);
  float m = -INFINITY, l = 0.f;
  for (int s = 0; s < a.splits; ++s) m = fmaxf(m, w[s * (a.d + 2)]);
  const float ref = m == -INFINITY ? 0.f : m;
  for (int s = 0; s < a.splits; ++s) l += exp2f(w[s * (a.d + 2)] - ref) * w[s * (a.d + 2) + 1];
  for (int i = threadIdx.x; i < a.d; i += kAnyBlock) {
    float o = 0.f;
    for (int s = 0; s < a.splits; ++s)
      o = fmaf(exp2f(w[s * (a.d + 2)] - ref), w[s * (a.d + 2) + 2 + i], o);
    static_cast<TQ*>(a.out)[row * a.d + i] = Pack<TQ>::from_f(l == 0.f ? 0.f : o / l);
  }
  if (a.lse && threadIdx.x == 0) a.lse[row] = kLn2 * (ref + log2f(l));
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
  if (sms < 1) return 0;
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
  a.max_pages = (int)in->max_pages;
  a.scale_log2 = in->scale * kLog2e;
  a.splits = any_splits(in, sms);
  OnDevice on(in->device);
  if (on.err != cudaSuccess) return launch_failed(on.err, who);
  const bool e4m3 = c->dtype == RMSNORM_KV_E4M3;
  const void* fn = in->dtype == RMSNORM_TP_F32    ? any_fn<float>(e4m3)
                   : in->dtype == RMSNORM_TP_BF16 ? any_fn<__nv_bfloat16>(e4m3)
                                                  : any_fn<__half>(e4m3);
  const void* join = in->dtype == RMSNORM_TP_F32
                         ? reinterpret_cast<const void*>(attention_join_any_kernel<float>)
                     : in->dtype == RMSNORM_TP_BF16
                         ? reinterpret_cast<const void*>(attention_join_any_kernel<__nv_bfloat16>)
                         : reinterpret_cast<const void*>(attention_join_any_kernel<__half>);
  void* args[] = {&a};
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e = launch_dependent(fn, dim3((unsigned)a.hq, (unsigned)a.batch, (unsigned)a.splits),
                                   dim3(kAnyBlock), 0, args, st);
  if (e == cudaSuccess)
    e = launch_dependent(join, dim3((unsigned)(a.batch * a.hq)), dim3(kAnyBlock), 0, args, st);
  return e == cudaSuccess ? RMSNORM_TP_OK : launch_failed(e, who);
}

}  // extern "C"
