// Rows of the paged cache read back by slot, and what the operators on heads
// share on the host: the cache's checks and the dependent launch.
#include <atomic>

#include "heads_common.cuh"

namespace rtp {

int sm_count(int device) {
  static std::atomic<int> known[64];
  if (device < 0) return 0;
  int n = device < 64 ? known[device].load(std::memory_order_relaxed) : 0;
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
      cudaGetLastError();
      return 0;
    }
    if (device < 64) known[device].store(n, std::memory_order_relaxed);
  }
  return n;
}

cudaError_t launch_dependent(const void* fn, dim3 grid, dim3 block, size_t smem, void** args,
                             cudaStream_t stream) {
  if (!get_dependent_launch()) return cudaLaunchKernel(fn, grid, block, args, smem, stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelExC(&cfg, fn, args);
}

int check_cache(const char* who, const rmsnorm_kv_cache* c) {
  if (!c) return refuse(RMSNORM_TP_ERR_INVALID, "%s: NULL cache", who);
  if (c->dtype < RMSNORM_TP_F32 || c->dtype > RMSNORM_KV_E4M3)
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: unknown cache dtype %d", who, c->dtype);
  if (c->page_size < 1 || c->kv_heads < 1 || c->kv_heads > 65536 || c->num_pages < 0 ||
      c->num_pages > (int64_t(1) << 31) - 1)
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: a cache of %lld pages of %d tokens and %d heads", who,
                  (long long)c->num_pages, c->page_size, c->kv_heads);
  if (c->head_dim < 16 || c->head_dim > 256 || c->head_dim % 16)
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: cache head_dim %d must be a multiple of 16 up to 256", who,
                  c->head_dim);
  if (c->num_pages > 0 && (!c->k || !c->v))
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: NULL cache tensor", who);
  if (c->num_pages > 0 && c->dtype == RMSNORM_KV_E4M3 && (!c->k_scale || !c->v_scale))
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: an e4m3 cache without scales", who);
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15u)
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: the cache must be 16-byte aligned", who);
  return RMSNORM_TP_OK;
}

namespace {

struct ReadArgs {
  const void* k;
  const void* v;
  const float* ks;
  const float* vs;
  void* ko;
  void* vo;
  const int64_t* slots;
  int64_t num_slots, count;
  int page, heads, d;
};

constexpr int kBlock = 256;

// One thread per 16 elements of an output row.
template <typename TC, typename T>
__global__ void __launch_bounds__(kBlock) kv_read_kernel(const __grid_constant__ ReadArgs a) {
  constexpr bool kE4M3 = sizeof(TC) == 1;
  ptx::grid_dep_wait();
  const int per_row = a.d / 16;
  const int64_t n = a.count * a.heads * per_row;
  const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if (i >= 2 * n) return;
  const bool is_v = i >= n;
  const int64_t u = is_v ? i - n : i;
  const int64_t row = u / per_row;
  const int e0 = (int)(u - row * per_row) * 16;
  const int64_t t = row / a.heads;
  const int h = (int)(row - t * a.heads);
  const int64_t slot = a.slots[t];
  float f[16];
  if (slot < 0 || slot >= a.num_slots) {
#pragma unroll
    for (int e = 0; e < 16; ++e) f[e] = 0.f;
  } else {
    const int64_t pg = slot / a.page;
    const int64_t at = (pg * a.heads + h) * a.page + (slot - pg * a.page);
    const TC* x = static_cast<const TC*>(is_v ? a.v : a.k) + at * a.d + e0;
    const float scale = kE4M3 ? (is_v ? a.vs : a.ks)[at] : 1.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      if constexpr (kE4M3)
        f[e] = e4m3_to(reinterpret_cast<const unsigned char*>(x)[e]) * scale;
      else
        f[e] = Pack<TC>::to_f(x[e]);
    }
  }
  T* y = static_cast<T*>(is_v ? a.vo : a.ko) + row * a.d + e0;
#pragma unroll
  for (int e = 0; e < 16; ++e) y[e] = Pack<T>::from_f(f[e]);
}

template <typename T>
const void* read_fn(int cache_dtype) {
  switch (cache_dtype) {
    case RMSNORM_KV_E4M3:
      return reinterpret_cast<const void*>(kv_read_kernel<unsigned char, T>);
    case RMSNORM_TP_F32:
      return reinterpret_cast<const void*>(kv_read_kernel<float, T>);
    case RMSNORM_TP_BF16:
      return reinterpret_cast<const void*>(kv_read_kernel<__nv_bfloat16, T>);
    default:
      return reinterpret_cast<const void*>(kv_read_kernel<__half, T>);
  }
}

}  // namespace
}  // namespace rtp

extern "C" int rmsnorm_kv_read(const rmsnorm_kv_cache* c, void* k_out, void* v_out,
                               const int64_t* slots, int64_t count, int dtype, int device,
                               void* stream) {
  using namespace rtp;
  const char* who = "kv_read";
  const int rc = check_cache(who, c);
  if (rc != RMSNORM_TP_OK) return rc;
  if (dtype != RMSNORM_TP_F32 && dtype != RMSNORM_TP_BF16 && dtype != RMSNORM_TP_F16)
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: unknown dtype %d", who, dtype);
  if (count < 0 || count > (int64_t(1) << 31) / c->kv_heads)
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: %lld slots of %d heads: at most 2^31 rows", who,
                  (long long)count, c->kv_heads);
  if (count == 0) return RMSNORM_TP_OK;
  if (!k_out || !v_out || !slots) return refuse(RMSNORM_TP_ERR_INVALID, "%s: NULL tensor pointer", who);
  if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15u)
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: the outputs must be 16-byte aligned", who);
  ReadArgs a{c->k,  c->v,  c->k_scale, c->v_scale, k_out, v_out, slots, c->num_pages * c->page_size,
             count, c->page_size, c->kv_heads, c->head_dim};
  OnDevice on(device);
  if (on.err != cudaSuccess) return launch_failed(on.err, who);
  const void* fn = dtype == RMSNORM_TP_F32    ? read_fn<float>(c->dtype)
                   : dtype == RMSNORM_TP_BF16 ? read_fn<__nv_bfloat16>(c->dtype)
                                              : read_fn<__half>(c->dtype);
  const int64_t n = 2 * count * c->kv_heads * (c->head_dim / 16);
  void* args[] = {&a};
  const cudaError_t e = launch_dependent(fn, dim3((unsigned)((n + kBlock - 1) / kBlock)), dim3(kBlock), 0,
                                         args, reinterpret_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? RMSNORM_TP_OK : launch_failed(e, who);
}
