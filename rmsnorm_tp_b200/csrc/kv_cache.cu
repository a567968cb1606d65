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

// 8 elements from memory in fp32.
template <typename TC>
__device__ __forceinline__ void load8(const TC* p, float (&f)[8]) {
  if constexpr (sizeof(TC) == 1) {
    uint2 c;
    asm("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(c.x), "=r"(c.y) : "l"(p));
    const uint32_t w[2] = {c.x, c.y};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = e4m3x2_to((unsigned short)(w[i / 2] >> (16 * (i & 1))));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  } else if constexpr (sizeof(TC) == 2) {
    Pack<TC>::unpack(ptx::ld_stream_v4(p), f);
  } else {
    const uint4 a = ptx::ld_stream_v4(p), b = ptx::ld_stream_v4(p + 4);
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(w[e]);
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  if constexpr (sizeof(T) == 2) {
    ptx::st_v4(p, Pack<T>::pack(f));
  } else {
    const float a[4] = {f[0], f[1], f[2], f[3]}, b[4] = {f[4], f[5], f[6], f[7]};
    ptx::st_v4(p, Pack<T>::pack(a));
    ptx::st_v4(p + 4, Pack<T>::pack(b));
  }
}

// A thread brings 8 elements of K and of V of one row, so that a warp's 16-bit outputs
// are 512 bytes in one piece. Bound by HBM: each row read once, written once.
template <typename TC, typename T>
__global__ void __launch_bounds__(kBlock) kv_read_kernel(const __grid_constant__ ReadArgs a) {
  ptx::grid_dep_wait();
  ptx::grid_dep_launch_dependents();
  const unsigned tid = thread_here();
  const unsigned per_row = a.d / 8, rows = kBlock / per_row;   // 2 to 32; rows of this CTA
  const unsigned r = tid / per_row, e0 = (tid - r * per_row) * 8;
  const int64_t row = (int64_t)blockIdx.x * rows + r;
  if (r >= rows || row >= a.count * a.heads) return;
  const int64_t t = (unsigned)row / (unsigned)a.heads;   // at most 2^31 rows
  const int h = (int)(row - t * a.heads);
  const int64_t slot = a.slots[t];
  float k[8] = {}, v[8] = {};
  if (slot >= 0 && slot < a.num_slots) {
    int64_t pg;
    int off;
    page_of(slot, a.page, a.num_slots, pg, off);
    const int64_t at = (pg * a.heads + h) * a.page + off;
    load8(static_cast<const TC*>(a.k) + at * a.d + e0, k);
    load8(static_cast<const TC*>(a.v) + at * a.d + e0, v);
    if constexpr (sizeof(TC) == 1) {
      const float ks = a.ks[at], vs = a.vs[at];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        k[e] *= ks;
        v[e] *= vs;
      }
    }
  }
  store8(static_cast<T*>(a.ko) + row * a.d + e0, k);
  store8(static_cast<T*>(a.vo) + row * a.d + e0, v);
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
  const int64_t per_block = kBlock / (c->head_dim / 8), rows = count * c->kv_heads;
  void* args[] = {&a};
  const cudaError_t e = launch_dependent(fn, dim3((unsigned)((rows + per_block - 1) / per_block)),
                                         dim3(kBlock), 0, args, reinterpret_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? RMSNORM_TP_OK : launch_failed(e, who);
}
