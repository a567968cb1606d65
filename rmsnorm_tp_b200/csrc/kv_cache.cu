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
                             cudaStream_t stream, int cluster) {
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  if (get_dependent_launch()) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 0) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = (unsigned)cluster;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs++].val.clusterDim.z = 1;
  }
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
  FastDiv units, per_row, page_div;   // of a token (heads * d / 8), of a row (d / 8)
  int small;                          // num_slots under 2^31
};

constexpr int kBlock = 256;

// 8 elements of a cache row, zeros until they are loaded.
template <typename TC>
struct Eight {
  static constexpr int kWords = sizeof(TC) * 2;
  uint32_t w[kWords] = {};
  __device__ __forceinline__ void load(const TC* p) {
    if constexpr (kWords == 2) {
      asm("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
    } else {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4 x = ptx::ld_stream_v4(reinterpret_cast<const uint32_t*>(p) + i);
        w[i] = x.x, w[i + 1] = x.y, w[i + 2] = x.z, w[i + 3] = x.w;
      }
    }
  }
  // Scaled (e4m3 only) and rounded once.
  template <typename T>
  __device__ __forceinline__ void store(T* p, float scale) const {
    float f[8];
    if constexpr (kWords == 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 x = e4m3x2_to((unsigned short)(w[i / 2] >> (16 * (i & 1))));
        f[2 * i] = x.x * scale;
        f[2 * i + 1] = x.y * scale;
      }
    } else if constexpr (kWords == 4) {
      Pack<TC>::unpack(make_uint4(w[0], w[1], w[2], w[3]), f);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(w[e]);
    }
    if constexpr (sizeof(T) == 2) {
      ptx::st_v4(p, Pack<T>::pack(f));
    } else {
      const float a[4] = {f[0], f[1], f[2], f[3]}, b[4] = {f[4], f[5], f[6], f[7]};
      ptx::st_v4(p, Pack<T>::pack(a));
      ptx::st_v4(p + 4, Pack<T>::pack(b));
    }
  }
};

// A thread brings 8 elements of K and of V of one head of kTokens tokens, all asked for
// before the first is used; a warp's 16-bit outputs are 512 bytes in one piece. Bound by
// HBM: each row read once, written once. 32768 tokens of 8 heads of 128, e4m3 to bf16
// (203.7 MB): 33.9 us, 6.0 TB/s, 92 % of a copy (one token a thread and plain divisions: 41).
constexpr int kTokens = 4;

template <typename TC, typename T>
__global__ void __launch_bounds__(kBlock) kv_read_kernel(const __grid_constant__ ReadArgs a) {
  ptx::grid_dep_wait();
  const unsigned id = blockIdx.x * kBlock + thread_here();   // under 2^31
  const unsigned group = a.units.quotient(id), unit = id - group * a.units.by;
  const unsigned h = a.per_row.quotient(unit), e0 = (unit - h * a.per_row.by) * 8;
  const int64_t t0 = (int64_t)group * kTokens;
  if (t0 >= a.count) return;
  const int n = a.count - t0 < kTokens ? (int)(a.count - t0) : kTokens;
  int64_t at[kTokens];
#pragma unroll
  for (int i = 0; i < kTokens; ++i) at[i] = i < n ? a.slots[t0 + i] : -1;
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    if (at[i] < 0 || at[i] >= a.num_slots) {
      at[i] = -1;
      continue;
    }
    if (a.small) {
      const unsigned pg = a.page_div.quotient((unsigned)at[i]);
      at[i] = (int64_t)(pg * (uint64_t)a.heads + h) * a.page + ((unsigned)at[i] - pg * a.page);
    } else {
      const int64_t pg = at[i] / a.page;
      at[i] = (pg * a.heads + h) * a.page + (at[i] - pg * a.page);
    }
  }
  Eight<TC> k[kTokens], v[kTokens];
  float ks[kTokens], vs[kTokens];
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    ks[i] = vs[i] = 1.f;
    if (at[i] < 0) continue;
    k[i].load(static_cast<const TC*>(a.k) + at[i] * a.d + e0);
    v[i].load(static_cast<const TC*>(a.v) + at[i] * a.d + e0);
    if constexpr (sizeof(TC) == 1) {
      ks[i] = a.ks[at[i]];
      vs[i] = a.vs[at[i]];
    }
  }
  const int64_t step = (int64_t)a.heads * a.d;
  T* ko = static_cast<T*>(a.ko) + t0 * step + (int64_t)h * a.d + e0;
  T* vo = static_cast<T*>(a.vo) + t0 * step + (int64_t)h * a.d + e0;
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    if (i < n) {
      k[i].template store<T>(ko, ks[i]);
      v[i].template store<T>(vo, vs[i]);
    }
    ko += step;
    vo += step;
  }
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
  // a thread for every 8 elements of 4 tokens, numbered in 31 bits
  const int64_t units = (int64_t)c->kv_heads * (c->head_dim / 8);
  if (count < 0 || count / kTokens >= ((int64_t(1) << 31) - kBlock) / units - 1)   // (no product that wraps)
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: %lld slots of %d heads of %d: at most 2^36 elements", who,
                  (long long)count, c->kv_heads, c->head_dim);
  if (count == 0) return RMSNORM_TP_OK;
  if (!k_out || !v_out || !slots) return refuse(RMSNORM_TP_ERR_INVALID, "%s: NULL tensor pointer", who);
  if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15u)
    return refuse(RMSNORM_TP_ERR_INVALID, "%s: the outputs must be 16-byte aligned", who);
  ReadArgs a = {};
  a.k = c->k;
  a.v = c->v;
  a.ks = c->k_scale;
  a.vs = c->v_scale;
  a.ko = k_out;
  a.vo = v_out;
  a.slots = slots;
  a.num_slots = c->num_pages * c->page_size;
  a.count = count;
  a.page = c->page_size;
  a.heads = c->kv_heads;
  a.d = c->head_dim;
  a.per_row = FastDiv::of(c->head_dim / 8);
  a.units = FastDiv::of((unsigned)c->kv_heads * (c->head_dim / 8));
  a.page_div = FastDiv::of(c->page_size);
  a.small = a.num_slots < (int64_t(1) << 31);
  OnDevice on(device);
  if (on.err != cudaSuccess) return launch_failed(on.err, who);
  const void* fn = dtype == RMSNORM_TP_F32    ? read_fn<float>(c->dtype)
                   : dtype == RMSNORM_TP_BF16 ? read_fn<__nv_bfloat16>(c->dtype)
                                              : read_fn<__half>(c->dtype);
  const int64_t threads = (count + kTokens - 1) / kTokens * a.units.by;
  void* args[] = {&a};
  const cudaError_t e = launch_dependent(fn, dim3((unsigned)((threads + kBlock - 1) / kBlock)), dim3(kBlock),
                                         0, args, reinterpret_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? RMSNORM_TP_OK : launch_failed(e, who);
}
