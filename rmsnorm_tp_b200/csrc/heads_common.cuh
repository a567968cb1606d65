// Shared by the operators on query / key heads, the paged cache and the
// single-token attention (qk_rope.cu, kv_cache.cu, paged_attention.cu):
// argument checks, launches, and the element conversions of the cache.
#pragma once

#include <cuda_fp8.h>
#include <stdarg.h>
#include <stdio.h>

#include "../../include/rmsnorm_tp_b200.h"
#include "device_common.cuh"
#include "internal.h"

namespace rtp {

// Records a formatted message as the calling thread's last error, returns `code`.
inline int refuse(int code, const char* fmt, ...) {
  char buf[384];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return record_error(code, buf);
}

// Makes `device` current for the scope (the tensors' device need not be the
// caller's current one), restoring the caller's device after.
struct OnDevice {
  int prev = -1;
  bool switched = false;
  cudaError_t err;
  explicit OnDevice(int device) {
    err = cudaGetDevice(&prev);
    if (err == cudaSuccess && prev != device) {
      err = cudaSetDevice(device);
      switched = err == cudaSuccess;
    }
  }
  ~OnDevice() {
    if (switched) cudaSetDevice(prev);
  }
};

// SM count of `device` (cached), 0 on failure.
int sm_count(int device);

// Launch with programmatic stream serialization when dependent launch is on.
// Every kernel launched through here starts with grid_dep_wait().
// cluster > 0: in clusters of so many CTAs.
cudaError_t launch_dependent(const void* fn, dim3 grid, dim3 block, size_t smem, void** args,
                             cudaStream_t stream, int cluster = 0);

inline int launch_failed(cudaError_t e, const char* who) {
  cudaGetLastError();   // a refused launch leaves the error behind otherwise
  return refuse(RMSNORM_TP_ERR_CUDA, "%s: kernel launch: %s (%s)", who, cudaGetErrorString(e),
                cudaGetErrorName(e));
}

// Checks the cache a call is given; 0 or a recorded error.
int check_cache(const char* who, const rmsnorm_kv_cache* c);

// Extent of a [tokens, heads, dim] view whose last stride is 1.
struct View {
  uintptr_t base;
  int64_t n0, n1, dim, s0, s1;   // elements
  int eb;
  uintptr_t bytes() const {      // from the first element to behind the last
    if (n0 == 0 || n1 == 0) return 0;
    return (uintptr_t)(((n0 - 1) * s0 + (n1 - 1) * s1 + dim) * eb);
  }
};
inline View view_of(const void* p, int64_t tokens, int64_t heads, int64_t dim, const int64_t* st,
                    int eb) {
  // a stride of an axis of one entry says nothing: leave it out
  return View{reinterpret_cast<uintptr_t>(p), tokens, heads, dim, tokens > 1 ? st[0] : heads * dim,
              heads > 1 ? st[1] : dim, eb};
}

// `bytes` bytes in one piece.
inline View span_of(const void* p, uint64_t bytes) {
  const int64_t n = (int64_t)bytes;
  return View{reinterpret_cast<uintptr_t>(p), n > 0, 1, n, n, n, 1};
}

// Whether b's rows lie between a's, both views' rows being multiples of `stride` apart.
inline bool rows_between(const View& a, const View& b, int64_t stride) {
  const int64_t step = stride * a.eb;
  int64_t d = (int64_t)(b.base - a.base) % step;
  if (d < 0) d += step;
  return d >= a.dim * a.eb && d + b.dim * b.eb <= step;
}

// Whether two views may share an element. Exact for column blocks of one matrix
// (the same token stride) and for heads that lie between one another's (q, k and v of a head
// side by side: the same head stride, of which the token stride is a multiple, or the other
// way round), else by their extents.
inline bool views_overlap(const View& a, const View& b) {
  const uintptr_t an = a.bytes(), bn = b.bytes();
  if (an == 0 || bn == 0) return false;
  if (!(a.base < b.base + bn && b.base < a.base + an)) return false;
  if (a.n0 > 1 && b.n0 > 1 && a.s0 == b.s0 && a.s0 > 0 && a.eb == b.eb) {
    const int64_t step = a.s0 * a.eb;
    const int64_t ra = ((a.n1 - 1) * a.s1 + a.dim) * a.eb, rb = ((b.n1 - 1) * b.s1 + b.dim) * b.eb;
    int64_t d = ((int64_t)(b.base - a.base)) % step;
    if (d < 0) d += step;
    if (ra <= step && rb <= step && d >= ra && d + rb <= step) return false;
  }
  if (a.eb == b.eb) {
    const bool heads = a.n1 > 1 && b.n1 > 1 && a.s1 == b.s1, tokens = a.n0 > 1 && b.n0 > 1 && a.s0 == b.s0;
    const auto whole = [](int64_t n, int64_t stride, int64_t of) { return n <= 1 || stride % of == 0; };
    if (heads && a.s1 > 0 && whole(a.n0, a.s0, a.s1) && whole(b.n0, b.s0, a.s1) && rows_between(a, b, a.s1)) return false;
    if (tokens && a.s0 > 0 && whole(a.n1, a.s1, a.s0) && whole(b.n1, b.s1, a.s0) && rows_between(a, b, a.s0)) return false;
  }
  return true;
}
inline bool views_same(const View& a, const View& b) {
  return a.base == b.base && a.s0 == b.s0 && a.s1 == b.s1 && a.eb == b.eb;
}
// Whether a written view's own rows are apart.
inline bool view_apart(const View& a) {
  const bool heads_inside = a.s1 >= a.dim && a.s0 >= (a.n1 - 1) * a.s1 + a.dim;
  const bool tokens_inside = a.s0 >= a.dim && a.s1 >= (a.n0 - 1) * a.s0 + a.dim;
  return heads_inside || tokens_inside;
}

// threadIdx.x as a value made after this point: addresses formed with it cannot be loaded
// before a preceding grid_dep_wait, read-only loads among them.
__device__ __forceinline__ int thread_here() {
  int t = threadIdx.x;
  asm volatile("" : "+r"(t));
  return t;
}

// ---- asynchronous copies into shared memory (16 bytes a thread) -----------------
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// With `live` false nothing is read and zeros are written.
__device__ __forceinline__ void cp_async16_if(uint32_t dst, const void* src, bool live) {
  const int n = live ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async4_if(uint32_t dst, const void* src, bool live) {
  const int n = live ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Waits until at most N of this thread's groups are under way.
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Division of 32-bit numbers under 2^31 by a number that the host knows, by the multiplier
// rounded up (Granlund and Montgomery, Division by Invariant Integers using Multiplication,
// 1994): n / by = (umulhi(n, mul) + n) >> shift, with mul = floor(2^32 (2^shift - by) / by) + 1.
struct FastDiv {
  unsigned by, mul, shift;
  static FastDiv of(unsigned by) {
    unsigned shift = 0;   // ceil(log2(by))
    while ((1ull << shift) < by) ++shift;
    return FastDiv{by, (unsigned)(((1ull << 32) * ((1ull << shift) - by)) / by + 1), shift};
  }
  __device__ __forceinline__ unsigned quotient(unsigned n) const { return (__umulhi(n, mul) + n) >> shift; }
};

// Page and offset of a slot; 32-bit division where the cache's slots allow it.
__device__ __forceinline__ void page_of(int64_t slot, int page, int64_t num_slots, int64_t& pg, int& off) {
  if (num_slots <= 0xFFFFFFFFll) {
    const unsigned p = (unsigned)slot / (unsigned)page;
    pg = p;
    off = (int)((unsigned)slot - p * (unsigned)page);
  } else {
    pg = slot / page;
    off = (int)(slot - pg * page);
  }
}

// ---- cache elements -----------------------------------------------------------
constexpr float kE4M3Max = 448.f;
// Smallest row maximum a scale is made of (2^-100): keeps 448 / maximum finite
// and the scale a normal number, also for a row of zeros.
constexpr float kE4M3Floor = 7.8886090522101181e-31f;

__device__ __forceinline__ unsigned short e4m3x2_of(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ unsigned char e4m3_of(float v) {
  return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float2 e4m3x2_to(unsigned short c) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(c, __NV_E4M3);
  return __half22float2(__half2(h));
}
__device__ __forceinline__ float e4m3_to(unsigned char c) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw(c, __NV_E4M3);
  return __half2float(__half(h));
}

}  // namespace rtp
