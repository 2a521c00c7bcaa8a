// What the operators around the expert products share (tokens.cu, swiglu.cu,
// w4.cu): element types, wide loads and stores, and the host-side checks.
#pragma once

#include <cuda_fp16.h>

#include "kernels.cuh"

namespace moe {

// Defined in api.cu: MOE_OK when the current device is an sm_100 one, and its
// number of SMs; and the status of a CUDA call, kept for
// moe_fp8_ds_last_cuda_error_string.
int require_device(int* sm_count);
int cuda_status(cudaError_t e);

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float(float v) { return v; }
template <> __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// One rounding to the nearest value of T.
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float(float v) { return v; }
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }

// Two values rounded to T, the first in the low half.
template <typename T> __device__ __forceinline__ uint32_t two_of(float a, float b);
template <> __device__ __forceinline__ uint32_t two_of<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return reinterpret_cast<const uint32_t&>(v);
}
template <> __device__ __forceinline__ uint32_t two_of<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return reinterpret_cast<const uint32_t&>(v);
}

// N elements that are moved by as few accesses as their size allows.
template <typename T, int N>
struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Pack {
  T v[N];
};

template <int BYTES> struct Word;
template <> struct Word<1> { using type = uint8_t; };
template <> struct Word<2> { using type = uint16_t; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<16> { using type = uint4; };

// Loads and stores of data that is used once: no reuse is asked of the caches.
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_stream(const T* p) {
  constexpr int kBytes = N * sizeof(T), kWord = kBytes < 16 ? kBytes : 16;
  using W = typename Word<kWord>::type;
  Pack<T, N> out;
#pragma unroll
  for (int i = 0; i < kBytes / kWord; ++i)
    reinterpret_cast<W*>(&out)[i] = __ldcs(reinterpret_cast<const W*>(p) + i);
  return out;
}
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_cached(const T* p) {
  constexpr int kBytes = N * sizeof(T), kWord = kBytes < 16 ? kBytes : 16;
  using W = typename Word<kWord>::type;
  Pack<T, N> out;
#pragma unroll
  for (int i = 0; i < kBytes / kWord; ++i)
    reinterpret_cast<W*>(&out)[i] = *(reinterpret_cast<const W*>(p) + i);
  return out;
}
template <typename T, int N>
__device__ __forceinline__ void store_wide(T* p, const Pack<T, N>& x) {
  constexpr int kBytes = N * sizeof(T), kWord = kBytes < 16 ? kBytes : 16;
  using W = typename Word<kWord>::type;
#pragma unroll
  for (int i = 0; i < kBytes / kWord; ++i)
    *(reinterpret_cast<W*>(p) + i) = reinterpret_cast<const W*>(&x)[i];
}
template <> __device__ __forceinline__ uint8_t from_float(float v) { return (uint8_t)v; }   // for zeros
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> zero_pack() {
  Pack<T, N> z;
#pragma unroll
  for (int i = 0; i < N; ++i) z.v[i] = from_float<T>(0.f);
  return z;
}

// Asynchronous 16-byte copies to shared memory that bypass the L1 cache.
__device__ __forceinline__ void copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

inline int dtype_bytes(int t) { return t == MOE_F32 ? 4 : t == MOE_F16 || t == MOE_BF16 ? 2 : 0; }

// The widest access of at most `most` elements of `bytes` each (a power of
// two) that divides rows of `width` elements and the alignment of every
// pointer.
inline int vector_elements(int64_t width, int bytes, int most, std::initializer_list<const void*> ptrs) {
  int n = most;
  auto fits = [&](int k) {
    if (width % k) return false;
    for (const void* p : ptrs)
      if (p && reinterpret_cast<uintptr_t>(p) % (uintptr_t)(k * bytes < 16 ? k * bytes : 16)) return false;
    return true;
  };
  while (n > 1 && !fits(n)) n >>= 1;
  return n;
}

inline bool aligned_to(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes == 0; }

}  // namespace moe
