// SwiGLU between the two expert products, y = up * gate * sigmoid(gate) for rows
// x = [up | gate] (the order of W13's halves), with its input kept for the
// backward pass in 8 bits: every 1x128 block of up and of gate (blocks start at
// each half's first column, the last may be shorter) becomes e4m3 codes
//   s = amax / 448 (1 when that is 0),  q = e4m3(x / s),  both in fp32,
// the layer's activation format.  The backward pass computes from q * s:
//   grad_up   = g * gate * sig
//   grad_gate = g * up * sig * (1 + gate * (1 - sig))
// A block that holds an infinity or a NaN is kept as NaN.
//
// Both passes are bound by memory: 2 + 1 elements (forward, nothing kept), 2 + 1
// elements + 2 bytes (forward), 1 + 2 elements + 2 bytes (backward) for each
// column, so the kept codes cost the backward pass half of the reads that kept
// 16-bit inputs would.
#include <type_traits>

#include "rows.cuh"

namespace moe {
namespace {

constexpr int kLanes = 16;                       // threads of one 1x128 block
constexpr int kElems = kBlock / kLanes;          // 8 columns a thread
constexpr int kThreads = 256;
constexpr int kRowsAtOnce = kThreads / kLanes;   // rows of a CTA in one step

// sigmoid in fp32, 1 / (1 + exp(-v)), down to the least fp32 number: from v = -88 on exp(-v) leaves fp32, while
// up * v * sigmoid(v) is a number that bf16 and fp32 hold.  16-bit outputs keep 11 bits at most, so they take the
// hardware's approximations of 2^x and 1 / d, with t = exp(-v / 2) and the sum 2^24 times smaller, which nothing
// overflows where the result is not 0: 2^-24 / (2^-24 + 2^-24 t t).  It is off by less than 5 + 1.173 |v|
// units of 2^-23.  fp32 outputs get the full exp and division; below -kFar their sigmoid is exp(v) itself (FAR:
// a block's gates may be there).
constexpr float kFar = 80.f;
template <typename T, bool FAR>
__device__ __forceinline__ float sigmoid(float v) {
  if constexpr (sizeof(T) == 2) {
    float t, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(v * -0.72134752f));   // log2(e) / 2
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(t * 0x1p-24f, t, 0x1p-24f)));
    return r * 0x1p-24f;
  }
  if (FAR && v < -kFar) return expf(v);
  return 1.f / (1.f + expf(-v));
}

// A thread's 8 columns of a block, as 8 / N accesses of N elements: access j
// covers columns (j * 16 + lane) * N ..., so neighbours read neighbours.  They stay
// as they came until they are worked on, so that several rows' loads fit the
// registers.
template <typename T, int N>
struct Piece {
  Pack<T, N> v[kElems / N];
};

template <int N>
__device__ __forceinline__ int column(int j, int lane) { return (j * kLanes + lane) * N; }

template <typename T, int N>
__device__ __forceinline__ void load_piece(const T* p, int lane, int width, Piece<T, N>& x) {
#pragma unroll
  for (int j = 0; j < kElems / N; ++j) {
    const int c = column<N>(j, lane);
    if (c < width) x.v[j] = load_stream<T, N>(p + c);   // width is a multiple of N
    else x.v[j] = zero_pack<T, N>();
  }
}
template <typename T, int N>
__device__ __forceinline__ void to_floats(const Piece<T, N>& x, float (&v)[kElems]) {
#pragma unroll
  for (int j = 0; j < kElems / N; ++j)
#pragma unroll
    for (int i = 0; i < N; ++i) v[j * N + i] = to_float(x.v[j].v[i]);
}
template <typename T, int N>
__device__ __forceinline__ void store_piece(T* p, int lane, int width, const float (&v)[kElems]) {
#pragma unroll
  for (int j = 0; j < kElems / N; ++j) {
    const int c = column<N>(j, lane);
    if (c >= width) continue;
    Pack<T, N> x;
    if constexpr (sizeof(T) == 2 && N >= 2) {    // two at a time: one instruction
#pragma unroll
      for (int i = 0; i < N; i += 2)
        reinterpret_cast<uint32_t*>(&x)[i / 2] = two_of<T>(v[j * N + i], v[j * N + i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) x.v[i] = from_float<T>(v[j * N + i]);
    }
    store_wide<T, N>(p + c, x);
  }
}

// Bits of the largest magnitude among a thread's columns (as fp32): a NaN's are above an
// infinity's.  16-bit columns are compared two at a time.
template <typename T> __device__ __forceinline__ uint32_t max_abs2(uint32_t a, uint32_t b);   // signs are of no use
template <> __device__ __forceinline__ uint32_t max_abs2<__nv_bfloat16>(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
template <> __device__ __forceinline__ uint32_t max_abs2<__half>(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
template <typename T, int N>
__device__ __forceinline__ uint32_t largest(const Piece<T, N>& x, const float (&v)[kElems]) {
  uint32_t bits = 0;
  if constexpr (sizeof(T) == 2 && N >= 2) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&x);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kElems / 2; ++i) m = max_abs2<T>(m, w[i]);
    m &= 0x7fff7fffu;
    const Pack<T, 2> two = reinterpret_cast<const Pack<T, 2>&>(m);
    bits = max(__float_as_uint(to_float(two.v[0])), __float_as_uint(to_float(two.v[1])));
  } else {
#pragma unroll
    for (int i = 0; i < kElems; ++i) bits = max(bits, __float_as_uint(v[i]) & 0x7fffffffu);
  }
  return bits;
}

// v / s, correctly rounded, by Markstein's theorem (IBM Journal of Research and
// Development 34, 1990): with r the correctly rounded 1 / s and q within a unit in the
// last place of v / s, q + (v - q s) r rounds to the correctly rounded quotient, as long
// as nothing leaves the range of normal numbers.  Written as q - (q s - v) r it keeps a
// zero's sign, as the division does: q s - v is +0 there, and q - 0 is q.  PLAIN is the
// division itself, for scales near the ends of the range.  (32768 x 4096 bf16: 152 us with divisions.)
template <bool PLAIN>
__device__ __forceinline__ float2 quotients(float2 v, float s, float r) {
  if (PLAIN) return make_float2(__fdiv_rn(v.x, s), __fdiv_rn(v.y, s));
  const float2 q = __fmul2_rn(v, make_float2(r, r));
  const float2 over = __ffma2_rn(q, make_float2(s, s), make_float2(-v.x, -v.y));
  return __ffma2_rn(over, make_float2(-r, -r), q);
}

template <int N, bool PLAIN>
__device__ __forceinline__ void store_codes(uint8_t* q, int lane, int width, const float (&v)[kElems], float s, float r) {
  auto two = [&](int i) {
    return (uint32_t)__nv_cvt_float2_to_fp8x2(quotients<PLAIN>(make_float2(v[i], v[i + 1]), s, r), __NV_SATFINITE, __NV_E4M3);
  };
#pragma unroll
  for (int j = 0; j < kElems / N; ++j) {
    const int c = column<N>(j, lane);
    if (c >= width) continue;
    if constexpr (N == 8) *reinterpret_cast<uint2*>(q + c) = make_uint2(two(0) | two(2) << 16, two(4) | two(6) << 16);
    else if constexpr (N == 4) *reinterpret_cast<uint32_t*>(q + c) = two(4 * j) | two(4 * j + 2) << 16;
    else if constexpr (N == 2) *reinterpret_cast<uint16_t*>(q + c) = (uint16_t)two(2 * j);
    else q[c] = f32_to_e4m3(quotients<PLAIN>(make_float2(v[j], 0.f), s, r).x);
  }
}

// Codes of a block and its scale (the same in all 16 lanes); `bits` becomes the largest magnitude's.
template <typename T, int N>
__device__ __forceinline__ float keep_block(uint8_t* q, int lane, int width, const Piece<T, N>& x, const float (&v)[kElems],
                                            uint32_t& bits) {
  bits = largest<T, N>(x, v);
#pragma unroll
  for (int off = kLanes / 2; off; off >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, off));
  float s = __fdiv_rn(__uint_as_float(bits), kFp8Max);
  if (s == 0.f) s = 1.f;
  if (bits >= 0x7f800000u) s = __int_as_float(0x7fc00000);
  if (s > 0x1p-90f && s < 0x1p90f) store_codes<N, false>(q, lane, width, v, s, __frcp_rn(s));
  else store_codes<N, true>(q, lane, width, v, s, 0.f);
  return s;
}

// Codes to the values that they stand for.
template <int N>
__device__ __forceinline__ void kept_values(const Piece<uint8_t, N>& q, float s, float (&v)[kElems]) {
#pragma unroll
  for (int j = 0; j < kElems / N; ++j) {
    if constexpr (N == 1) {
      v[j] = e4m3_to_f32(q.v[j].v[0]) * s;
    } else {
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const __nv_fp8x2_storage_t two = reinterpret_cast<const __nv_fp8x2_storage_t*>(&q.v[j])[i / 2];
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3);
        const float2 f = __half22float2(__half2(h));
        v[j * N + i] = f.x * s;
        v[j * N + i + 1] = f.y * s;
      }
    }
  }
}

// A CTA takes block `b` of U * 16 rows, so the scales of a block (stored by
// block, [2 * blocks][R]) are written as whole lines; neighbouring CTAs take
// neighbouring blocks.  U rows are in flight in each thread.
template <typename T, int N, int U, bool KEEP>
__global__ void __launch_bounds__(kThreads, 5)   // 32768 x 4096 fp16: 63 us, unbounded 66
swiglu_kernel(const T* __restrict__ x, int R, int I, int blocks, T* __restrict__ y, uint8_t* __restrict__ q,
              float* __restrict__ scale) {
  griddep_wait();
  griddep_launch_dependents();
  const int tile = (int)blockIdx.x / blocks, b = (int)blockIdx.x - tile * blocks;
  const int lane = (int)threadIdx.x % kLanes;
  const int64_t row0 = (int64_t)tile * (U * kRowsAtOnce) + threadIdx.x / kLanes;
  const int col = b * kBlock, width = I - col < kBlock ? I - col : kBlock;
  Piece<T, N> up_in[U], gate_in[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t r = row0 + u * kRowsAtOnce;
    const T* p = x + (size_t)r * 2 * I + col;
    const int w = r < R ? width : 0;
    load_piece<T, N>(p, lane, w, up_in[u]);
    load_piece<T, N>(p + I, lane, w, gate_in[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t r = row0 + u * kRowsAtOnce;
    const int w = r < R ? width : 0;
    float up[kElems], gate[kElems], out[kElems];
    to_floats<T, N>(up_in[u], up);
    to_floats<T, N>(gate_in[u], gate);
    uint32_t bits = 0;                             // of the block's largest gate
    if constexpr (KEEP) {
      uint8_t* p = q + (size_t)r * 2 * I + col;
      const float su = keep_block<T, N>(p, lane, w, up_in[u], up, bits), sg = keep_block<T, N>(p + I, lane, w, gate_in[u], gate, bits);
      if (lane == 0 && r < R) {
        scale[(size_t)b * R + r] = su;
        scale[(size_t)(blocks + b) * R + r] = sg;
      }
    }
    bool far = false;                              // a thread's gates, or the block's where they were compared
    if constexpr (sizeof(T) == 4) {
      far = bits > __float_as_uint(kFar);
#pragma unroll
      for (int i = 0; i < kElems; ++i) far |= !KEEP && gate[i] < -kFar;
    }
    if (!far) {
#pragma unroll
      for (int i = 0; i < kElems; ++i) out[i] = gate[i] * sigmoid<T, false>(gate[i]) * up[i];
    } else {
#pragma unroll
      for (int i = 0; i < kElems; ++i) out[i] = gate[i] * sigmoid<T, true>(gate[i]) * up[i];
    }
    store_piece<T, N>(y + (size_t)r * I + col, lane, w, out);
  }
}

template <typename T, int N, int U>
__global__ void __launch_bounds__(kThreads)
swiglu_backward_kernel(const T* __restrict__ g, const uint8_t* __restrict__ q, const float* __restrict__ scale,
                       int R, int I, int blocks, T* __restrict__ grad_x) {
  griddep_wait();
  griddep_launch_dependents();
  const int tile = (int)blockIdx.x / blocks, b = (int)blockIdx.x - tile * blocks;
  const int lane = (int)threadIdx.x % kLanes;
  const int64_t row0 = (int64_t)tile * (U * kRowsAtOnce) + threadIdx.x / kLanes;
  const int col = b * kBlock, width = I - col < kBlock ? I - col : kBlock;
  Piece<T, N> dy_in[U];
  Piece<uint8_t, N> up_in[U], gate_in[U];
  float su[U], sg[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t r = row0 + u * kRowsAtOnce;
    const int w = r < R ? width : 0;
    const uint8_t* p = q + (size_t)r * 2 * I + col;
    su[u] = r < R ? __ldg(scale + (size_t)b * R + r) : 0.f;
    sg[u] = r < R ? __ldg(scale + (size_t)(blocks + b) * R + r) : 0.f;
    load_piece<uint8_t, N>(p, lane, w, up_in[u]);
    load_piece<uint8_t, N>(p + I, lane, w, gate_in[u]);
    load_piece<T, N>(g + (size_t)r * I + col, lane, w, dy_in[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t r = row0 + u * kRowsAtOnce;
    const int w = r < R ? width : 0;
    float up[kElems], gate[kElems], dy[kElems], du[kElems], dg[kElems];
    kept_values<N>(up_in[u], su[u], up);
    kept_values<N>(gate_in[u], sg[u], gate);
    to_floats<T, N>(dy_in[u], dy);
    auto gradients = [&](auto far) {
#pragma unroll
      for (int i = 0; i < kElems; ++i) {
        const float sig = sigmoid<T, decltype(far)::value>(gate[i]), gs = dy[i] * sig;
        du[i] = gs * gate[i];
        dg[i] = gs * up[i] * (1.f + gate[i] * (1.f - sig));
      }
    };
    if (sizeof(T) == 2 || sg[u] < kFar / kFp8Max) gradients(std::false_type{});   // the block's largest gate is 448 times its scale
    else gradients(std::true_type{});
    T* p = grad_x + (size_t)r * 2 * I + col;
    store_piece<T, N>(p, lane, w, du);
    store_piece<T, N>(p + I, lane, w, dg);
  }
}

// ---------------------------------------------------------------- host side
struct SwigluGrid {
  int blocks;
  int64_t ctas;
};
SwigluGrid swiglu_grid(int R, int I, int U) {
  const int blocks = (I + kBlock - 1) / kBlock;
  return {blocks, ((int64_t)R + U * kRowsAtOnce - 1) / (U * kRowsAtOnce) * blocks};
}

template <typename T, int N, int U>
int run_forward_u(const void* x, int R, int I, void* y, void* q, float* scale, cudaStream_t s) {
  const SwigluGrid g = swiglu_grid(R, I, U);
  if (g.ctas > INT32_MAX) return MOE_ERR_TOO_LARGE;
  auto kern = q ? swiglu_kernel<T, N, U, true> : swiglu_kernel<T, N, U, false>;
  return cuda_status(launch_pdl(kern, dim3((unsigned)g.ctas), dim3(kThreads), 0, s, static_cast<const T*>(x), R, I,
                                g.blocks, static_cast<T*>(y), static_cast<uint8_t*>(q), scale));
}
template <typename T, int N, int U>
int run_backward_u(const void* dy, const void* q, const float* scale, int R, int I, void* dx, cudaStream_t s) {
  const SwigluGrid g = swiglu_grid(R, I, U);
  if (g.ctas > INT32_MAX) return MOE_ERR_TOO_LARGE;
  return cuda_status(launch_pdl(swiglu_backward_kernel<T, N, U>, dim3((unsigned)g.ctas), dim3(kThreads), 0, s,
                                static_cast<const T*>(dy), static_cast<const uint8_t*>(q), scale, R, I, g.blocks,
                                static_cast<T*>(dx)));
}

// Rows in flight in a thread: two where that still makes 8 CTAs for each SM and a thread's accesses
// are of 16 bytes, or in the forward passes of 4 columns.  (us for the forward pass / the one that keeps codes / the
// backward pass, two rows and one: 32768 x 4096 bf16 62 / 111 / 94 and 73 / 117 / 100, fp16 63 / 109 / 103 and 67 /
// 115 / 99; 16384 x 4096 fp32 61 / 81 / 73 and 60 / 81 / 83, 16384 x 2004 fp32 30 / 50 / 44 and 30 / 46 / 43; 512 x 4096 bf16 4.5 / 4.6 / 4.6 either way; four
// columns at a time, 32768 x 2008 bf16, 35 / 62 / 53 and 37 / 63 / 51; single ones, 32768 x 2002 bf16, 43 / 100 / 86
// and 45 / 84 / 71.)
constexpr int kFlight = 2;
bool many_rows(int R, int I) { return swiglu_grid(R, I, kFlight).ctas >= 148 * 8; }

template <typename T, int N>
int run_forward(const void* x, int R, int I, void* y, void* q, float* scale, cudaStream_t s) {
  if constexpr (N >= 4)
    if (many_rows(R, I)) return run_forward_u<T, N, kFlight>(x, R, I, y, q, scale, s);
  return run_forward_u<T, N, 1>(x, R, I, y, q, scale, s);
}
template <typename T, int N>
int run_backward(const void* dy, const void* q, const float* scale, int R, int I, void* dx, cudaStream_t s) {
  if constexpr (N * sizeof(T) >= 16)
    if (many_rows(R, I)) return run_backward_u<T, N, kFlight>(dy, q, scale, R, I, dx, s);
  return run_backward_u<T, N, 1>(dy, q, scale, R, I, dx, s);
}

// Columns a thread moves at a time: 16 bytes where the rows and halves allow it.
template <typename T>
int forward_typed(const void* x, int R, int I, void* y, void* q, float* scale, cudaStream_t s) {
  constexpr int kMost = 16 / (int)sizeof(T);
  int n = vector_elements(I, sizeof(T), kMost, {x, y});
  n = vector_elements(I, 1, n, {q});
  switch (n) {
    case 8: if constexpr (kMost >= 8) return run_forward<T, 8>(x, R, I, y, q, scale, s);
    case 4: return run_forward<T, 4>(x, R, I, y, q, scale, s);
    case 2: return run_forward<T, 2>(x, R, I, y, q, scale, s);
    default: return run_forward<T, 1>(x, R, I, y, q, scale, s);
  }
}
template <typename T>
int backward_typed(const void* dy, const void* q, const float* scale, int R, int I, void* dx, cudaStream_t s) {
  constexpr int kMost = 16 / (int)sizeof(T);
  int n = vector_elements(I, sizeof(T), kMost, {dy, dx});
  n = vector_elements(I, 1, n, {q});
  switch (n) {
    case 8: if constexpr (kMost >= 8) return run_backward<T, 8>(dy, q, scale, R, I, dx, s);
    case 4: return run_backward<T, 4>(dy, q, scale, R, I, dx, s);
    case 2: return run_backward<T, 2>(dy, q, scale, R, I, dx, s);
    default: return run_backward<T, 1>(dy, q, scale, R, I, dx, s);
  }
}

int check_swiglu(int32_t R, int32_t I, int32_t dtype) {
  if (R < 0 || I < 1 || !dtype_bytes(dtype)) return MOE_ERR_INVALID_ARGUMENT;
  return I > INT32_MAX / 2 ? MOE_ERR_TOO_LARGE : MOE_OK;
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

MOE_API int moe_swiglu_forward(const void* x, int32_t num_rows, int32_t inter, int32_t dtype, void* y, void* codes,
                               float* scales, void* stream) {
  int st = check_swiglu(num_rows, inter, dtype);
  if (st != MOE_OK) return st;
  if (num_rows == 0) return MOE_OK;
  if (!x || !y || !codes != !scales) return MOE_ERR_INVALID_ARGUMENT;
  if (!aligned_to(x, dtype_bytes(dtype)) || !aligned_to(y, dtype_bytes(dtype)) || !aligned_to(scales, 4))
    return MOE_ERR_MISALIGNED;
  if ((st = require_device(nullptr)) != MOE_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == MOE_BF16) return forward_typed<__nv_bfloat16>(x, num_rows, inter, y, codes, scales, s);
  if (dtype == MOE_F16) return forward_typed<__half>(x, num_rows, inter, y, codes, scales, s);
  return forward_typed<float>(x, num_rows, inter, y, codes, scales, s);
}

MOE_API int moe_swiglu_backward(const void* grad_y, const void* codes, const float* scales, int32_t num_rows,
                                int32_t inter, int32_t dtype, void* grad_x, void* stream) {
  int st = check_swiglu(num_rows, inter, dtype);
  if (st != MOE_OK) return st;
  if (num_rows == 0) return MOE_OK;
  if (!grad_y || !codes || !scales || !grad_x) return MOE_ERR_INVALID_ARGUMENT;
  if (!aligned_to(grad_y, dtype_bytes(dtype)) || !aligned_to(grad_x, dtype_bytes(dtype)) || !aligned_to(scales, 4))
    return MOE_ERR_MISALIGNED;
  if ((st = require_device(nullptr)) != MOE_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == MOE_BF16) return backward_typed<__nv_bfloat16>(grad_y, codes, scales, num_rows, inter, grad_x, s);
  if (dtype == MOE_F16) return backward_typed<__half>(grad_y, codes, scales, num_rows, inter, grad_x, s);
  return backward_typed<float>(grad_y, codes, scales, num_rows, inter, grad_x, s);
}

}  // extern "C"
