// Products of few rows with 4-bit weights: for expert e, its rows x[r] and the
// matrix of codes q[e] (N x D, one scale and possibly one zero point for each
// group of G columns)
//   y[r, n] = sum over groups g of scale[e,n,g] * sum_{k in g} (q[e,n,k] - zero[e,n,g]) * x[r,k].
//
// The weights of the experts that have rows are read once, and reading them
// bounds the product up to about 16 rows an expert (4 bits a weight against
// 2 * rows operations).  Rows are few, so weights are on the M side of
// mma.sync m16n8k16 (tcgen05 would need the decoded weights in shared memory or
// TMEM, eight times the bytes that are read, to multiply tiles of mostly
// missing rows): codes go from memory to registers, become the exact 16-bit
// values q - zero there, and multiply up to 8 rows of x at a time.  A group's
// sum is made in fp32 and scaled in fp32, so nothing is rounded before the output.
//
// Layout (made once, by the caller): 16 x 64 tiles of codes in the order in
// which a warp's lanes take them, 16 bytes a lane.  With lane = 4 * g + t, 32-bit
// word j holds columns c = 32 * (j / 2) + 8 * t + 4 * (j % 2) + {0, 1, 2, 3} of
// rows g and g + 8: nibbles 0, 4 = (g; c, c + 1), 1, 5 = (g + 8; c, c + 1), 2, 6 =
// (g; c + 2, c + 3), 3, 7 = (g + 8; c + 2, c + 3), so that (word >> 4i) & 0x000f000f
// is the i-th A register of step j, and a lane's B registers are 16 consecutive
// bytes of x.  Scales are [E][N / 16][groups][8][2] (rows g, g + 8 together), zero
// points likewise.
#include "rows.cuh"

namespace moe {
namespace {

constexpr int kW4Threads = 256;
constexpr int kW4Warps = kW4Threads / 32;
constexpr int kMaxRows = 32;              // rows of x in one unit of work
constexpr int kMaxExperts = 1024;
constexpr int kTileK = 64;                // columns of a tile
constexpr int kUnitTiles = 4;             // 16-row tiles of a unit
constexpr int kSumFloats = 1152;          // a warp's sums: 16 rows x 68 or 32 rows x 36, padded

struct W4Params {
  const void* x;
  const uint4* codes;      // [E][n_tiles][k_tiles][32]
  const uint32_t* scales;  // [E][n_tiles][groups][8] pairs of 16-bit scales
  const uint16_t* zeros;   // [E][n_tiles][groups][8] pairs of 8-bit zero points, or null
  const int32_t* offsets;  // [E + 1], or null: one matrix for all rows
  void* y;
  int R, N, D, E, n_tiles, k_tiles, groups, group_shift;
  int out_f32, zero_rest;
};

template <typename T> struct Half2;
template <> struct Half2<__nv_bfloat16> {
  static constexpr uint32_t kBase = 0x43004300u;   // 128, 128: the last mantissa bits count ones
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  static __device__ __forceinline__ float2 scales(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <> struct Half2<__half> {
  static constexpr uint32_t kBase = 0x64006400u;   // 1024, 1024
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  static __device__ __forceinline__ float2 scales(uint32_t v) {
    return __half22float2(*reinterpret_cast<__half2*>(&v));
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

__device__ __forceinline__ uint4 load_codes(const uint4* p) {   // read once
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// One warp's part of a unit: MT tiles of 16 weight rows times NT * 8 rows of x
// over the tiles [k0, k1) of columns; sums[mt][nt] are the mma's C registers.
template <typename T, int NT, int MT, bool SMALL, bool ZEROS>
__device__ __forceinline__ void warp_product(const W4Params& p, int e, int m0, int r0, int cnt, int k0, int k1,
                                             float (&sums)[MT][NT][4]) {
  using H = Half2<T>;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const size_t tile0 = (size_t)e * p.n_tiles + m0;
  const uint4* codes = p.codes + tile0 * p.k_tiles * 32 + lane;
  const uint32_t* scales = p.scales + tile0 * p.groups * 8 + g;
  const uint16_t* zeros = ZEROS ? p.zeros + tile0 * p.groups * 8 + g : nullptr;
  const int m_here = p.n_tiles - m0 < MT ? p.n_tiles - m0 : MT;
  const uint4* x[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
    x[nt] = nt * 8 + g < cnt
                ? reinterpret_cast<const uint4*>(static_cast<const T*>(p.x) + (size_t)(r0 + nt * 8 + g) * p.D) + t
                : nullptr;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) sums[mt][nt][i] = 0.f;
  uint4 next[MT];
  auto fetch = [&](int k) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
      if (mt < m_here) next[mt] = load_codes(codes + ((size_t)mt * p.k_tiles + k) * 32);
  };
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) next[mt] = make_uint4(0, 0, 0, 0);
  if (k0 < k1) fetch(k0);
#pragma unroll 1
  for (int k = k0; k < k1; ++k) {
    uint32_t word[MT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      word[mt][0] = next[mt].x; word[mt][1] = next[mt].y; word[mt][2] = next[mt].z; word[mt][3] = next[mt].w;
    }
    if (k + 1 < k1) fetch(k + 1);
    uint4 b[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        b[nt][h] = x[nt] && k * kTileK + 32 * h < p.D ? __ldg(x[nt] + k * 8 + h * 4) : make_uint4(0, 0, 0, 0);
    constexpr int kParts = SMALL ? 2 : 1;       // groups of 32 columns: two in a tile
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
      const int group = (k * kTileK + part * 32) >> p.group_shift;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        if (mt >= m_here) continue;
        const size_t at = ((size_t)mt * p.groups + group) * 8;
        const float2 s = H::scales(__ldg(scales + at));
        uint32_t z0 = H::kBase | 0x00080008u, z1 = z0;
        if (ZEROS) {
          const uint32_t z = __ldg(zeros + at);
          z0 = H::kBase | (z & 0xff) * 0x00010001u;
          z1 = H::kBase | (z >> 8) * 0x00010001u;
        }
        float c[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) c[nt][i] = 0.f;
#pragma unroll
        for (int j = part * 2; j < (SMALL ? part * 2 + 2 : 4); ++j) {
          uint32_t a[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            a[i] = H::sub(((word[mt][j] >> (4 * i)) & 0x000f000fu) | H::kBase, (i & 1) ? z1 : z0);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint4 v = b[nt][j >> 1];
            H::mma(c[nt], a, (j & 1) ? v.z : v.x, (j & 1) ? v.w : v.y);
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) sums[mt][nt][i] = fmaf(i < 2 ? s.x : s.y, c[nt][i], sums[mt][nt][i]);
      }
    }
  }
}

// A unit: kUnitN weight rows of expert e from row n0, rows [r0, r0 + cnt) of x.
// The warps split the columns; their sums meet in shared memory and are added in
// warp order.
template <typename T, int NT, int MT, bool SMALL, bool ZEROS>
__device__ __forceinline__ void run_unit(const W4Params& p, int e, int m0, int m1, int r0, int cnt, float* s_out) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int k0 = (int)((int64_t)p.k_tiles * warp / kW4Warps), k1 = (int)((int64_t)p.k_tiles * (warp + 1) / kW4Warps);
  constexpr int kStride = MT * 16 + 4;   // of the sums in shared memory: a warp's stores hit 32 banks
  static_assert(NT * 8 * kStride <= kSumFloats, "sums of a unit");
  for (int m = m0; m < m1; m += MT) {
    float sums[MT][NT][4];
    warp_product<T, NT, MT, SMALL, ZEROS>(p, e, m, r0, cnt, k0, k1, sums);
    float* mine = s_out + (size_t)warp * kSumFloats;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          mine[(nt * 8 + 2 * t + (i & 1)) * kStride + mt * 16 + g + 8 * (i >> 1)] = sums[mt][nt][i];
    __syncthreads();
    for (int o = threadIdx.x; o < cnt * MT * 16; o += kW4Threads) {
      const int row = o / (MT * 16), n = o % (MT * 16), col = m * 16 + n;
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kW4Warps; ++w) v += s_out[w * kSumFloats + row * kStride + n];
      if (col >= p.N) continue;
      const size_t at = (size_t)(r0 + row) * p.N + col;
      if (p.out_f32) static_cast<float*>(p.y)[at] = v;
      else static_cast<T*>(p.y)[at] = from_float<T>(v);
    }
    __syncthreads();
  }
}

template <typename T, bool SMALL, bool ZEROS>
__global__ void __launch_bounds__(kW4Threads, 2) w4_kernel(const W4Params p) {
  __shared__ float s_out[kW4Warps * kSumFloats];
  __shared__ int s_units[kMaxExperts + 1];
  griddep_wait();
  griddep_launch_dependents();
  const int blocks = (p.n_tiles + kUnitTiles - 1) / kUnitTiles;
  auto rows_of = [&](int e, int* first) {      // whatever the offsets say, within [0, R]
    if (!p.offsets) { *first = 0; return p.R; }
    int a = __ldg(p.offsets + e), b = __ldg(p.offsets + e + 1);
    a = a < 0 ? 0 : a > p.R ? p.R : a;
    b = b < a ? a : b > p.R ? p.R : b;
    *first = a;
    return b - a;
  };
  // Units of work of the experts before e: the same in every CTA.
  for (int e = threadIdx.x; e < p.E; e += kW4Threads) {
    int first;
    s_units[e] = (rows_of(e, &first) + kMaxRows - 1) / kMaxRows;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    int sum = 0;
    const int lane = threadIdx.x;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int e = e0 + lane, v = e < p.E ? s_units[e] : 0;
      int incl = v;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += o;
      }
      if (e < p.E) s_units[e] = sum + incl - v;
      sum += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) s_units[p.E] = sum;
  }
  __syncthreads();
  // Unit u: chunk of rows c, block of weight rows; a chunk's blocks follow one another.
  const int64_t units = (int64_t)s_units[p.E] * blocks;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int c = (int)(u / blocks), m0 = (int)(u - (int64_t)c * blocks) * kUnitTiles;
    int lo = 0, hi = p.E;                      // the expert e with s_units[e] <= c < s_units[e + 1]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_units[mid] <= c) lo = mid; else hi = mid;
    }
    int first;
    const int rows = rows_of(lo, &first), chunks = (rows + kMaxRows - 1) / kMaxRows, i = c - s_units[lo];
    const int a = (int)((int64_t)rows * i / chunks), cnt = (int)((int64_t)rows * (i + 1) / chunks) - a;
    const int m1 = m0 + kUnitTiles < p.n_tiles ? m0 + kUnitTiles : p.n_tiles;
    if (cnt <= 8) run_unit<T, 1, 4, SMALL, ZEROS>(p, lo, m0, m1, first + a, cnt, s_out);
    else if (cnt <= 16) run_unit<T, 2, 4, SMALL, ZEROS>(p, lo, m0, m1, first + a, cnt, s_out);
    else run_unit<T, 4, 2, SMALL, ZEROS>(p, lo, m0, m1, first + a, cnt, s_out);
  }
  if (p.zero_rest && p.offsets) {              // rows of no expert
    int a = __ldg(p.offsets), b = __ldg(p.offsets + p.E);
    a = a < 0 ? 0 : a > p.R ? p.R : a;
    b = b < a ? a : b > p.R ? p.R : b;
    const int64_t rest = (int64_t)(p.R - (b - a)) * p.N;
    for (int64_t i = (int64_t)blockIdx.x * kW4Threads + threadIdx.x; i < rest; i += (int64_t)gridDim.x * kW4Threads) {
      int64_t r = i / p.N;
      const int64_t n = i - r * p.N;
      if (r >= a) r += b - a;
      if (p.out_f32) static_cast<float*>(p.y)[r * p.N + n] = 0.f;
      else static_cast<T*>(p.y)[r * p.N + n] = from_float<T>(0.f);
    }
  }
}

template <typename T>
int run_w4(const W4Params& p, bool small, int sms, cudaStream_t s) {
  auto kern = small ? (p.zeros ? w4_kernel<T, true, true> : w4_kernel<T, true, false>)
                    : (p.zeros ? w4_kernel<T, false, true> : w4_kernel<T, false, false>);
  return cuda_status(launch_pdl(kern, dim3(2 * sms), dim3(kW4Threads), 0, s, p));
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

MOE_API int moe_w4_matvec(const void* x, const void* codes, const void* scales, const void* zeros,
                          const int32_t* offsets, int32_t num_rows, int32_t num_experts, int32_t n, int32_t d,
                          int32_t group_size, int32_t dtype, int32_t out_dtype, int32_t zero_other_rows, void* y,
                          void* stream) {
  if (num_rows < 0 || num_experts < 1 || n < 1 || d < 1) return MOE_ERR_INVALID_ARGUMENT;
  if (group_size != 32 && group_size != 64 && group_size != 128) return MOE_ERR_INVALID_ARGUMENT;
  if (d % group_size || (!offsets && num_experts != 1)) return MOE_ERR_INVALID_ARGUMENT;
  if ((dtype != MOE_F16 && dtype != MOE_BF16) || (out_dtype != dtype && out_dtype != MOE_F32))
    return MOE_ERR_INVALID_ARGUMENT;
  if (num_experts > kMaxExperts || n > INT32_MAX - 64 || d > INT32_MAX - 64) return MOE_ERR_TOO_LARGE;
  if (num_rows == 0) return MOE_OK;
  if (!x || !codes || !scales || !y) return MOE_ERR_INVALID_ARGUMENT;
  if (!aligned_to(x, 16) || !aligned_to(codes, 16) || !aligned_to(scales, 4) || !aligned_to(zeros, 2) ||
      !aligned_to(offsets, 4) || !aligned_to(y, dtype_bytes(out_dtype)))
    return MOE_ERR_MISALIGNED;
  int sms = 0;
  const int st = require_device(&sms);
  if (st != MOE_OK) return st;
  W4Params p;
  p.x = x;
  p.codes = static_cast<const uint4*>(codes);
  p.scales = static_cast<const uint32_t*>(scales);
  p.zeros = static_cast<const uint16_t*>(zeros);
  p.offsets = offsets;
  p.y = y;
  p.R = num_rows; p.N = n; p.D = d; p.E = num_experts;
  p.n_tiles = (n + 15) / 16;
  p.k_tiles = (d + kTileK - 1) / kTileK;
  p.groups = group_size == 32 ? 2 * p.k_tiles : d / group_size;   // whole tiles
  p.group_shift = group_size == 32 ? 5 : group_size == 64 ? 6 : 7;
  p.out_f32 = out_dtype == MOE_F32;
  p.zero_rest = zero_other_rows != 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == MOE_BF16 ? run_w4<__nv_bfloat16>(p, group_size == 32, sms, s)
                           : run_w4<__half>(p, group_size == 32, sms, s);
}

}  // extern "C"
