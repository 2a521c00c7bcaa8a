// Products of few rows with 4-bit weights: for expert e, its rows x[r] and the
// matrix of codes q[e] (N x D, one scale and possibly one zero point for each
// group of G columns)
//   y[r, n] = sum over groups g of scale[e,n,g] * sum_{k in g} (q[e,n,k] - zero[e,n,g]) * x[r,k].
//
// The codes of the experts that have rows are read once, and reading them should
// bound the product, so the work on each code has to be small.  It is with fp16
// operands (mma.sync m16n8k16, fp32 sums, weights on the M side): the number 0..15 in
// the low bits of an fp16 is exactly q * 2^-24 (below 2^-14 fp16 is evenly
// spaced), four bits higher it is 16 * q * 2^-24, so a 32-bit word of eight codes
// becomes four operand registers by four masks, one shift and four subtractions of
// the zero point, all exact.  The factors 2^24 and 1/16 go into the scales and the
// last step; a group's sum is scaled in fp32, and only the output is rounded.
// (e4m3 operands, where a byte 0..15 is q * 2^-9, need half the masks, but mma.sync
// with e4m3 is converted to fp16 here: measured four times the instructions.
// tcgen05 would want the decoded weights in shared memory or TMEM and 128-row tiles; a
// decode batch has too few rows of x for that to pay.)
//
// fp16 rows of x are the other operand as they are.  bf16 rows are first brought
// to fp16 by a power of two for each row that puts its largest magnitude into
// [2^14, 2^15): exact for values down to 2^-28 of the largest, below that off by at
// most 2^-39 of it.  (Next to an infinity or a NaN the finite values vanish, as they
// do in the sum.)
//
// Layout (made once, by the caller): 16 x 64 tiles of codes in the order in
// which a warp's lanes take them, 16 bytes a lane.  With lane = 4 * g + t, 32-bit
// word j holds columns c = 32 * (j / 2) + 8 * t + 4 * (j % 2) + {0, 2, 1, 3} in its
// bytes 0 to 3, row g in the low half of a byte and row g + 8 in the high half: a
// lane's share of x is then 16 consecutive bytes for each 32 columns.  Scales are
// [E][N / 16][groups][8][2] (rows g, g + 8 together), zero points likewise.
#include "rows.cuh"

namespace moe {
namespace {

constexpr int kWarps = 8;                 // of a CTA; they split the columns
constexpr int kThreads = kWarps * 32;
constexpr int kCtasPerSm = 2;
constexpr int kM = 4;                     // 16-row tiles of weights in a task
constexpr int kMaxRows = 16;              // rows of x in a task
constexpr int kStages = 4;                // of a warp's ring of tiles
constexpr int kTileK = 64;                // columns of a tile
constexpr int kMaxExperts = 1024;
constexpr int kSumM = 2;                  // rows of tiles whose sums are joined at a time
constexpr int kSumStride = kSumM * 16 + 4;   // of the sums in shared memory: a warp's stores hit 32 banks

struct W4Params {
  const __half* x;         // [R, D]
  const int32_t* row_exp;  // [R]: the exponent taken out of a bf16 row, or null: 0
  const uint4* codes;      // [E][n_tiles][k_tiles][32]
  const uint32_t* scales;  // [E][n_tiles][groups][8] pairs of 16-bit scales
  const uint32_t* zeros;   // [E][n_tiles][groups][4] pairs of pairs of 8-bit zero points, or null
  const int32_t* offsets;  // [E + 1], or null: one matrix for all rows
  void* y;
  int R, N, D, E, n_tiles, k_tiles, groups, group_shift;
  int out_f32, zero_rest;
};

// --------------------------------------------------------------------------
// bf16 rows to fp16: a CTA takes a row, finds its largest magnitude and scales by
// 2^-exp.  Reads and writes R * D * 2 bytes, a few microseconds of latency.
// --------------------------------------------------------------------------
constexpr int kConvertThreads = 256;

__global__ void __launch_bounds__(kConvertThreads)
w4_convert_kernel(const __nv_bfloat16* __restrict__ x, int D, __half* __restrict__ out, int32_t* __restrict__ row_exp) {
  __shared__ float s_max[kConvertThreads / 32];
  griddep_wait();
  griddep_launch_dependents();
  const size_t base = (size_t)blockIdx.x * D;
  float amax = 0.f;
  for (int i = threadIdx.x * 8; i < D; i += kConvertThreads * 8) {   // D is a multiple of 32
    const Pack<__nv_bfloat16, 8> v = load_cached<__nv_bfloat16, 8>(x + base + i);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float a = fabsf(to_float(v.v[j]));
      amax = a < INFINITY ? fmaxf(amax, a) : INFINITY;
    }
  }
#pragma unroll
  for (int off = 16; off; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = amax;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kConvertThreads / 32; ++i) amax = fmaxf(amax, s_max[i]);
  // amax * 2^-exp in [2^14, 2^15), as far as 2^-exp is a normal number
  int exp = (int)((__float_as_uint(amax) >> 23) & 0xff) - 127 - 14;
  exp = exp < -120 ? -120 : exp;
  const float down = __uint_as_float((uint32_t)(127 - exp) << 23);
  for (int i = threadIdx.x * 8; i < D; i += kConvertThreads * 8) {
    const Pack<__nv_bfloat16, 8> v = load_cached<__nv_bfloat16, 8>(x + base + i);
    Pack<__half, 8> h;
#pragma unroll
    for (int j = 0; j < 8; ++j) h.v[j] = __float2half_rn(to_float(v.v[j]) * down);
    store_wide<__half, 8>(out + base + i, h);
  }
  if (threadIdx.x == 0) row_exp[blockIdx.x] = exp;
}

// --------------------------------------------------------------------------
// The product.
// --------------------------------------------------------------------------
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t sub_f16x2(uint32_t a, uint32_t b) {   // subnormal numbers included
  uint32_t d;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// Asynchronous copies to shared memory.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <typename T> __device__ __forceinline__ float2 pair_of(uint32_t v);
template <> __device__ __forceinline__ float2 pair_of<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 pair_of<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<__half2*>(&v));
}

// One step of a warp's ring: a tile of each of kM rows of tiles, their scales and
// zero points.
template <bool SMALL, bool ZEROS>
struct Stage {
  static constexpr int kParts = SMALL ? 2 : 1;   // groups in a tile
  uint4 codes[kM][32];
  uint32_t scales[kParts][kM][8];
  uint32_t zeros[ZEROS ? kParts : 1][kM][4];
};

// A task: tiles [m0, m0 + m) of rows of expert e's matrix, times rows [r0, r0 + cnt) of x.
struct Task {
  int e, m0, m, r0, cnt;
};

// Start the copies of tile k of a task.
template <bool SMALL, bool ZEROS>
__device__ __forceinline__ void fill(const W4Params& p, const Task& w, int k, Stage<SMALL, ZEROS>* st) {
  const int lane = threadIdx.x & 31;
  const size_t tile0 = (size_t)w.e * p.n_tiles + w.m0;
  const uint4* codes = p.codes + (tile0 * p.k_tiles + k) * 32 + lane;
#pragma unroll
  for (int m = 0; m < kM; ++m)
    if (m < w.m) copy16(smem_u32(&st->codes[m][lane]), codes + (size_t)m * p.k_tiles * 32);
#pragma unroll
  for (int part = 0; part < Stage<SMALL, ZEROS>::kParts; ++part) {
    const int group = (k * kTileK + part * 32) >> p.group_shift;
    const int m = lane >> 3, g = lane & 7;
    if (m < w.m) copy4(smem_u32(&st->scales[part][m][g]), p.scales + ((tile0 + m) * p.groups + group) * 8 + g);
    if (ZEROS) {
      const int mz = (lane >> 2) & 3, gz = lane & 3;
      if (lane < 16 && mz < w.m)
        copy4(smem_u32(&st->zeros[part][mz][gz]), p.zeros + ((tile0 + mz) * p.groups + group) * 4 + gz);
    }
  }
}

// A lane's share of a tile's columns of x: rows nt * 8 + g of the task, columns 8 t .. + 7 of each 32.
template <int NT>
__device__ __forceinline__ void load_x(const W4Params& p, const __half* const (&rows)[NT], int k, uint4 (&x)[NT][2]) {
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int col = k * kTileK + h * 32;
      x[nt][h] = rows[nt] && col < p.D ? __ldg(reinterpret_cast<const uint4*>(rows[nt] + col)) : make_uint4(0, 0, 0, 0);
    }
}

template <typename T, int NT, bool SMALL, bool ZEROS>
__device__ __forceinline__ void multiply(const Stage<SMALL, ZEROS>* st, int m_here, const uint4 (&x)[NT][2],
                                         float (&sums)[kM][NT][4]) {
  const int lane = threadIdx.x & 31, g = lane >> 2;
#pragma unroll
  for (int m = 0; m < kM; ++m) {
    if (m >= m_here) break;
    const uint4 c = st->codes[m][lane];
    const uint32_t word[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int part = 0; part < Stage<SMALL, ZEROS>::kParts; ++part) {
      uint32_t z0 = 0x00080008u, z1 = 0x00800080u;   // zero points, row g + 8's times 16 as its codes are
      if (ZEROS) {
        const uint32_t z = st->zeros[part][m][g >> 1] >> (16 * (g & 1));
        z0 = (z & 0xff) * 0x00010001u;
        z1 = (z >> 8 & 0xff) * 0x00100010u;
      }
      float a[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) a[nt][i] = 0.f;
#pragma unroll
      for (int j = 2 * part; j < (SMALL ? 2 * part + 2 : 4); ++j) {
        const uint32_t w = word[j], w8 = w >> 8;
        const uint32_t a0 = sub_f16x2(w & 0x000f000fu, z0), a1 = sub_f16x2(w & 0x00f000f0u, z1);
        const uint32_t a2 = sub_f16x2(w8 & 0x000f000fu, z0), a3 = sub_f16x2(w8 & 0x00f000f0u, z1);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const uint4 v = x[nt][j >> 1];
          mma_f16(a[nt], a0, a1, a2, a3, (j & 1) ? v.z : v.x, (j & 1) ? v.w : v.y);
        }
      }
      float2 s = pair_of<T>(st->scales[part][m][g]);
      s.y *= 0.0625f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {      // rows g and g + 8; two rows of x in each fma
          const float2 sum = __ffma2_rn(make_float2(a[nt][2 * h], a[nt][2 * h + 1]),
                                        h ? make_float2(s.y, s.y) : make_float2(s.x, s.x),
                                        make_float2(sums[m][nt][2 * h], sums[m][nt][2 * h + 1]));
          sums[m][nt][2 * h] = sum.x;
          sums[m][nt][2 * h + 1] = sum.y;
        }
    }
  }
}

template <bool SMALL, bool ZEROS>
constexpr size_t kRingBytes = sizeof(Stage<SMALL, ZEROS>) * kStages * kWarps;
constexpr size_t kSumBytes = sizeof(float) * kWarps * kMaxRows * kSumStride;

template <typename T, bool SMALL, bool ZEROS>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) w4_kernel(const W4Params p) {
  using St = Stage<SMALL, ZEROS>;
  extern __shared__ __align__(16) uint8_t s_mem[];
  __shared__ int s_chunks[kMaxExperts + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  St* ring = reinterpret_cast<St*>(s_mem) + warp * kStages;
  float* s_sums = reinterpret_cast<float*>(s_mem + kRingBytes<SMALL, ZEROS>);

  auto rows_of = [&](int e, int* first) {      // whatever the offsets say, within [0, R]
    if (!p.offsets) { *first = 0; return p.R; }
    int a = __ldg(p.offsets + e), b = __ldg(p.offsets + e + 1);
    a = a < 0 ? 0 : a > p.R ? p.R : a;
    b = b < a ? a : b > p.R ? p.R : b;
    *first = a;
    return b - a;
  };
  // Chunks of up to 16 rows before expert e: the same in every CTA.
  for (int e = threadIdx.x; e < p.E; e += kThreads) {
    int first;
    s_chunks[e] = (rows_of(e, &first) + kMaxRows - 1) / kMaxRows;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    int sum = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int e = e0 + lane, v = e < p.E ? s_chunks[e] : 0;
      int incl = v;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += o;
      }
      if (e < p.E) s_chunks[e] = sum + incl - v;
      sum += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) s_chunks[p.E] = sum;
  }
  __syncthreads();
  // The (chunk, row of tiles) pairs are dealt out evenly: CTA b takes [first, last).
  const int64_t total = (int64_t)s_chunks[p.E] * p.n_tiles;
  const int64_t first = total * blockIdx.x / gridDim.x, last = total * (blockIdx.x + 1) / gridDim.x;
  auto task_at = [&](int64_t at) {
    Task w;
    const int c = (int)(at / p.n_tiles);
    w.m0 = (int)(at - (int64_t)c * p.n_tiles);
    int lo = 0, hi = p.E;                      // the expert e with s_chunks[e] <= c < s_chunks[e + 1]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_chunks[mid] <= c) lo = mid; else hi = mid;
    }
    w.e = lo;
    int64_t left = last - at;
    if (left > p.n_tiles - w.m0) left = p.n_tiles - w.m0;
    const int steps = (int)((left + kM - 1) / kM);
    w.m = (int)((left + steps - 1) / steps);   // even tasks
    int r;
    const int rows = rows_of(lo, &r), chunks = (rows + kMaxRows - 1) / kMaxRows, i = c - s_chunks[lo];
    const int a = (int)((int64_t)rows * i / chunks);
    w.r0 = r + a;
    w.cnt = (int)((int64_t)rows * (i + 1) / chunks) - a;
    return w;
  };
  const int k0 = (int)((int64_t)p.k_tiles * warp / kWarps), k1 = (int)((int64_t)p.k_tiles * (warp + 1) / kWarps);

  griddep_wait();                              // x is there
  griddep_launch_dependents();
  // The copies run kStages - 1 steps ahead of the products, across tasks.
  int64_t ahead_at = first;
  int ahead_k = k0, ahead_slot = 0;
  Task ahead;
  if (first < last) ahead = task_at(first);
  auto advance = [&]() {
    if (ahead_at < last && k0 < k1) {
      fill(p, ahead, ahead_k, ring + ahead_slot);
      if (++ahead_k == k1) {
        ahead_k = k0;
        ahead_at += ahead.m;
        if (ahead_at < last) ahead = task_at(ahead_at);
      }
    }
    ahead_slot = ahead_slot + 1 == kStages ? 0 : ahead_slot + 1;
    copies_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) advance();
  int slot = 0;
  auto run = [&](const Task& w, auto nt_tag) {
    constexpr int NT = decltype(nt_tag)::value;
    float sums[kM][NT][4];
#pragma unroll
    for (int m = 0; m < kM; ++m)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[m][nt][i] = 0.f;
    const int g = lane >> 2, t = lane & 3;
    const __half* rows[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
      rows[nt] = nt * 8 + g < w.cnt ? p.x + (size_t)(w.r0 + nt * 8 + g) * p.D + 8 * t : nullptr;
    uint4 x[NT][2], next[NT][2];
    load_x<NT>(p, rows, k0, next);
#pragma unroll 1
    for (int k = k0; k < k1; ++k) {
      __syncwarp();                            // the slot that is filled next has been read by all lanes
      advance();
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) { x[nt][0] = next[nt][0]; x[nt][1] = next[nt][1]; }
      if (k + 1 < k1) load_x<NT>(p, rows, k + 1, next);
      copies_wait<kStages - 1>();
      __syncwarp();
      multiply<T, NT, SMALL, ZEROS>(ring + slot, w.m, x, sums);
      slot = slot + 1 == kStages ? 0 : slot + 1;
    }
    // The warps' sums meet in shared memory and are added in warp order.
    float* mine = s_sums + warp * (kMaxRows * kSumStride);
#pragma unroll
    for (int m1 = 0; m1 < kM; m1 += kSumM) {
      if (m1 >= w.m) break;
#pragma unroll
      for (int m = 0; m < kSumM; ++m)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            mine[(nt * 8 + 2 * t + (i & 1)) * kSumStride + m * 16 + g + 8 * (i >> 1)] = sums[m1 + m][nt][i];
      __syncthreads();
      const int width = (w.m - m1) * 16;
      for (int o = threadIdx.x; o < w.cnt * kSumM * 16; o += kThreads) {
        const int row = o / (kSumM * 16), n = o % (kSumM * 16), col = (w.m0 + m1) * 16 + n;
        if (n >= width || col >= p.N) continue;
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < kWarps; ++q) v += s_sums[(q * kMaxRows + row) * kSumStride + n];
        v = ldexpf(v, 24 + (p.row_exp ? __ldg(p.row_exp + w.r0 + row) : 0));
        const size_t at = (size_t)(w.r0 + row) * p.N + col;
        if (p.out_f32) static_cast<float*>(p.y)[at] = v;
        else static_cast<T*>(p.y)[at] = from_float<T>(v);
      }
      __syncthreads();
    }
  };
  for (int64_t at = first; at < last;) {
    const Task w = task_at(at);
    if (w.cnt <= 8) run(w, std::integral_constant<int, 1>{});
    else run(w, std::integral_constant<int, 2>{});
    at += w.m;
  }
  copies_wait<0>();
  if (p.zero_rest && p.offsets) {              // rows of no expert
    int a = __ldg(p.offsets), b = __ldg(p.offsets + p.E);
    a = a < 0 ? 0 : a > p.R ? p.R : a;
    b = b < a ? a : b > p.R ? p.R : b;
    const int64_t rest = (int64_t)(p.R - (b - a)) * p.N;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < rest; i += (int64_t)gridDim.x * kThreads) {
      int64_t r = i / p.N;
      const int64_t n = i - r * p.N;
      if (r >= a) r += b - a;
      if (p.out_f32) static_cast<float*>(p.y)[r * p.N + n] = 0.f;
      else static_cast<T*>(p.y)[r * p.N + n] = from_float<T>(0.f);
    }
  }
}

// Workspace of a bf16 call: the rows in fp16, then their exponents.
uint64_t rows_bytes(int64_t R, int64_t d) { return ((uint64_t)R * d * 2 + 255) & ~uint64_t(255); }

template <typename T, bool SMALL, bool ZEROS>
int launch_w4(const W4Params& p, const void* x, int sms, cudaStream_t s) {
  constexpr size_t kSmem = kRingBytes<SMALL, ZEROS> + kSumBytes;
  static_assert((kSmem + 4 * (kMaxExperts + 4) + 1024) * kCtasPerSm <= 227 * 1024, "shared memory of the resident CTAs");
  static std::atomic<void*> seen[kMaxCachedDevices];
  cudaError_t e = once_per_context(seen, [] {
    return cudaFuncSetAttribute(w4_kernel<T, SMALL, ZEROS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem);
  });
  if (e != cudaSuccess) return cuda_status(e);
  if (p.row_exp) {
    e = launch_pdl(w4_convert_kernel, dim3(p.R), dim3(kConvertThreads), 0, s, static_cast<const __nv_bfloat16*>(x),
                   p.D, const_cast<__half*>(p.x), const_cast<int32_t*>(p.row_exp));
    if (e != cudaSuccess) return cuda_status(e);
  }
  return cuda_status(launch_pdl(w4_kernel<T, SMALL, ZEROS>, dim3(kCtasPerSm * sms), dim3(kThreads), kSmem, s, p));
}

template <typename T>
int run_w4(const W4Params& p, const void* x, bool small, int sms, cudaStream_t s) {
  if (small) return p.zeros ? launch_w4<T, true, true>(p, x, sms, s) : launch_w4<T, true, false>(p, x, sms, s);
  return p.zeros ? launch_w4<T, false, true>(p, x, sms, s) : launch_w4<T, false, false>(p, x, sms, s);
}

int check_w4(int32_t R, int32_t d, int32_t group_size, int32_t dtype) {
  if (R < 0 || d < 1 || (group_size != 32 && group_size != 64 && group_size != 128) || d % group_size)
    return MOE_ERR_INVALID_ARGUMENT;
  if (dtype != MOE_F16 && dtype != MOE_BF16) return MOE_ERR_INVALID_ARGUMENT;
  return d > INT32_MAX - 64 ? MOE_ERR_TOO_LARGE : MOE_OK;
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

MOE_API int moe_w4_workspace_size(int32_t num_rows, int32_t d, int32_t group_size, int32_t dtype, uint64_t* bytes) {
  const int st = check_w4(num_rows, d, group_size, dtype);
  if (st != MOE_OK) return st;
  if (!bytes) return MOE_ERR_INVALID_ARGUMENT;
  *bytes = dtype == MOE_BF16 ? rows_bytes(num_rows, d) + (uint64_t)num_rows * sizeof(int32_t) : 0;
  return MOE_OK;
}

MOE_API int moe_w4_matvec(const void* x, const void* codes, const void* scales, const void* zeros,
                          const int32_t* offsets, int32_t num_rows, int32_t num_experts, int32_t n, int32_t d,
                          int32_t group_size, int32_t dtype, int32_t out_dtype, int32_t zero_other_rows, void* y,
                          void* workspace, uint64_t workspace_bytes, void* stream) {
  int st = check_w4(num_rows, d, group_size, dtype);
  if (st != MOE_OK) return st;
  if (num_experts < 1 || n < 1 || (!offsets && num_experts != 1)) return MOE_ERR_INVALID_ARGUMENT;
  if (out_dtype != dtype && out_dtype != MOE_F32) return MOE_ERR_INVALID_ARGUMENT;
  if (num_experts > kMaxExperts || n > INT32_MAX - 64) return MOE_ERR_TOO_LARGE;
  if (num_rows == 0) return MOE_OK;
  if (!x || !codes || !scales || !y) return MOE_ERR_INVALID_ARGUMENT;
  if (!aligned_to(x, 16) || !aligned_to(codes, 16) || !aligned_to(scales, 4) || !aligned_to(zeros, 4) ||
      !aligned_to(offsets, 4) || !aligned_to(y, dtype_bytes(out_dtype)) || !aligned_to(workspace, 256))
    return MOE_ERR_MISALIGNED;
  uint64_t need = 0;
  moe_w4_workspace_size(num_rows, d, group_size, dtype, &need);
  if (workspace_bytes < need || (need && !workspace)) return MOE_ERR_WORKSPACE_TOO_SMALL;
  int sms = 0;
  if ((st = require_device(&sms)) != MOE_OK) return st;
  W4Params p;
  p.R = num_rows; p.N = n; p.D = d; p.E = num_experts;
  p.n_tiles = (n + 15) / 16;
  p.k_tiles = (d + kTileK - 1) / kTileK;
  p.groups = group_size == 32 ? 2 * p.k_tiles : d / group_size;   // whole tiles
  p.group_shift = group_size == 32 ? 5 : group_size == 64 ? 6 : 7;
  p.x = static_cast<const __half*>(dtype == MOE_BF16 ? workspace : x);
  p.row_exp = dtype == MOE_BF16 ? reinterpret_cast<const int32_t*>(static_cast<const uint8_t*>(workspace) +
                                                                   rows_bytes(num_rows, d))
                                : nullptr;
  p.codes = static_cast<const uint4*>(codes);
  p.scales = static_cast<const uint32_t*>(scales);
  p.zeros = static_cast<const uint32_t*>(zeros);
  p.offsets = offsets;
  p.y = y;
  p.out_f32 = out_dtype == MOE_F32;
  p.zero_rest = zero_other_rows != 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == MOE_BF16 ? run_w4<__nv_bfloat16>(p, x, group_size == 32, sms, s)
                           : run_w4<__half>(p, x, group_size == 32, sms, s);
}

}  // extern "C"
