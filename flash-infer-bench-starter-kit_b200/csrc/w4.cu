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
// Layout (made once, by moe_w4_lay_out): records of 16 rows x 128 columns,
// [E][N / 16][D / 128][record], each one piece of memory that a warp streams:
//   two 16 x 64 tiles of codes in the order in which a warp's lanes take them, 16
//   bytes a lane.  With lane = 4 * g + t, 32-bit word j holds columns c = 32 * (j / 2) +
//   8 * t + 4 * (j % 2) + {0, 2, 1, 3} in its bytes 0 to 3, row g in the low half of a
//   byte and row g + 8 in the high half: a lane's share of x is then 16 consecutive
//   bytes for each 32 columns;
//   the record's scales [128 / G][8][2] (rows g, g + 8 together), then, if there are any,
//   its zero points likewise.
#include "rows.cuh"

namespace moe {
namespace {

constexpr int kWarps = 8;                 // of a CTA
constexpr int kThreads = kWarps * 32;
constexpr int kCtasPerSm = 2;
constexpr int kM = 4;                     // rows of records a warp works on together
constexpr int kMaxRows = 16;              // rows of x in a task
constexpr int kStages = 2;                // of a warp's ring of records
constexpr int kStepK = 128;               // columns of a record
constexpr int kMaxExperts = 1024;
constexpr int kSumM = 2;                  // rows of records whose sums are joined at a time
constexpr int kSumStride = kSumM * 16 + 4;   // of the sums in shared memory: a warp's stores hit 32 banks
constexpr size_t kSumBytes = sizeof(float) * kWarps * kMaxRows * kSumStride;

// Bytes of a record with groups of G columns.
__host__ __device__ constexpr int record_bytes(int G, bool zeros) { return 1024 + kStepK / G * (zeros ? 48 : 32); }

struct W4Params {
  const __half* x;         // [R, D]
  const int32_t* row_exp;  // [R]: the exponent taken out of a bf16 row, or null: 0
  const uint8_t* records;  // [E][n_tiles][k_steps][record]
  const int32_t* offsets;  // [E + 1], or null: one matrix for all rows
  void* y;
  int R, N, D, E, n_tiles, k_steps, k_split;
  int out_f32, zero_rest;
};

// --------------------------------------------------------------------------
// The layout: a thread makes 16 bytes.  Padding (rows behind N, columns behind D) is
// zero.
// --------------------------------------------------------------------------
__global__ void __launch_bounds__(256)
w4_lay_out_kernel(const uint8_t* __restrict__ codes, const uint16_t* __restrict__ scales,
                  const uint8_t* __restrict__ zeros, int N, int D, int G, int n_tiles, int k_steps, int64_t pieces,
                  uint8_t* __restrict__ out) {
  griddep_wait();
  griddep_launch_dependents();
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= pieces) return;
  const int groups = kStepK / G, per_record = record_bytes(G, zeros != nullptr) / 16;
  const int64_t record = at / per_record, tile = record / k_steps;
  const int piece = (int)(at - record * per_record), step = (int)(record - tile * k_steps);
  const int64_t e = tile / n_tiles;
  const int row0 = (int)(tile - e * n_tiles) * 16;
  union { uint4 v; uint8_t b[16]; uint16_t h[8]; } o;
  o.v = make_uint4(0, 0, 0, 0);
  if (piece < 64) {
    const int lane = piece & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int col = step * kStepK + (piece >> 5) * 64 + 32 * h + 8 * t;   // D is a multiple of 32
      uint32_t v[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = row0 + g + 8 * i;
        if (row < N && col < D)
          v[i] = *reinterpret_cast<const uint32_t*>(codes + ((size_t)e * N + row) * (D / 2) + col / 2);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {        // columns 4 j .. 4 j + 3 of the 8: two bytes of each row
        const uint32_t a0 = v[0] >> (16 * j) & 0xff, a1 = v[0] >> (16 * j + 8) & 0xff;
        const uint32_t b0 = v[1] >> (16 * j) & 0xff, b1 = v[1] >> (16 * j + 8) & 0xff;
        uint8_t* w = o.b + 8 * h + 4 * j;
        w[0] = (uint8_t)((a0 & 15) | (b0 & 15) << 4);
        w[1] = (uint8_t)((a1 & 15) | (b1 & 15) << 4);
        w[2] = (uint8_t)(a0 >> 4 | (b0 & 0xf0));
        w[3] = (uint8_t)(a1 >> 4 | (b1 & 0xf0));
      }
    }
  } else {
    const int tail = piece - 64;
    const bool is_zeros = tail >= 2 * groups;
    const int n = is_zeros ? 16 : 8, first = (is_zeros ? tail - 2 * groups : tail) * n;   // of the [groups][8][2] values
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (i >= n) break;
      const int v = first + i, group = step * groups + v / 16, row = row0 + (v & 15) / 2 + 8 * (v & 1);
      if (row >= N || group * G >= D) continue;
      const size_t src = ((size_t)e * N + row) * (D / G) + group;
      if (is_zeros) o.b[i] = zeros[src];
      else o.h[i] = scales[src];
    }
  }
  *reinterpret_cast<uint4*>(out + at * 16) = o.v;
}

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

// Tiles [m0, m0 + m) of rows of expert e's matrix, times rows [r0, r0 + cnt) of x: what a
// CTA does at a time.  `c` numbers the chunks of rows of x over all experts.
struct Task {
  int c, e, m0, m, r0, cnt;
};

// A step: kM records of 128 columns (`m_here` of them are there) times NT * 8 rows of x,
// half a record at a time so that the next half's x can be on its way.
template <typename T, int NT, int G, bool ZEROS>
struct Step {
  static constexpr int kRecord = record_bytes(G, ZEROS);
  static constexpr int kGroups = G == 32 ? 2 : 1;        // in half a record

  // A lane's share of half a record's columns of x.
  static __device__ __forceinline__ void load_x(const __half* const (&rows)[NT], int col, int D, uint4 (&x)[NT][2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool in = col + 32 * h < D;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        x[nt][h] = in ? __ldg(reinterpret_cast<const uint4*>(rows[nt] + col + 32 * h)) : make_uint4(0, 0, 0, 0);
    }
  }

  static __device__ __forceinline__ void multiply(const uint8_t* stage, int half, int m_here, const uint4 (&x)[NT][2],
                                                  float (&sums)[kM][NT][4]) {
    const int lane = threadIdx.x & 31, g = lane >> 2;
#pragma unroll
    for (int m = 0; m < kM; ++m) {
      if (m >= m_here) break;
      const uint8_t* rec = stage + m * kRecord;
      const uint4 c = *reinterpret_cast<const uint4*>(rec + half * 512 + lane * 16);
      const uint32_t word[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
      for (int part = 0; part < kGroups; ++part) {
        const int group = (half * 64 + part * 32) / G;
        uint32_t z0 = 0x00080008u, z1 = 0x00800080u;   // zero points, row g + 8's times 16 as its codes are
        if (ZEROS) {
          const uint32_t z = *reinterpret_cast<const uint16_t*>(rec + 1024 + kStepK / G * 32 + group * 16 + g * 2);
          z0 = (z & 0xff) * 0x00010001u;
          z1 = (z >> 8) * 0x00100010u;
        }
        float a[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) a[nt][i] = 0.f;
#pragma unroll
        for (int j = 2 * part; j < (G == 32 ? 2 * part + 2 : 4); ++j) {
          const uint32_t w = word[j], w8 = w >> 8;
          const uint32_t a0 = sub_f16x2(w & 0x000f000fu, z0), a1 = sub_f16x2(w & 0x00f000f0u, z1);
          const uint32_t a2 = sub_f16x2(w8 & 0x000f000fu, z0), a3 = sub_f16x2(w8 & 0x00f000f0u, z1);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint4 v = x[nt][j >> 1];
            mma_f16(a[nt], a0, a1, a2, a3, (j & 1) ? v.z : v.x, (j & 1) ? v.w : v.y);
          }
        }
        float2 s = pair_of<T>(*reinterpret_cast<const uint32_t*>(rec + 1024 + group * 32 + g * 4));
        s.y *= 0.0625f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {    // rows g and g + 8; two rows of x in each fma
            const float2 sum = __ffma2_rn(make_float2(a[nt][2 * h], a[nt][2 * h + 1]),
                                          h ? make_float2(s.y, s.y) : make_float2(s.x, s.x),
                                          make_float2(sums[m][nt][2 * h], sums[m][nt][2 * h + 1]));
            sums[m][nt][2 * h] = sum.x;
            sums[m][nt][2 * h + 1] = sum.y;
          }
      }
    }
  }
};

template <typename T, int G, bool ZEROS>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) w4_kernel(const W4Params p) {
  constexpr int kRecord = record_bytes(G, ZEROS), kStage = kM * kRecord;
  constexpr int kTail = (kRecord - 1024) / 16, kTails = (kM * kTail + 31) / 32;   // 16-byte pieces behind the codes
  extern __shared__ __align__(16) uint8_t s_mem[];
  __shared__ int s_chunks[kMaxExperts + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* ring = s_mem + warp * (kStages * kStage);
  float* s_sums = reinterpret_cast<float*>(s_mem + kWarps * kStages * kStage);
  // Warps split the columns k_split ways and the task's tiles kWarps / k_split ways.
  const int k_split = p.k_split, m_groups = kWarps / k_split, kw = warp % k_split, mg = warp / k_split;
  const int k0 = (int)((int64_t)p.k_steps * kw / k_split), k1 = (int)((int64_t)p.k_steps * (kw + 1) / k_split);

  // With bf16 rows the kernel before this one, which has started, brings them to
  // fp16; what came before that one is complete.
  if (!p.row_exp) griddep_wait();
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
  const int last_c = (int)(last / p.n_tiles), last_m = (int)(last - (int64_t)last_c * p.n_tiles);
  auto find_chunk = [&](Task& w) {             // the expert and rows of chunk c
    int lo = 0, hi = p.E;                      // s_chunks[lo] <= c < s_chunks[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_chunks[mid] <= w.c) lo = mid; else hi = mid;
    }
    w.e = lo;
    int r;
    const int rows = rows_of(lo, &r), chunks = (rows + kMaxRows - 1) / kMaxRows, i = w.c - s_chunks[lo];
    const int a = (int)((int64_t)rows * i / chunks);
    w.r0 = r + a;
    w.cnt = (int)((int64_t)rows * (i + 1) / chunks) - a;
  };
  auto size_task = [&](Task& w) {              // even tasks of at most kM * m_groups tiles; 0 at the end
    const int left = (w.c < last_c ? p.n_tiles : w.c == last_c ? last_m : 0) - w.m0;
    const int most = kM * m_groups, tasks = (left + most - 1) / most;
    w.m = left > 0 ? (left + tasks - 1) / tasks : 0;
  };
  auto next_task = [&](Task& w) {
    w.m0 += w.m;
    if (w.m0 == p.n_tiles) {
      w.m0 = 0;
      ++w.c;
      if (w.c < last_c || (w.c == last_c && last_m > 0)) find_chunk(w);
    }
    size_task(w);
  };
  // A warp's own tiles of a task: group mg of m_groups even ones.
  auto own_first = [&](const Task& w, int group) { return w.m * group / m_groups; };

  Task work;
  work.c = (int)(first / p.n_tiles);
  work.m0 = (int)(first - (int64_t)work.c * p.n_tiles);
  work.m = 0;
  if (first < last) {
    find_chunk(work);
    size_task(work);
  }
  // The copies run kStages - 1 steps ahead of the products, across tasks.
  Task ahead = work;
  const size_t m_stride = (size_t)p.k_steps * kRecord;
  const uint8_t* source = nullptr;             // this lane's first 16 bytes of the next step
  int ahead_m = 0, ahead_k = k0, ahead_slot = 0;
  auto start_ahead = [&]() {
    const int a = own_first(ahead, mg);
    ahead_m = own_first(ahead, mg + 1) - a;
    ahead_k = k0;
    source = p.records + ((size_t)ahead.e * p.n_tiles + ahead.m0 + a) * m_stride + (size_t)k0 * kRecord;
  };
  if (work.m) start_ahead();
  const bool idle = k0 == k1;                  // fewer steps than k_split
  auto advance = [&]() {
    if (ahead.m && !idle) {
      const uint32_t slot = smem_u32(ring + ahead_slot * kStage);
#pragma unroll
      for (int m = 0; m < kM; ++m)
        if (m < ahead_m) {
          const uint8_t* src = source + m * m_stride + lane * 16;
          copy16(slot + m * kRecord + lane * 16, src);
          copy16(slot + m * kRecord + 512 + lane * 16, src + 512);
        }
#pragma unroll
      for (int q = 0; q < kTails; ++q) {
        const int i = lane + 32 * q, m = i / kTail, off = 1024 + (i - m * kTail) * 16;
        if (m < ahead_m) copy16(slot + m * kRecord + off, source + m * m_stride + off);
      }
      source += kRecord;
      if (++ahead_k == k1) {
        next_task(ahead);
        if (ahead.m) start_ahead();
      }
    }
    ahead_slot = ahead_slot + 1 == kStages ? 0 : ahead_slot + 1;
    copies_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) advance();
  if (p.row_exp) griddep_wait();               // x is there
  griddep_launch_dependents();

  int slot = 0;
  auto run = [&](const Task& w, auto nt_tag) {
    constexpr int NT = decltype(nt_tag)::value;
    using S = Step<T, NT, G, ZEROS>;
    const int g = lane >> 2, t = lane & 3;
    const int m_first = own_first(w, mg), m_here = own_first(w, mg + 1) - m_first;
    float sums[kM][NT][4];
#pragma unroll
    for (int m = 0; m < kM; ++m)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[m][nt][i] = 0.f;
    const __half* rows[NT];                    // columns of missing rows come from the first: they go nowhere
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
      rows[nt] = p.x + (size_t)(w.r0 + (nt * 8 + g < w.cnt ? nt * 8 + g : 0)) * p.D + 8 * t;
    uint4 x[2][NT][2];
    S::load_x(rows, k0 * kStepK, p.D, x[0]);
#pragma unroll 1
    for (int k = k0; k < k1; ++k) {
      __syncwarp();                            // the slot that is filled next has been read by all lanes
      advance();
      S::load_x(rows, k * kStepK + 64, p.D, x[1]);
      copies_wait<kStages - 1>();
      __syncwarp();
      const uint8_t* stage = ring + slot * kStage;
      S::multiply(stage, 0, m_here, x[0], sums);
      S::load_x(rows, (k + 1) * kStepK, k + 1 < k1 ? p.D : 0, x[0]);
      S::multiply(stage, 1, m_here, x[1], sums);
      slot = slot + 1 == kStages ? 0 : slot + 1;
    }
    // The warps' sums meet in shared memory and are added in the columns' order.
    float* mine = s_sums + warp * (kMaxRows * kSumStride);
    const int most = (w.m + m_groups - 1) / m_groups;
#pragma unroll
    for (int m1 = 0; m1 < kM; m1 += kSumM) {
      if (m1 >= most) break;
#pragma unroll
      for (int m = 0; m < kSumM; ++m)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            mine[(nt * 8 + 2 * t + (i & 1)) * kSumStride + m * 16 + g + 8 * (i >> 1)] = sums[m1 + m][nt][i];
      __syncthreads();
      for (int o = threadIdx.x; o < m_groups * w.cnt * kSumM * 16; o += kThreads) {
        const int group = o / (w.cnt * kSumM * 16), i = o - group * (w.cnt * kSumM * 16);
        const int row = i / (kSumM * 16), n = i % (kSumM * 16);
        const int tile = own_first(w, group) + m1 + n / 16, col = (w.m0 + tile) * 16 + n % 16;
        if (tile >= own_first(w, group + 1) || col >= p.N) continue;
        float v = 0.f;
        for (int q = 0; q < k_split; ++q) v += s_sums[((group * k_split + q) * kMaxRows + row) * kSumStride + n];
        v = ldexpf(v, 24 + (p.row_exp ? __ldg(p.row_exp + w.r0 + row) : 0));
        const size_t at = (size_t)(w.r0 + row) * p.N + col;
        if (p.out_f32) static_cast<float*>(p.y)[at] = v;
        else static_cast<T*>(p.y)[at] = from_float<T>(v);
      }
      __syncthreads();
    }
  };
  for (; work.m; next_task(work)) {
    if (work.cnt <= 8) run(work, std::integral_constant<int, 1>{});
    else run(work, std::integral_constant<int, 2>{});
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

template <typename T, int G, bool ZEROS>
int launch_w4(const W4Params& p, const void* x, int sms, cudaStream_t s) {
  constexpr size_t kSmem = (size_t)kWarps * kStages * kM * record_bytes(G, ZEROS) + kSumBytes;
  static_assert((kSmem + 4 * (kMaxExperts + 4) + 1024) * kCtasPerSm <= 227 * 1024, "shared memory of the resident CTAs");
  static std::atomic<void*> seen[kMaxCachedDevices];
  cudaError_t e = once_per_context(seen, [] {
    return cudaFuncSetAttribute(w4_kernel<T, G, ZEROS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem);
  });
  if (e != cudaSuccess) return cuda_status(e);
  if (p.row_exp) {
    e = launch_pdl(w4_convert_kernel, dim3(p.R), dim3(kConvertThreads), 0, s, static_cast<const __nv_bfloat16*>(x),
                   p.D, const_cast<__half*>(p.x), const_cast<int32_t*>(p.row_exp));
    if (e != cudaSuccess) return cuda_status(e);
  }
  return cuda_status(launch_pdl(w4_kernel<T, G, ZEROS>, dim3(kCtasPerSm * sms), dim3(kThreads), kSmem, s, p));
}

template <typename T, int G>
int run_w4_g(const W4Params& p, const void* x, bool zeros, int sms, cudaStream_t s) {
  return zeros ? launch_w4<T, G, true>(p, x, sms, s) : launch_w4<T, G, false>(p, x, sms, s);
}
template <typename T>
int run_w4(const W4Params& p, const void* x, int G, bool zeros, int sms, cudaStream_t s) {
  if (G == 32) return run_w4_g<T, 32>(p, x, zeros, sms, s);
  if (G == 64) return run_w4_g<T, 64>(p, x, zeros, sms, s);
  return run_w4_g<T, 128>(p, x, zeros, sms, s);
}

bool group_ok(int32_t d, int32_t group_size) {
  return d >= 1 && (group_size == 32 || group_size == 64 || group_size == 128) && d % group_size == 0;
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

MOE_API int moe_w4_layout_size(int32_t num_experts, int32_t n, int32_t d, int32_t group_size, int32_t with_zeros,
                               uint64_t* bytes) {
  if (num_experts < 1 || n < 1 || !group_ok(d, group_size) || !bytes) return MOE_ERR_INVALID_ARGUMENT;
  if (num_experts > kMaxExperts || n > (1 << 30) || d > (1 << 24)) return MOE_ERR_TOO_LARGE;
  *bytes = (uint64_t)num_experts * ((n + 15) / 16) * ((d + kStepK - 1) / kStepK) * record_bytes(group_size, with_zeros);
  return MOE_OK;
}

MOE_API int moe_w4_lay_out(const void* codes, const void* scales, const void* zeros, int32_t num_experts, int32_t n,
                           int32_t d, int32_t group_size, void* layout, void* stream) {
  uint64_t bytes = 0;
  int st = moe_w4_layout_size(num_experts, n, d, group_size, zeros != nullptr, &bytes);
  if (st != MOE_OK) return st;
  if (!codes || !scales || !layout) return MOE_ERR_INVALID_ARGUMENT;
  if (!aligned_to(codes, 4) || !aligned_to(scales, 2) || !aligned_to(layout, 16)) return MOE_ERR_MISALIGNED;
  if ((st = require_device(nullptr)) != MOE_OK) return st;
  const uint64_t blocks = (bytes / 16 + 255) / 256;
  if (blocks > INT32_MAX) return MOE_ERR_TOO_LARGE;
  return cuda_status(launch_pdl(w4_lay_out_kernel, dim3((unsigned)blocks), dim3(256), 0,
                                static_cast<cudaStream_t>(stream), static_cast<const uint8_t*>(codes),
                                static_cast<const uint16_t*>(scales), static_cast<const uint8_t*>(zeros), n, d,
                                group_size, (n + 15) / 16, (d + kStepK - 1) / kStepK, (int64_t)(bytes / 16),
                                static_cast<uint8_t*>(layout)));
}

MOE_API int moe_w4_workspace_size(int32_t num_rows, int32_t d, int32_t dtype, uint64_t* bytes) {
  if (num_rows < 0 || d < 1 || (dtype != MOE_F16 && dtype != MOE_BF16) || !bytes) return MOE_ERR_INVALID_ARGUMENT;
  *bytes = dtype == MOE_BF16 ? rows_bytes(num_rows, d) + (uint64_t)num_rows * sizeof(int32_t) : 0;
  return MOE_OK;
}

MOE_API int moe_w4_matvec(const void* x, const void* layout, const int32_t* offsets, int32_t num_rows,
                          int32_t num_experts, int32_t n, int32_t d, int32_t group_size, int32_t with_zeros,
                          int32_t dtype, int32_t out_dtype, int32_t zero_other_rows, void* y, void* workspace,
                          uint64_t workspace_bytes, void* stream) {
  uint64_t need = 0;
  int st = moe_w4_layout_size(num_experts, n, d, group_size, with_zeros, &need);
  if (st == MOE_OK) st = moe_w4_workspace_size(num_rows, d, dtype, &need);
  if (st != MOE_OK) return st;
  if ((!offsets && num_experts != 1) || (out_dtype != dtype && out_dtype != MOE_F32)) return MOE_ERR_INVALID_ARGUMENT;
  if (num_rows == 0) return MOE_OK;
  if (!x || !layout || !y) return MOE_ERR_INVALID_ARGUMENT;
  if (!aligned_to(x, 16) || !aligned_to(layout, 16) || !aligned_to(offsets, 4) ||
      !aligned_to(y, dtype_bytes(out_dtype)) || !aligned_to(workspace, 256))
    return MOE_ERR_MISALIGNED;
  if (workspace_bytes < need || (need && !workspace)) return MOE_ERR_WORKSPACE_TOO_SMALL;
  int sms = 0;
  if ((st = require_device(&sms)) != MOE_OK) return st;
  W4Params p;
  p.R = num_rows; p.N = n; p.D = d; p.E = num_experts;
  p.n_tiles = (n + 15) / 16;
  p.k_steps = (d + kStepK - 1) / kStepK;
  p.k_split = p.k_steps >= 32 ? 8 : p.k_steps >= 16 ? 4 : p.k_steps >= 8 ? 2 : 1;
  p.x = static_cast<const __half*>(dtype == MOE_BF16 ? workspace : x);
  p.row_exp = dtype == MOE_BF16 ? reinterpret_cast<const int32_t*>(static_cast<const uint8_t*>(workspace) +
                                                                   rows_bytes(num_rows, d))
                                : nullptr;
  p.records = static_cast<const uint8_t*>(layout);
  p.offsets = offsets;
  p.y = y;
  p.out_f32 = out_dtype == MOE_F32;
  p.zero_rest = zero_other_rows != 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == MOE_BF16 ? run_w4<__nv_bfloat16>(p, x, group_size, with_zeros != 0, sms, s)
                           : run_w4<__half>(p, x, group_size, with_zeros != 0, sms, s);
}

}  // extern "C"
