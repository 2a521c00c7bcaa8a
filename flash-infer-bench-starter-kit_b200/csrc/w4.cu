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
// bf16 rows of x are brought to fp16 by a power of two for each row that puts its
// largest magnitude into [2^14, 2^15): exact for values down to 2^-28 of the largest,
// below that off by at most 2^-39 of it.  (Next to an infinity or a NaN the finite
// values vanish, as they do in the sum.)
//
// Layout (made once, by moe_w4_lay_out): records of 16 rows x 128 columns, in the
// order in which a CTA streams them, so that what it takes at a time is one or two
// pieces of memory: [E][groups of 8 rows of records][stages of 4 columns of records]
// [8][4][record], where the last group and the last stage may be smaller.  A record is
//   two 16 x 64 tiles of codes in the order in which a warp's lanes take them, 16
//   bytes a lane.  With lane = 4 * g + t, 32-bit word j holds columns c = 32 * (j / 2) +
//   8 * t + 4 * (j % 2) + {0, 2, 1, 3} in its bytes 0 to 3, row g in the low half of a
//   byte and row g + 8 in the high half: a lane's share of x is then 16 consecutive
//   bytes for each 32 columns;
//   the record's scales [128 / G][8][2] (rows g, g + 8 together), then, if there are any,
//   its zero points likewise.
#include <type_traits>

#include "rows.cuh"

namespace moe {
namespace {

constexpr int kStepK = 128;               // columns of a record
constexpr int kSplit = 4;                 // warps along the columns: a stage holds 4 steps
constexpr int kGroupsM = 4;               // groups of warps along the rows of tiles
constexpr int kM = 2;                     // rows of tiles (of records) of a warp
constexpr int kTaskM = kM * kGroupsM;     // of a task
constexpr int kConsumers = kSplit * kGroupsM;       // warps that multiply; one more copies
constexpr int kThreads = (kConsumers + 1) * 32;
constexpr int kStages = 3;
constexpr int kMaxRows = 24;              // rows of x in a task
constexpr int kMaxExperts = 1024;
constexpr int kStageK = kSplit * kStepK;  // columns of a stage
constexpr int kRowPiece = kStageK * 2;    // bytes of a row of x in a stage
constexpr int kSumStride = kM * 16 + 4;   // of the sums in shared memory: a warp's stores hit 32 banks
constexpr size_t kSumBytes = sizeof(float) * kConsumers * 8 * kSumStride;

// Bytes of a record with groups of G columns.
__host__ __device__ constexpr int record_bytes(int G, bool zeros) { return 1024 + kStepK / G * (zeros ? 48 : 32); }

struct W4Params {
  const uint8_t* x;        // [stages][R][kRowPiece]
  const int32_t* row_exp;  // [R]: the exponent taken out of a row
  const uint8_t* records;  // as above
  const int32_t* offsets;  // [E + 1], or null: one matrix for all rows
  void* y;
  int R, N, E, n_tiles, k_steps, stages;
  int out_f32, zero_rest;
};

// Set when a wait gave up; read and cleared by moe_w4_read_device_error.
__device__ int g_w4_error;

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
  const int64_t record = at / per_record, per_expert = (int64_t)n_tiles * k_steps, e = record / per_expert;
  const int piece = (int)(at - record * per_record);
  const int in_expert = (int)(record - e * per_expert), group = in_expert / (kTaskM * k_steps);
  const int in_group = in_expert - group * (kTaskM * k_steps);
  const int tiles = n_tiles - group * kTaskM < kTaskM ? n_tiles - group * kTaskM : kTaskM;
  const int stage = in_group / (tiles * kSplit), in_stage = in_group - stage * (tiles * kSplit);
  const int steps = k_steps - stage * kSplit < kSplit ? k_steps - stage * kSplit : kSplit;
  const int row0 = (group * kTaskM + in_stage / steps) * 16, step = stage * kSplit + in_stage % steps;
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
      const int v = first + i, of = step * groups + v / 16, row = row0 + (v & 15) / 2 + 8 * (v & 1);
      if (row >= N || of * G >= D) continue;
      const size_t src = ((size_t)e * N + row) * (D / G) + of;
      if (is_zeros) o.b[i] = zeros[src];
      else o.h[i] = scales[src];
    }
  }
  *reinterpret_cast<uint4*>(out + at * 16) = o.v;
}

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

// --------------------------------------------------------------------------
// Rows of x for the product: a CTA takes 8 rows, finds the largest magnitude of each
// (bf16) and writes them in fp16 by stages of 512 columns, zeros behind D; 16-byte pieces 4
// apart change places in odd rows, so that a warp's reads of 8 rows hit 32 banks.
// Reads and writes R * D * 2 bytes, out of and into L2: latency.
// --------------------------------------------------------------------------
constexpr int kRowsThreads = 512;

template <typename T>
__global__ void __launch_bounds__(kRowsThreads)
w4_rows_kernel(const T* __restrict__ x, int R, int D, int stages, uint8_t* __restrict__ out,
               int32_t* __restrict__ row_exp) {
  constexpr int kWarps = kRowsThreads / 32;
  constexpr bool kScaled = !std::is_same<T, __half>::value;
  __shared__ float s_max[kWarps];
  griddep_wait();
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // warps w and w + 8: the two halves of row w
  const int row = blockIdx.x * 8 + (warp & 7);
  int exp = 0;
  if constexpr (kScaled) {
    float amax = 0.f;
    if (row < R)
#pragma unroll 4
      for (int i = (warp >> 3) * 256 + lane * 8; i < D; i += 512) {   // D is a multiple of 32
        const Pack<T, 8> v = load_cached<T, 8>(x + (size_t)row * D + i);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float a = fabsf(to_float(v.v[j]));
          amax = a < INFINITY ? fmaxf(amax, a) : INFINITY;
        }
      }
#pragma unroll
    for (int off = 16; off; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
    if (lane == 0) s_max[warp] = amax;
    __syncthreads();
    amax = fmaxf(s_max[warp & 7], s_max[(warp & 7) + 8]);
    // amax * 2^-exp in [2^14, 2^15), as far as 2^-exp is a normal number
    exp = (int)((__float_as_uint(amax) >> 23) & 0xff) - 127 - 14;
    exp = exp < -120 ? -120 : exp;
  }
  if (row >= R) return;
  const float down = __uint_as_float((uint32_t)(127 - exp) << 23);
#pragma unroll 4
  for (int i = (warp >> 3) * 256 + lane * 8; i < stages * kStageK; i += 512) {
    Pack<__half, 8> o = zero_pack<__half, 8>();
    if (i < D) {
      const Pack<T, 8> v = load_cached<T, 8>(x + (size_t)row * D + i);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        o.v[j] = kScaled ? __float2half_rn(to_float(v.v[j]) * down) : from_float<__half>(to_float(v.v[j]));
    }
    const int stage = i / kStageK, piece = (i % kStageK / 8) ^ ((row & 1) << 2);
    store_wide<__half, 8>(reinterpret_cast<__half*>(out + ((size_t)stage * R + row) * kRowPiece) + piece * 8, o);
  }
  if (warp < 8 && lane == 0) row_exp[row] = exp;
}

// --------------------------------------------------------------------------
// The product.
// --------------------------------------------------------------------------
// One piece of memory into shared memory, counted by an mbarrier; 16-byte aligned.
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

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

// The tasks of a CTA.  The (chunk, row of tiles) pairs are dealt out evenly: CTA b takes the
// pairs [total * b / CTAs, total * (b + 1) / CTAs), in even tasks of at most kTaskM tiles.
struct Tasks {
  const W4Params* p;
  const int* chunks_before;   // [E + 1]
  int last_c, last_m;

  // Rows of expert e, whatever the offsets say within [0, R].
  static __device__ __forceinline__ int rows_of(const W4Params& p, int e, int* first) {
    if (!p.offsets) { *first = 0; return p.R; }
    int a = __ldg(p.offsets + e), b = __ldg(p.offsets + e + 1);
    a = a < 0 ? 0 : a > p.R ? p.R : a;
    b = b < a ? a : b > p.R ? p.R : b;
    *first = a;
    return b - a;
  }
  __device__ __forceinline__ Task begin() {
    const int64_t total = (int64_t)chunks_before[p->E] * p->n_tiles;
    const int64_t first = total * blockIdx.x / gridDim.x, last = total * (blockIdx.x + 1) / gridDim.x;
    last_c = (int)(last / p->n_tiles);
    last_m = (int)(last - (int64_t)last_c * p->n_tiles);
    Task w;
    w.c = (int)(first / p->n_tiles);
    w.m0 = (int)(first - (int64_t)w.c * p->n_tiles);
    w.m = w.e = w.r0 = w.cnt = 0;
    if (first < last) {
      find_chunk(w);
      size_task(w);
    }
    return w;
  }
  __device__ __forceinline__ void find_chunk(Task& w) const {   // the expert and rows of chunk c
    int lo = 0, hi = p->E;                                     // chunks_before[lo] <= c < chunks_before[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (chunks_before[mid] <= w.c) lo = mid; else hi = mid;
    }
    w.e = lo;
    int r;
    const int rows = rows_of(*p, lo, &r), chunks = (rows + kMaxRows - 1) / kMaxRows, i = w.c - chunks_before[lo];
    const int a = (int)((int64_t)rows * i / chunks);
    w.r0 = r + a;
    w.cnt = (int)((int64_t)rows * (i + 1) / chunks) - a;
  }
  __device__ __forceinline__ void size_task(Task& w) const {    // 0 tiles: the end
    const int left = (w.c < last_c ? p->n_tiles : w.c == last_c ? last_m : 0) - w.m0;
    const int tasks = (left + kTaskM - 1) / kTaskM;
    w.m = left > 0 ? (left + tasks - 1) / tasks : 0;
  }
  __device__ __forceinline__ void next(Task& w) const {
    w.m0 += w.m;
    if (w.m0 == p->n_tiles) {
      w.m0 = 0;
      ++w.c;
      if (w.c < last_c || (w.c == last_c && last_m > 0)) find_chunk(w);
    }
    size_task(w);
  }
};
// The tiles of a task that a group of warps has: [own_first(m, group), own_first(m, group + 1)).
__device__ __forceinline__ int own_first(int m, int group) { return m * group / kGroupsM; }

// One step of a warp: kM records (`m_here` of them are there) of 128 columns, times NT * 8 rows of x.
template <typename T, int NT, int G, bool ZEROS>
__device__ __forceinline__ void multiply(const uint8_t* records, int m_stride, int m_here, const uint8_t* x_stage,
                                         int odd, int kw, float (&sums)[kM][NT][4]) {
  constexpr int kRecord = record_bytes(G, ZEROS);
  constexpr int kParts = G == 32 ? 2 : 1;          // groups in half a record
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    uint4 x[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        x[nt][h] = *reinterpret_cast<const uint4*>(
            x_stage + (nt * 8 + g) * kRowPiece + ((kw * (kStepK / 8) + half * 8 + h * 4 + t) ^ (((g ^ odd) & 1) << 2)) * 16);
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
      const int group = (half * 64 + part * 32) / G;
#pragma unroll
      for (int m = 0; m < kM; ++m) {
        if (m >= m_here) break;
        const uint8_t* rec = records + m * m_stride;
        const uint4 c = *reinterpret_cast<const uint4*>(rec + half * 512 + lane * 16);
        const uint32_t word[4] = {c.x, c.y, c.z, c.w};
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
          for (int h = 0; h < 2; ++h) {            // rows g and g + 8; two rows of x in each fma
            const float2 sum = __ffma2_rn(make_float2(a[nt][2 * h], a[nt][2 * h + 1]), h ? make_float2(s.y, s.y) : make_float2(s.x, s.x),
                                          make_float2(sums[m][nt][2 * h], sums[m][nt][2 * h + 1]));
            sums[m][nt][2 * h] = sum.x;
            sums[m][nt][2 * h + 1] = sum.y;
          }
      }
    }
  }
}

// A CTA of 16 warps that multiply (4 along the columns times 4 along the rows of tiles)
// and one that copies.  A stage of the ring holds 4 steps of columns of up to 8 rows of tiles
// and of up to 24 rows of x, about 60 KB in two or three copies (a copy for every
// row of tiles and of x made the copying warp the limit: 42 us of copies alone for 8
// matrices of 4096 x 7168, the memory's rate being 19 us).
template <typename T, int G, bool ZEROS>
__global__ void __launch_bounds__(kThreads, 1) w4_kernel(const W4Params p) {
  constexpr int kRecord = record_bytes(G, ZEROS), kWeights = kTaskM * kSplit * kRecord;   // bytes of a stage
  constexpr int kStage = kWeights + kMaxRows * kRowPiece;
  extern __shared__ __align__(128) uint8_t s_mem[];
  __shared__ int s_chunks[kMaxExperts + 1];
  __shared__ __align__(8) uint64_t s_full[kStages], s_empty[kStages];
  __shared__ volatile int s_abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* s_sums = reinterpret_cast<float*>(s_mem + kStages * kStage);

  // The kernel before this one, which has started, makes the rows of x; what came before
  // that one is complete, so the offsets and weights may be read.
  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], kConsumers);
    }
    fence_mbar_init();
  }
  // Chunks of up to kMaxRows rows before expert e: the same in every CTA.
  for (int e = threadIdx.x; e < p.E; e += kThreads) {
    int first;
    s_chunks[e] = (Tasks::rows_of(p, e, &first) + kMaxRows - 1) / kMaxRows;
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
  Tasks tasks;
  tasks.p = &p;
  tasks.chunks_before = s_chunks;
  Task work = tasks.begin();

  if (warp == kConsumers) {
    // ---- copies
    auto copy_weights = [&](const Task& w, int stage, int slot) {
      const int left = p.k_steps - stage * kSplit, steps = left < kSplit ? left : kSplit;
      // the task's tiles lie in one group of 8 or in two: lane 0 and lane 1
      const int group = w.m0 / kTaskM, in_first = kTaskM - w.m0 % kTaskM < w.m ? kTaskM - w.m0 % kTaskM : w.m;
      if (lane == 0) mbar_arrive_expect_tx(&s_full[slot], w.m * steps * kRecord + w.cnt * kRowPiece);
      __syncwarp();
      const int m = lane == 0 ? in_first : w.m - in_first;
      if (lane < 2 && m > 0) {
        const int at = (group + lane) * kTaskM, tiles = p.n_tiles - at < kTaskM ? p.n_tiles - at : kTaskM;
        const size_t record = ((size_t)w.e * p.n_tiles + at) * p.k_steps + stage * kSplit * tiles +
                              (lane == 0 ? w.m0 % kTaskM : 0) * steps;
        bulk_copy(smem_u32(s_mem + slot * kStage + (lane == 0 ? 0 : in_first * steps * kRecord)),
                  p.records + record * kRecord, m * steps * kRecord, &s_full[slot]);
      }
    };
    auto copy_rows = [&](const Task& w, int stage, int slot) {
      if (lane == 0)
        bulk_copy(smem_u32(s_mem + slot * kStage + kWeights), p.x + ((size_t)stage * p.R + w.r0) * kRowPiece,
                  w.cnt * kRowPiece, &s_full[slot]);
    };
    auto step_on = [&](Task& w, int& stage) {
      if (++stage == p.stages) {
        stage = 0;
        tasks.next(w);
      }
    };
    // The first stages' weights do not wait for the rows of x.
    Task w = work;
    int stage = 0, issued = 0;
    for (; issued < kStages && w.m; ++issued) {
      copy_weights(w, stage, issued);
      step_on(w, stage);
    }
    griddep_wait();
    griddep_launch_dependents();
    fence_proxy_async();
    {
      Task first = work;
      int st = 0;
      for (int i = 0; i < issued; ++i) {
        copy_rows(first, st, i);
        step_on(first, st);
      }
    }
    int slot = 0;
    uint32_t parity = 0;
    bool ok = true;
    for (; w.m && ok; ++issued) {
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(&s_empty[slot], parity, &s_abort));
      if (!ok) break;
      copy_weights(w, stage, slot);
      copy_rows(w, stage, slot);
      step_on(w, stage);
      if (++slot == kStages) { slot = 0; parity ^= 1; }
    }
    if (!ok) {                                     // let the copies that are under way land
      if (lane == 0) {
        raise_error(&g_w4_error, kDevTimeoutProducer);
        volatile int none = 0;
        for (int i = issued > kStages ? issued - kStages : 0; i < issued; ++i)
          mbar_wait_bounded(&s_full[i % kStages], (uint32_t)(i / kStages) & 1u, &none);
      }
      __syncwarp();
    }
    return;
  }

  // ---- products
  griddep_wait();                                  // row_exp
  griddep_launch_dependents();
  const int kw = warp % kSplit, mg = warp / kSplit, g = lane >> 2, t = lane & 3;
  int slot = 0;
  uint32_t parity = 0;
  bool ok = true;                                  // after a wait that gave up: go on without work
  auto run = [&](const Task& w, auto nt_tag) {
    constexpr int NT = decltype(nt_tag)::value;
    const int m_first = own_first(w.m, mg), m_here = own_first(w.m, mg + 1) - m_first;
    float sums[kM][NT][4];
#pragma unroll
    for (int m = 0; m < kM; ++m)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[m][nt][i] = 0.f;
#pragma unroll 1
    for (int stage = 0; stage < p.stages; ++stage) {
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait_bounded(&s_full[slot], parity, &s_abort));
      const uint8_t* at = s_mem + slot * kStage;
      const int left = p.k_steps - stage * kSplit, stride = (left < kSplit ? left : kSplit) * kRecord;
      if (ok && m_here > 0 && kw < left)
        multiply<T, NT, G, ZEROS>(at + m_first * stride + kw * kRecord, stride, m_here, at + kWeights, w.r0, kw, sums);
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_empty[slot]);
      if (++slot == kStages) { slot = 0; parity ^= 1; }
    }
    // The warps' sums meet in shared memory and are added in the columns' order, 8 rows
    // of x at a time.
    float* mine = s_sums + warp * (8 * kSumStride);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int m = 0; m < kM; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          mine[(2 * t + (i & 1)) * kSumStride + m * 16 + g + 8 * (i >> 1)] = sums[m][nt][i];
      named_bar_sync(1, kConsumers * 32);
      for (int o = threadIdx.x; o < kGroupsM * 8 * kM * 16; o += kConsumers * 32) {
        const int group = o / (8 * kM * 16), row = o / (kM * 16) % 8, n = o % (kM * 16);
        const int tile = own_first(w.m, group) + n / 16, col = (w.m0 + tile) * 16 + n % 16;
        if (tile >= own_first(w.m, group + 1) || nt * 8 + row >= w.cnt || col >= p.N) continue;
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < kSplit; ++q) v += s_sums[((group * kSplit + q) * 8 + row) * kSumStride + n];
        const int r = w.r0 + nt * 8 + row;
        v = ldexpf(v, 24 + __ldg(p.row_exp + r));
        const size_t to = (size_t)r * p.N + col;
        if (p.out_f32) static_cast<float*>(p.y)[to] = v;
        else static_cast<T*>(p.y)[to] = from_float<T>(v);
      }
      named_bar_sync(1, kConsumers * 32);
    }
  };
  for (; work.m; tasks.next(work)) {
    if (work.cnt <= 8) run(work, std::integral_constant<int, 1>{});
    else if (work.cnt <= 16) run(work, std::integral_constant<int, 2>{});
    else run(work, std::integral_constant<int, 3>{});
  }
  if (!ok && lane == 0) raise_error(&g_w4_error, kDevTimeoutMma);
  if (p.zero_rest && p.offsets) {                  // rows of no expert
    int a = __ldg(p.offsets), b = __ldg(p.offsets + p.E);
    a = a < 0 ? 0 : a > p.R ? p.R : a;
    b = b < a ? a : b > p.R ? p.R : b;
    const int64_t rest = (int64_t)(p.R - (b - a)) * p.N;
    for (int64_t i = (int64_t)blockIdx.x * (kConsumers * 32) + threadIdx.x; i < rest;
         i += (int64_t)gridDim.x * (kConsumers * 32)) {
      int64_t r = i / p.N;
      const int64_t n = i - r * p.N;
      if (r >= a) r += b - a;
      if (p.out_f32) static_cast<float*>(p.y)[r * p.N + n] = 0.f;
      else static_cast<T*>(p.y)[r * p.N + n] = from_float<T>(0.f);
    }
  }
}

// Workspace: the rows of x by stages, then their exponents.
int stages_of(int64_t d) { return (int)((d + kStageK - 1) / kStageK); }
uint64_t rows_bytes(int64_t R, int64_t d) { return (uint64_t)R * stages_of(d) * kRowPiece; }

template <typename T, int G, bool ZEROS>
int launch_w4(const W4Params& p, const void* x, int d, int sms, cudaStream_t s) {
  constexpr size_t kSmem = (size_t)kStages * (kTaskM * kSplit * record_bytes(G, ZEROS) + kMaxRows * kRowPiece) + kSumBytes;
  static_assert(kSmem + 4 * (kMaxExperts + 4) + 1024 <= 227 * 1024, "shared memory");
  static std::atomic<void*> seen[kMaxCachedDevices];
  cudaError_t e = once_per_context(seen, [] {
    return cudaFuncSetAttribute(w4_kernel<T, G, ZEROS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem);
  });
  if (e != cudaSuccess) return cuda_status(e);
  e = launch_pdl(w4_rows_kernel<T>, dim3((p.R + 7) / 8), dim3(kRowsThreads), 0, s, static_cast<const T*>(x),
                 p.R, d, p.stages, const_cast<uint8_t*>(p.x), const_cast<int32_t*>(p.row_exp));
  if (e != cudaSuccess) return cuda_status(e);
  return cuda_status(launch_pdl(w4_kernel<T, G, ZEROS>, dim3(sms), dim3(kThreads), kSmem, s, p));
}

template <typename T, int G>
int run_w4_g(const W4Params& p, const void* x, int d, bool zeros, int sms, cudaStream_t s) {
  return zeros ? launch_w4<T, G, true>(p, x, d, sms, s) : launch_w4<T, G, false>(p, x, d, sms, s);
}
template <typename T>
int run_w4(const W4Params& p, const void* x, int d, int G, bool zeros, int sms, cudaStream_t s) {
  if (G == 32) return run_w4_g<T, 32>(p, x, d, zeros, sms, s);
  if (G == 64) return run_w4_g<T, 64>(p, x, d, zeros, sms, s);
  return run_w4_g<T, 128>(p, x, d, zeros, sms, s);
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

MOE_API int moe_w4_workspace_size(int32_t num_rows, int32_t d, uint64_t* bytes) {
  if (num_rows < 0 || d < 1 || !bytes) return MOE_ERR_INVALID_ARGUMENT;
  *bytes = rows_bytes(num_rows, d) + (uint64_t)num_rows * sizeof(int32_t);
  return MOE_OK;
}

MOE_API int moe_w4_matvec(const void* x, const void* layout, const int32_t* offsets, int32_t num_rows,
                          int32_t num_experts, int32_t n, int32_t d, int32_t group_size, int32_t with_zeros,
                          int32_t dtype, int32_t out_dtype, int32_t zero_other_rows, void* y, void* workspace,
                          uint64_t workspace_bytes, void* stream) {
  uint64_t need = 0;
  int st = moe_w4_layout_size(num_experts, n, d, group_size, with_zeros, &need);
  if (st == MOE_OK) st = moe_w4_workspace_size(num_rows, d, &need);
  if (st != MOE_OK) return st;
  if (dtype != MOE_F16 && dtype != MOE_BF16) return MOE_ERR_INVALID_ARGUMENT;
  if ((!offsets && num_experts != 1) || (out_dtype != dtype && out_dtype != MOE_F32)) return MOE_ERR_INVALID_ARGUMENT;
  if (num_rows == 0) return MOE_OK;
  if (!x || !layout || !y) return MOE_ERR_INVALID_ARGUMENT;
  if (!aligned_to(x, 16) || !aligned_to(layout, 16) || !aligned_to(offsets, 4) ||
      !aligned_to(y, dtype_bytes(out_dtype)) || !aligned_to(workspace, 16))
    return MOE_ERR_MISALIGNED;
  if (workspace_bytes < need || !workspace) return MOE_ERR_WORKSPACE_TOO_SMALL;
  int sms = 0;
  if ((st = require_device(&sms)) != MOE_OK) return st;
  W4Params p;
  p.R = num_rows; p.N = n; p.E = num_experts;
  p.n_tiles = (n + 15) / 16;
  p.k_steps = (d + kStepK - 1) / kStepK;
  p.stages = stages_of(d);
  p.x = static_cast<const uint8_t*>(workspace);
  p.row_exp = reinterpret_cast<const int32_t*>(p.x + rows_bytes(num_rows, d));
  p.records = static_cast<const uint8_t*>(layout);
  p.offsets = offsets;
  p.y = y;
  p.out_f32 = out_dtype == MOE_F32;
  p.zero_rest = zero_other_rows != 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == MOE_BF16 ? run_w4<__nv_bfloat16>(p, x, d, group_size, with_zeros != 0, sms, s)
                           : run_w4<__half>(p, x, d, group_size, with_zeros != 0, sms, s);
}

MOE_API int moe_w4_read_device_error(void* stream, int32_t* device_error) {
  if (!device_error) return MOE_ERR_INVALID_ARGUMENT;
  const int st = require_device(nullptr);
  if (st != MOE_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int32_t v = 0;
  const int32_t none = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(&v, g_w4_error, 4, 0, cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaMemcpyToSymbolAsync(g_w4_error, &none, 4, 0, cudaMemcpyHostToDevice, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e != cudaSuccess) return cuda_status(e);
  *device_error = v;
  return v ? MOE_ERR_DEVICE_TIMEOUT : MOE_OK;
}

}  // extern "C"
