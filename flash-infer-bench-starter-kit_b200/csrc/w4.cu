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
// becomes four operand registers by four masks and one shift.  A group's sum starts at
// -zero * (sum of x over the group), made once for each row of x, and is scaled in
// fp32; the factors 2^24 and 1/16 are left to the last step, and only the output is
// rounded.
// What else was built and measured (us, caches flushed before a call; 8 matrices of
// 4096 x 7168 times a row each / 32 of them times 16 rows; this form 37 / 139, and 30 /
// 131 call after call on weights from memory): zero points subtracted from the operands, 16 more
// instructions for each 16 x 64 codes, 40 / 208; e4m3 operands, where a byte 0..15 is
// q * 2^-9, 55 / 428 (four times the executed instructions); tcgen05.mma with the decoded weights in tensor memory, 112 / 410 (8
// products of N = 16 and their hand-overs took 2000 clocks for 128 x 128 codes that
// arrive in 360).
//
// Rows of x are brought to fp16 by a power of two for each row that puts its largest
// magnitude into [2^14, 2^15): exact for bf16 values down to 2^-28 of the largest,
// below that off by at most 2^-39 of it; fp16 rows stay as they are.  A row with an
// infinity or a NaN has no finite products.
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
//   the record's scales [8][128 / G][2] (for row g of the first 8: group by group, row g's and
//   row g + 8's together), then, if there are any, its zero points likewise: a lane's
//   share of them is together.
#include <mutex>
#include <type_traits>

#include "rows.cuh"

namespace moe {
namespace {

constexpr int kStepK = 128;               // columns of a record
constexpr int kSplit = 4;                 // warps along the columns: a stage holds 4 steps
constexpr int kGroupsM = 2;               // groups of warps along the rows of tiles
constexpr int kM = 4;                     // rows of tiles (of records) of a warp
constexpr int kTaskM = kM * kGroupsM;     // of a task
constexpr int kConsumers = kSplit * kGroupsM;       // warps that multiply
constexpr int kGroupSums = 8 * kM * 16;             // sums of a group's tiles and 8 rows of x
constexpr int kThreads = (kConsumers + 4) * 32;     // a warpgroup beside them: one of its warps copies
// Registers a thread: 168 at launch (384 threads share 64,512), then few for that
// warpgroup and the rest for the two that multiply: 128 * 40 + 256 * 232 = 64,512.
constexpr int kFewRegisters = 40, kManyRegisters = 232;
constexpr int kMaxStages = 16;            // of the ring, as many as fit
constexpr int kEarly = 4;                 // stages whose weights are copied before the rows of x are there
// Rows of x in a task.  Four products of 8 rows side by side fit the registers except with
// groups of 32, where they spill: 32 rows of all of 32 experts of 7168 x 2048 217 us, in two
// tasks 195 us (4096 x 7168 in groups of 128: 211 and, in two tasks, 267 us).
__host__ __device__ constexpr int max_rows(int G) { return G == 32 ? 24 : 32; }
constexpr int kMaxExperts = 1024;
constexpr int kStageK = kSplit * kStepK;  // columns of a stage
constexpr int kRowPiece = kStageK * 2 + 64;   // bytes of a row of x in a stage: 512 fp16, then 16 sums of x
constexpr int kSumStride = kM * 16 + 4;   // of the sums in shared memory: a warp's stores hit 32 banks
constexpr int kSumFloats = kConsumers * 8 * kSumStride;
constexpr size_t kSumBytes = sizeof(float) * 2 * kSumFloats;   // two buffers
constexpr size_t kSmem = 225 * 1024 - 8 * (kMaxExperts + 4);   // dynamic: the ring, then the sums

// Bytes of a record with groups of G columns.
__host__ __device__ constexpr int record_bytes(int G, bool zeros) { return 1024 + kStepK / G * (zeros ? 48 : 32); }

struct W4Params {
  const uint8_t* x;        // [stages][R][kRowPiece]
  const int32_t* row_exp;  // [R]: the exponent taken out of a row
  const uint8_t* records;  // as above
  const int32_t* offsets;  // [E + 1], or null: one matrix for all rows
  void* y;
  int R, N, E, n_tiles, k_steps, stages, max_rows;
  int out_f32, zero_rest;
};

// Set when a wait gave up; taken by moe_w4_read_device_error: in one step, so that no error which is raised
// meanwhile on another stream is cleared unread.
__device__ int g_w4_error, g_w4_taken;
__global__ void w4_take_error_kernel() { g_w4_taken = atomicExch(&g_w4_error, 0); }

// Whether this process has launched products on the current device: else its word is 0, and reading it needs
// neither a stream nor a device of the right kind.
std::atomic<bool> g_w4_launched[kMaxCachedDevices];
bool w4_launched(bool now) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return now;
  if (dev < 0 || dev >= kMaxCachedDevices) return true;
  if (now) g_w4_launched[dev].store(true, std::memory_order_release);
  return g_w4_launched[dev].load(std::memory_order_acquire);
}

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
    const int n = is_zeros ? 16 : 8, first = (is_zeros ? tail - 2 * groups : tail) * n;   // of the [8][groups][2] values
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (i >= n) break;
      const int v = first + i, of = step * groups + v / 2 % groups, row = row0 + v / 2 / groups + 8 * (v & 1);
      if (row >= N || of * G >= D) continue;
      const size_t src = ((size_t)e * N + row) * (D / G) + of;
      if (is_zeros) o.b[i] = zeros[src];
      else o.h[i] = scales[src];
    }
  }
  *reinterpret_cast<uint4*>(out + at * 16) = o.v;
}

// d = a * b + c; d may be c.
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1, float c0, float c1, float c2, float c3) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

// --------------------------------------------------------------------------
// Rows of x for the product: a CTA takes a row, finds its largest magnitude (bf16) and
// writes it in fp16 by stages of 512 columns, zeros behind D, each followed by
// -2^-24 * (sum of x) over its groups (at most 128 columns).  Reads and writes R * D * 2
// bytes, out of and into L2: latency, so the row is read once, all of it at a time up
// to 8192 columns.
// --------------------------------------------------------------------------
constexpr int kRowsThreads = 512, kRowsHeld = 2;   // threads; 8-column pieces each keeps in registers

template <typename T, int G>
__global__ void __launch_bounds__(kRowsThreads)
w4_rows_kernel(const T* __restrict__ x, int R, int D, int stages, uint8_t* __restrict__ out,
               int32_t* __restrict__ row_exp) {
  constexpr bool kScaled = !std::is_same<T, __half>::value;
  __shared__ float s_max[kRowsThreads / 32];
  griddep_wait();
  griddep_launch_dependents();
  const int row = blockIdx.x, width = stages * kStageK;
  const T* src = x + (size_t)row * D;
  Pack<T, 8> held[kRowsHeld];
#pragma unroll
  for (int i = 0; i < kRowsHeld; ++i) {
    const int col = (i * kRowsThreads + (int)threadIdx.x) * 8;            // D is a multiple of 32
    held[i] = col < D ? load_cached<T, 8>(src + col) : zero_pack<T, 8>();
  }
  int exp = 0;
  if constexpr (kScaled) {
    float amax = 0.f;
    auto look = [&](const Pack<T, 8>& v) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float a = fabsf(to_float(v.v[j]));
        amax = a < INFINITY ? fmaxf(amax, a) : INFINITY;
      }
    };
#pragma unroll
    for (int i = 0; i < kRowsHeld; ++i) look(held[i]);
    for (int col = (kRowsHeld * kRowsThreads + (int)threadIdx.x) * 8; col < D; col += kRowsThreads * 8)
      look(load_cached<T, 8>(src + col));
#pragma unroll
    for (int off = 16; off; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = amax;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kRowsThreads / 32; ++i) amax = fmaxf(amax, s_max[i]);
    // amax * 2^-exp in [2^14, 2^15), as far as 2^-exp is a normal number
    exp = (int)((__float_as_uint(amax) >> 23) & 0xff) - 127 - 14;
    exp = exp < -120 ? -120 : exp;
  }
  const float down = __uint_as_float((uint32_t)(127 - exp) << 23);
  auto put = [&](int col, const Pack<T, 8>& v) {   // by all threads of a group's columns together
    Pack<__half, 8> o;
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      o.v[j] = __float2half_rn(kScaled ? to_float(v.v[j]) * down : to_float(v.v[j]));
      sum += to_float(o.v[j]);
    }
#pragma unroll
    for (int off = 1; off < G / 8; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    uint8_t* piece = out + ((size_t)(col / kStageK) * R + row) * kRowPiece;
    if (col >= width) return;
    store_wide<__half, 8>(reinterpret_cast<__half*>(piece) + col % kStageK, o);
    if (col % G == 0) reinterpret_cast<float*>(piece + kStageK * 2)[col % kStageK / G] = -0x1p-24f * sum;
  };
#pragma unroll
  for (int i = 0; i < kRowsHeld; ++i) put((i * kRowsThreads + (int)threadIdx.x) * 8, held[i]);
  for (int base = kRowsHeld * kRowsThreads * 8; base < width; base += kRowsThreads * 8) {   // whole CTAs
    const int col = base + (int)threadIdx.x * 8;
    put(col, col < D ? load_cached<T, 8>(src + col) : zero_pack<T, 8>());
  }
  if (threadIdx.x == 0) row_exp[row] = exp;
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

// The tasks of a CTA.  The (chunk, row of tiles) pairs are dealt out in runs of equal cost, and a
// CTA's run is split into even tasks of at most kTaskM tiles.
struct Tasks {
  const W4Params* p;
  const int* chunks_before;   // [E + 1]
  const int* cost_before;     // [E + 1]: of a row of tiles of all chunks before expert e
  int last_c, last_m, tiles;

  // No task has more tiles than this.
  __device__ __forceinline__ int most() const { return tiles < kTaskM ? tiles : kTaskM; }
  // Rows of expert e, whatever the offsets say within [0, R].
  static __device__ __forceinline__ int rows_of(const W4Params& p, int e, int* first) {
    if (!p.offsets) { *first = 0; return p.R; }
    int a = __ldg(p.offsets + e), b = __ldg(p.offsets + e + 1);
    a = a < 0 ? 0 : a > p.R ? p.R : a;
    b = b < a ? a : b > p.R ? p.R : b;
    *first = a;
    return b - a;
  }
  // Division of 64-bit numbers that mostly fit 32 bits.
  static __device__ __forceinline__ uint64_t divide(uint64_t a, uint32_t b) {
    return a >> 32 ? a / b : (uint64_t)((uint32_t)a / b);
  }
  // The pair (chunk, row of tiles), as chunk * n_tiles + tile, at which a run starts whose cost begins at `at`.
  __device__ __forceinline__ int start_of(int64_t at) const {
    int lo = 0, hi = p->E;                                     // cost_before[lo] * n_tiles <= at
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if ((int64_t)cost_before[mid] * p->n_tiles <= at) lo = mid; else hi = mid;
    }
    const int chunks = chunks_before[lo + 1] - chunks_before[lo];
    if (chunks <= 0) return chunks_before[p->E] * p->n_tiles;  // the end
    const uint32_t cost = (uint32_t)(cost_before[lo + 1] - cost_before[lo]) / (uint32_t)chunks;
    const int tile = (int)divide((uint64_t)(at - (int64_t)cost_before[lo] * p->n_tiles), cost), most = chunks * p->n_tiles;
    return chunks_before[lo] * p->n_tiles + (tile < most ? tile : most);
  }
  __device__ __forceinline__ Task begin() {
    const int64_t total = (int64_t)cost_before[p->E] * p->n_tiles;
    const int64_t each = (int64_t)divide((uint64_t)total, gridDim.x);
    const uint32_t more = (uint32_t)(total - each * gridDim.x);
    auto cost_at = [&](uint32_t b) { return each * b + more * b / gridDim.x; };
    const int first = start_of(cost_at(blockIdx.x)), last = start_of(cost_at(blockIdx.x + 1));
    tiles = last - first;
    last_c = last / p->n_tiles;
    last_m = last - last_c * p->n_tiles;
    Task w;
    w.c = first / p->n_tiles;
    w.m0 = first - w.c * p->n_tiles;
    w.m = w.e = w.r0 = w.cnt = 0;
    if (tiles > 0) {
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
    const int rows = rows_of(*p, lo, &r), chunks = (rows + p->max_rows - 1) / p->max_rows, i = w.c - chunks_before[lo];
    const int each = rows / chunks, more = rows - each * chunks;   // even chunks
    w.r0 = r + each * i + (i < more ? i : more);
    w.cnt = each + (i < more ? 1 : 0);
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
// What a tile costs with this many rows of x, in sixths of the cost with 8.  All of 32 experts with 8, 16, 24 and
// 32 rows take, call after call, 93, 131, 167 and 202 us (4096 x 7168, groups of 128), 96, 137 and 177 us (groups
// of 64, which go by the same costs) and 71, 103 and 148 us (7168 x 2048, groups of 32; 25 to 32 rows are two chunks).
// 512 rows over the 32 experts as a router leaves them: 175 us with 6, 8, 11, 14 here, 165 us with these.
template <int G>
__device__ __forceinline__ int chunk_cost(int rows) {
  return rows <= 8 ? 6 : rows <= 16 ? (G == 32 ? 9 : 8) : rows <= 24 ? (G == 32 ? 12 : 10) : 12;
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
// The tiles of a task that a group of warps has: [own_first(m, group), own_first(m, group + 1)).
__device__ __forceinline__ int own_first(int m, int group) { return m * group / kGroupsM; }

// The ring between the copying warp and the warps that multiply.  Waits are bounded; when one gives up, no
// copy may be issued into a slot whose last one has not landed, and none may be under way when the CTA
// ends, since the shared memory is another CTA's then.  So a warp frees only slots that it has seen full
// (a slot counts as freed when all have), and the copying warp, whichever way its loop ended, stays until the
// others are through with all stages, or else until what it has issued has landed.  (It stays at a barrier:
// polling the stages instead, beside warps that multiply, took a row times 4096 x 7168 from 11.0 to 13.2 us.)
constexpr int kRingBarrier = 4;           // of the named barriers
template <unsigned long long LIMIT_NS>
struct Ring {
  uint64_t* full;             // [stages], one arrival (the copying warp's) and the bytes
  uint64_t* empty;            // [stages], kConsumers arrivals
  volatile int* abort_flag;   // set by the first wait that gives up
  int stages;

  // mbar_wait_bounded, with the clock left alone until a thousand polls have failed: reading it takes
  // longer than most waits here.
  static __device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, volatile int* flag) {
#pragma unroll 1
    for (int i = 0; i < 1024; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    return mbar_wait_bounded(bar, parity, flag, LIMIT_NS);
  }
  // Whole warps.  Has the slot's next stage come?
  __device__ __forceinline__ bool take(int slot, uint32_t parity) const {
    return __all_sync(0xffffffffu, wait_for(&full[slot], parity, abort_flag));
  }
  // The warp is done with a slot; `taken` is what take said of it.
  __device__ __forceinline__ void free_slot(int slot, bool taken) const {
    __syncwarp();
    if ((threadIdx.x & 31) == 0 && taken) mbar_arrive(&empty[slot]);
  }
  // The copying warp: may the slot be filled again?
  __device__ __forceinline__ bool reserve(int slot, uint32_t parity) const {
    return __all_sync(0xffffffffu, wait_for(&empty[slot], parity, abort_flag));
  }
  // A multiplying warp, after its last stage, taken or not.
  __device__ __forceinline__ void leave() const {
    __syncwarp();
    asm volatile("bar.arrive %0, %1;" ::"n"(kRingBarrier), "n"((kConsumers + 1) * 32) : "memory");
  }
  // The copying warp, at its end: have all of its `issued` stages landed?  Where no wait gave up they have been
  // taken; else the waits for them share one limit.
  __device__ __forceinline__ bool drain(int issued) const {
    __syncwarp();
    named_bar_sync(kRingBarrier, (kConsumers + 1) * 32);
    if (!*abort_flag) return true;
    bool landed = true;
    if ((threadIdx.x & 31) == 0) {
      volatile int gave_up = 0;
      for (int i = issued > stages ? issued - stages : 0; i < issued; ++i)
        landed &= wait_for(&full[i % stages], (uint32_t)(i / stages) & 1u, &gave_up);
    }
    return __all_sync(0xffffffffu, landed);
  }
};

// One step of a warp: M records of 128 columns, `m_stride` bytes apart, times NT * 8 rows of x.  The
// records are worked on side by side, so that M * NT chains of products are under way.
template <typename T, int NT, int M, int G, bool ZEROS>
__device__ __forceinline__ void multiply(const uint8_t* records, int m_stride, const uint8_t* x_stage, int kw,
                                         float (&sums)[kM][NT][4]) {
  constexpr int kParts = kStepK / G, kWords = 8 / kParts;   // groups of the step, words of a lane in each
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  float x_sum[NT][2][kParts];                      // -2^-24 * sums of x, rows 2t and 2t + 1
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const Pack<float, kParts> v = *reinterpret_cast<const Pack<float, kParts>*>(
          x_stage + (nt * 8 + 2 * t + i) * kRowPiece + kStageK * 2 + kw * kParts * 4);
#pragma unroll
      for (int part = 0; part < kParts; ++part) x_sum[nt][i][part] = v.v[part];
    }
  // Scales and zero points come for the whole step together: with groups of 32 a row of each of 32
  // experts of 7168 x 2048, with zero points, takes 77 us so and 81 with an access for each group.  With
  // groups of 64 it takes more registers than there are (32 experts of 4096 x 7168 x 24 rows: 189 us so,
  // 185 us group by group).
  constexpr bool kTogether = kParts != 2;
  Pack<uint32_t, kParts> scale[M];                 // of each group: row g's in the low half, row g + 8's
  uint32_t zero[M][(kParts + 1) / 2];              // two groups a word, a byte for each of the rows
#pragma unroll
  for (int m = 0; kTogether && m < M; ++m) {
    const uint8_t* tail = records + m * m_stride + 1024;
    scale[m] = *reinterpret_cast<const Pack<uint32_t, kParts>*>(tail + g * kParts * 4);
    if constexpr (ZEROS && kParts == 1) zero[m][0] = *reinterpret_cast<const uint16_t*>(tail + 32 + g * 2);
    if constexpr (ZEROS && kParts > 1) {
      using Words = Pack<uint32_t, kParts / 2>;
      const Words v = *reinterpret_cast<const Words*>(tail + kParts * 32 + g * kParts * 2);
#pragma unroll
      for (int i = 0; i < kParts / 2; ++i) zero[m][i] = v.v[i];
    }
  }
  float a[M][NT][4];
  uint4 x[NT][2], codes[M];
#pragma unroll
  for (int j = 0; j < 8; ++j) {                    // 16 columns each
    const int part = j / kWords;
    if (j % 4 == 0) {                              // half a record
#pragma unroll
      for (int m = 0; m < M; ++m)
        codes[m] = *reinterpret_cast<const uint4*>(records + m * m_stride + j / 4 * 512 + lane * 16);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          x[nt][h] = *reinterpret_cast<const uint4*>(x_stage + (nt * 8 + g) * kRowPiece +
                                                     (kw * kStepK + j / 4 * 64 + h * 32 + t * 8) * 2);
    }
    const bool first = j % kWords == 0;
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const uint32_t w = j % 4 == 0 ? codes[m].x : j % 4 == 1 ? codes[m].y : j % 4 == 2 ? codes[m].z : codes[m].w;
      const uint32_t w8 = w >> 8;
      const uint32_t a0 = w & 0x000f000fu, a1 = w & 0x00f000f0u, a2 = w8 & 0x000f000fu, a3 = w8 & 0x00f000f0u;
      // Zero points z as the numbers 2^23 + z and, for row g + 8 whose codes are 16 times theirs,
      // 2^27 + 16 * z: with -2^23 or -2^27 times the other factor added, an fma gives the product of z
      // alone, rounded once.
      float z0 = 0.f, z1 = 0.f;
      if (ZEROS && first) {
        if constexpr (!kTogether)
          if (part == 0) zero[m][0] = *reinterpret_cast<const uint32_t*>(records + m * m_stride + 1024 + kParts * 32 + g * 4);
        z0 = __uint_as_float(__byte_perm(zero[m][part / 2], 0x4b000000u, 0x7440 + part % 2 * 2));
        z1 = __uint_as_float(__byte_perm(zero[m][part / 2], 0x4d000000u, 0x7441 + part % 2 * 2));
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const uint4 v = x[nt][j % 4 >> 1];
        const uint32_t b0 = (j & 1) ? v.z : v.x, b1 = (j & 1) ? v.w : v.y;
        const float xs0 = x_sum[nt][0][part], xs1 = x_sum[nt][1][part];
        if (first && ZEROS)
          mma_f16(a[m][nt], a0, a1, a2, a3, b0, b1, fmaf(z0, xs0, -0x1p23f * xs0), fmaf(z0, xs1, -0x1p23f * xs1),
                  fmaf(z1, xs0, -0x1p27f * xs0), fmaf(z1, xs1, -0x1p27f * xs1));
        else if (first)
          mma_f16(a[m][nt], a0, a1, a2, a3, b0, b1, 8.f * xs0, 8.f * xs1, 128.f * xs0, 128.f * xs1);
        else
          mma_f16(a[m][nt], a0, a1, a2, a3, b0, b1, a[m][nt][0], a[m][nt][1], a[m][nt][2], a[m][nt][3]);
      }
    }
    if (j % kWords != kWords - 1) continue;
#pragma unroll
    for (int m = 0; m < M; ++m) {
      if constexpr (!kTogether)
        scale[m].v[part] = *reinterpret_cast<const uint32_t*>(records + m * m_stride + 1024 + (g * kParts + part) * 4);
      const float2 s = pair_of<T>(scale[m].v[part]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {              // rows g and g + 8; two rows of x in each fma
          const float2 sum = __ffma2_rn(make_float2(a[m][nt][2 * h], a[m][nt][2 * h + 1]),
                                        h ? make_float2(s.y, s.y) : make_float2(s.x, s.x),
                                        make_float2(sums[m][nt][2 * h], sums[m][nt][2 * h + 1]));
          sums[m][nt][2 * h] = sum.x;
          sums[m][nt][2 * h + 1] = sum.y;
        }
    }
  }
}

// Measured, 32 experts of 4096 x 7168 in groups of 128, rows for each, caches flushed before a call: 8 107 us
// (69% of the memory's rate), 16 139, 24 176, 32 211; call after call 93 (79%), 131, 167, 202.  Up to 8 rows memory and the copies' start bound it; beyond, the
// products do: an mma.sync holds a scheduler for 8 clocks (2.0 an SM, measured), and the 4 to 10 other
// instructions that each comes with (5 of them decode 8 codes for all rows) hardly overlap with it.
//
// A CTA of 8 warps that multiply (4 along the columns times 2 along the rows of tiles)
// and one that copies.  A stage of the ring holds 4 steps of columns of up to 8 rows of tiles
// and of up to 32 rows of x, about 60 KB in two or three copies (a copy for every
// row of tiles and of x made the copying warp the limit: 42 us of copies alone for 8
// matrices of 4096 x 7168, the memory's rate being 19 us).
template <typename T, int G, bool ZEROS>
__global__ void __launch_bounds__(kThreads, 1) w4_kernel(const W4Params p) {
  constexpr int kRecord = record_bytes(G, ZEROS);
  extern __shared__ __align__(128) uint8_t s_mem[];
  __shared__ int s_chunks[kMaxExperts + 1], s_cost[kMaxExperts + 1];
  __shared__ __align__(8) uint64_t s_full[kMaxStages], s_empty[kMaxStages];
  __shared__ volatile int s_abort;
  __shared__ int s_most_rows;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* s_sums = reinterpret_cast<float*>(s_mem + (kSmem - kSumBytes));

  // The kernel before this one, which has started, makes the rows of x; what came before
  // that one is complete, so the offsets and weights may be read.
  if (threadIdx.x < kMaxStages) {
    mbar_init(&s_full[threadIdx.x], 1);
    mbar_init(&s_empty[threadIdx.x], kConsumers);
    fence_mbar_init();
  }
  if (threadIdx.x == 0) {
    s_abort = 0;
    s_most_rows = 0;
  }
  __syncthreads();
  // Chunks of up to max_rows rows before expert e: the same in every CTA.
  for (int e = threadIdx.x; e < p.E; e += kThreads) {
    int first;
    const int rows = Tasks::rows_of(p, e, &first), chunks = (rows + p.max_rows - 1) / p.max_rows;
    s_chunks[e] = chunks;
    if (chunks) atomicMax(&s_most_rows, (rows + chunks - 1) / chunks);
    s_cost[e] = chunks ? chunks * chunk_cost<G>((rows + chunks - 1) / chunks) : 0;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    int sum = 0, cost_sum = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int e = e0 + lane, v = e < p.E ? s_chunks[e] : 0, cost = e < p.E ? s_cost[e] : 0;
      int incl = v, cost_incl = cost;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, incl, off), oc = __shfl_up_sync(0xffffffffu, cost_incl, off);
        if (lane >= off) {
          incl += o;
          cost_incl += oc;
        }
      }
      if (e < p.E) {
        s_chunks[e] = sum + incl - v;
        s_cost[e] = cost_sum + cost_incl - cost;
      }
      sum += __shfl_sync(0xffffffffu, incl, 31);
      cost_sum += __shfl_sync(0xffffffffu, cost_incl, 31);
    }
    if (lane == 0) {
      s_chunks[p.E] = sum;
      s_cost[p.E] = cost_sum;
    }
  }
  __syncthreads();
  Tasks tasks;
  tasks.p = &p;
  tasks.chunks_before = s_chunks;
  tasks.cost_before = s_cost;
  Task work = tasks.begin();
  // Stages of the ring are as large as this CTA's tasks can need, and as many as fit: where a
  // CTA has one or two rows of tiles, all of their columns can be on their way at once.
  const int weights_bytes = tasks.most() * kSplit * kRecord, stage_bytes = weights_bytes + s_most_rows * kRowPiece;
  const int fit = (int)(kSmem - kSumBytes) / (stage_bytes > 0 ? stage_bytes : 1);
  const int stages = fit < kMaxStages ? fit : kMaxStages;
  const Ring<kWaitLimitNs> ring = {s_full, s_empty, &s_abort, stages};

  if (warp >= kConsumers) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegisters));
    if (warp > kConsumers) return;
    // ---- copies
    // Lane 0 and, where a task's tiles lie in two groups of 8, lane 1 copy the weights.
    struct Source {
      const uint8_t* at;      // this lane's records of the stage
      int m, step, tiles, skip, dst;
    };
    auto source_of = [&](const Task& w) {
      Source src;
      const int in_first = kTaskM - w.m0 % kTaskM < w.m ? kTaskM - w.m0 % kTaskM : w.m;
      const int at = (w.m0 / kTaskM + (lane & 1)) * kTaskM;
      src.m = lane == 0 ? in_first : lane == 1 ? w.m - in_first : 0;
      src.tiles = p.n_tiles - at < kTaskM ? p.n_tiles - at : kTaskM;
      src.at = p.records + ((size_t)w.e * p.n_tiles + at) * p.k_steps * kRecord;
      src.step = src.tiles * kSplit * kRecord;
      src.skip = lane == 0 ? w.m0 % kTaskM : 0;      // tiles of the group before the task's
      src.dst = lane == 0 ? 0 : in_first;            // tiles of the task before this lane's
      return src;
    };
    auto copy_weights = [&](const Task& w, Source& src, int stage, int slot) {
      const int left = p.k_steps - stage * kSplit, bytes = (left < kSplit ? left : kSplit) * kRecord;
      if (lane == 0) mbar_arrive_expect_tx(&s_full[slot], w.m * bytes + w.cnt * kRowPiece);
      __syncwarp();
      if (src.m > 0)
        bulk_copy(smem_u32(s_mem + slot * stage_bytes + src.dst * bytes), src.at + src.skip * bytes, src.m * bytes,
                  &s_full[slot]);
      src.at += src.step;
    };
    auto copy_rows = [&](const Task& w, int stage, int slot) {
      if (lane == 2)
        bulk_copy(smem_u32(s_mem + slot * stage_bytes + weights_bytes), p.x + ((size_t)stage * p.R + w.r0) * kRowPiece,
                  w.cnt * kRowPiece, &s_full[slot]);
    };
    auto step_on = [&](Task& w, int& stage) {
      if (++stage < p.stages) return false;
      stage = 0;
      tasks.next(w);
      return true;
    };
    // The weights of the first stages do not wait for the rows of x.
    Task w = work;
    Source src = source_of(w);
    int stage = 0, issued = 0;
    for (; issued < kEarly && issued < stages && w.m; ++issued) {
      copy_weights(w, src, stage, issued);
      if (step_on(w, stage)) src = source_of(w);
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
    int slot = issued == stages ? 0 : issued;
    uint32_t parity = issued == stages ? 0 : 1;    // a fresh slot counts as freed
    bool ok = true;
    for (; w.m; ++issued) {
      ok = ring.reserve(slot, parity);
      if (!ok) break;
      copy_weights(w, src, stage, slot);
      copy_rows(w, stage, slot);
      if (step_on(w, stage)) src = source_of(w);
      if (++slot == stages) { slot = 0; parity ^= 1; }
    }
    ok &= ring.drain(issued);
    if (!ok && lane == 0) raise_error(&g_w4_error, kDevTimeoutProducer);
    return;
  }

  // ---- products
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegisters));
  griddep_wait();                                  // row_exp
  griddep_launch_dependents();
  const int kw = warp % kSplit, mg = warp / kSplit, g = lane >> 2, t = lane & 3;
  // With few tiles the groups of warps take turns at the stages instead of sharing out the tiles:
  // one row of x and a matrix of 4096 x 7168, replayed call after call, 12.3 -> 11.0 us, 32 rows and 2048 x 7168
  // 17.3 -> 15.9 us.
  const bool turns = tasks.most() <= kM;
  const int parties = turns ? kConsumers * 32 : kSplit * 32;   // threads that add up the same sums
  int buffer = 0;
  int slot = 0;
  uint32_t parity = 0;
  bool ok = true;                                  // after a wait that gave up: go on without work
  auto run = [&](const Task& w, auto nt_tag) {
    constexpr int NT = decltype(nt_tag)::value;
    const int m_first = turns ? 0 : own_first(w.m, mg), m_here = (turns ? w.m : own_first(w.m, mg + 1)) - m_first;
    float sums[kM][NT][4];
#pragma unroll
    for (int m = 0; m < kM; ++m)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[m][nt][i] = 0.f;
#pragma unroll 1
    for (int stage = 0; stage < p.stages; ++stage) {
      if (ok) ok = ring.take(slot, parity);
      const uint8_t* at = s_mem + slot * stage_bytes;
      const int left = p.k_steps - stage * kSplit, stride = (left < kSplit ? left : kSplit) * kRecord;
      if (ok && kw < left && (!turns || stage % kGroupsM == mg)) {
        const uint8_t* records = at + m_first * stride + kw * kRecord;
        const uint8_t* x = at + weights_bytes;
        if (m_here == kM) multiply<T, NT, kM, G, ZEROS>(records, stride, x, kw, sums);
        else if (m_here == 1) multiply<T, NT, 1, G, ZEROS>(records, stride, x, kw, sums);
        else if (kM > 2 && m_here == 2) multiply<T, NT, 2, G, ZEROS>(records, stride, x, kw, sums);
        else if (kM > 3 && m_here == 3) multiply<T, NT, 3, G, ZEROS>(records, stride, x, kw, sums);
      }
      ring.free_slot(slot, ok);
      if (++slot == stages) { slot = 0; parity ^= 1; }
    }
    // The sums of the warps that share tiles (a group, or all when they take turns) meet in shared
    // memory and are added in the columns' order, 8 rows of x at a time.  A group waits for no
    // other, so one adds up while another multiplies, and as the rounds take two buffers in turn, one
    // barrier each is enough: who writes a buffer again has passed the barrier between, and by then
    // all had read it.  (One buffer and all warps at both barriers: 2 to 9% more time.)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float* mine = s_sums + buffer * kSumFloats + warp * (8 * kSumStride);
#pragma unroll
      for (int m = 0; m < kM; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          mine[(2 * t + (i & 1)) * kSumStride + m * 16 + g + 8 * (i >> 1)] = sums[m][nt][i];
      named_bar_sync(turns ? 1 : 2 + mg, parties);
      const float* theirs = s_sums + buffer * kSumFloats + (turns ? 0 : mg * kSplit) * (8 * kSumStride);
      buffer ^= 1;
      for (int i = (int)threadIdx.x % parties; i < kGroupSums; i += parties) {
        const int n = i % (kM * 16), row = i / (kM * 16), tile = n / 16, in = nt * 8 + row;
        const int col = (w.m0 + m_first + tile) * 16 + n % 16;
        if (tile >= m_here || in >= w.cnt || col >= p.N) continue;
        const int up = (n & 8 ? 20 : 24) + __ldg(p.row_exp + w.r0 + in);   // rows g + 8 were 16 times theirs
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < kSplit; ++q) v += theirs[(q * 8 + row) * kSumStride + n];
        if (turns) {                               // what the other groups have of the same tiles
#pragma unroll
          for (int q = kSplit; q < kConsumers; ++q) v += theirs[(q * 8 + row) * kSumStride + n];
        }
        // v * 2^up, -100 <= up <= 138, in two factors of the same direction: no infinity on the way to a
        // finite product, no rounding on the way to a normal one
        v = v * power_of_two(up >> 1) * power_of_two(up - (up >> 1));
        const size_t to = (size_t)(w.r0 + in) * p.N + col;
        if (p.out_f32) static_cast<float*>(p.y)[to] = v;
        else static_cast<T*>(p.y)[to] = from_float<T>(v);
      }
    }
  };
  for (; work.m; tasks.next(work)) {
    if (work.cnt <= 8) run(work, std::integral_constant<int, 1>{});
    else if (work.cnt <= 16) run(work, std::integral_constant<int, 2>{});
    else if (work.cnt <= 24) run(work, std::integral_constant<int, 3>{});
    else if constexpr (max_rows(G) > 24) run(work, std::integral_constant<int, 4>{});
  }
  ring.leave();
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

// Self-test of the ring's failure path: the product's ring with waits of a few ms, four slots of 1 KB and
// `issues` stages, of which the copying warp issues all copies but number `missing`, so that the waits for
// that one run out.  report: [0] stages issued, [1] the fewest stages that a multiplying warp took, [2] wrong words
// in what was taken, [3] whether reserve ran out, [4] whether drain found a copy missing, [5] how many of the
// last four stages had landed when the copying warp left.
constexpr int kTestSlots = 4, kTestBytes = 1024;
__global__ void __launch_bounds__((kConsumers + 1) * 32)
w4_selftest_ring_kernel(const uint32_t* __restrict__ src, int issues, int missing, int* __restrict__ report) {
  __shared__ __align__(128) uint32_t s_slots[kTestSlots][kTestBytes / 4];
  __shared__ __align__(8) uint64_t s_full[kTestSlots], s_empty[kTestSlots];
  __shared__ volatile int s_abort;
  __shared__ int s_taken, s_wrong;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Ring<2000000> ring = {s_full, s_empty, &s_abort, kTestSlots};
  if (threadIdx.x < kTestSlots) {
    mbar_init(&s_full[threadIdx.x], 1);
    mbar_init(&s_empty[threadIdx.x], kConsumers);
    fence_mbar_init();
  }
  if (threadIdx.x == 0) {
    s_abort = 0;
    s_taken = issues;
    s_wrong = 0;
  }
  __syncthreads();
  if (warp == kConsumers) {
    bool ok = true;
    int issued = 0;
    for (; issued < issues; ++issued) {
      const int slot = issued % kTestSlots;
      ok = ring.reserve(slot, (uint32_t)(issued / kTestSlots + 1) & 1u);
      if (!ok) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(&s_full[slot], kTestBytes);
        if (issued != missing) bulk_copy(smem_u32(s_slots[slot]), src + issued * (kTestBytes / 4), kTestBytes, &s_full[slot]);
      }
      __syncwarp();
    }
    const bool landed = ring.drain(issued);
    if (lane == 0) {
      int there = 0;
      for (int i = issued > kTestSlots ? issued - kTestSlots : 0; i < issued; ++i)
        there += mbar_try_wait(&s_full[i % kTestSlots], (uint32_t)(i / kTestSlots) & 1u);
      report[0] = issued;
      report[3] = !ok;
      report[4] = !landed;
      report[5] = there;
    }
  } else {
    bool ok = true;
    for (int i = 0; i < issues; ++i) {
      const int slot = i % kTestSlots;
      if (ok && !(ok = ring.take(slot, (uint32_t)(i / kTestSlots) & 1u)) && lane == 0) atomicMin(&s_taken, i);
      if (ok)
        for (int k = lane; k < kTestBytes / 4; k += 32)
          if (s_slots[slot][k] != __ldg(src + i * (kTestBytes / 4) + k)) atomicAdd(&s_wrong, 1);
      ring.free_slot(slot, ok);
    }
    ring.leave();
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    report[1] = s_taken;
    report[2] = s_wrong;
    if (s_taken < issues) raise_error(&g_w4_error, kDevTimeoutMma);
  }
}

// Workspace: the rows of x by stages, then their exponents.
int stages_of(int64_t d) { return (int)((d + kStageK - 1) / kStageK); }
uint64_t rows_bytes(int64_t R, int64_t d) { return (uint64_t)R * stages_of(d) * kRowPiece; }

template <typename T, int G, bool ZEROS>
int launch_w4(const W4Params& p, const void* x, int d, int sms, cudaStream_t s) {
  static_assert(2 * (kTaskM * kSplit * record_bytes(G, ZEROS) + max_rows(G) * kRowPiece) + kSumBytes <= kSmem,
                "two stages");
  static std::atomic<void*> seen[kMaxCachedDevices];
  cudaError_t e = once_per_context(seen, [] {
    w4_launched(true);
    return cudaFuncSetAttribute(w4_kernel<T, G, ZEROS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem);
  });
  if (e != cudaSuccess) return cuda_status(e);
  e = launch_pdl(w4_rows_kernel<T, G>, dim3(p.R), dim3(kRowsThreads), 0, s, static_cast<const T*>(x),
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
  W4Params p;
  p.R = num_rows; p.N = n; p.E = num_experts;
  p.n_tiles = (n + 15) / 16;
  p.k_steps = (d + kStepK - 1) / kStepK;
  p.stages = stages_of(d);
  // whatever the offsets, (chunk, row of tiles) pairs and the chunks' costs (chunk_cost, at
  // most 16) are numbered in 32 bits
  p.max_rows = max_rows(group_size);
  const int64_t most_chunks = (int64_t)num_experts * (((int64_t)num_rows + p.max_rows - 1) / p.max_rows);
  if (most_chunks * (p.n_tiles > 16 ? p.n_tiles : 16) > INT32_MAX) return MOE_ERR_TOO_LARGE;
  int sms = 0;
  if ((st = require_device(&sms)) != MOE_OK) return st;
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

MOE_API int moe_w4_selftest_ring(const void* src, int32_t issues, int32_t missing, int32_t* report, void* stream) {
  if (!src || !report || issues < 0 || issues > 4096 || missing < 0) return MOE_ERR_INVALID_ARGUMENT;
  if (!aligned_to(src, 16) || !aligned_to(report, 4)) return MOE_ERR_MISALIGNED;
  const int st = require_device(nullptr);
  if (st != MOE_OK) return st;
  w4_launched(true);
  w4_selftest_ring_kernel<<<1, (kConsumers + 1) * 32, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint32_t*>(src), issues, missing, report);
  return cuda_status(cudaGetLastError());
}

MOE_API int moe_w4_read_device_error(void* stream, int32_t* device_error) {
  if (!device_error) return MOE_ERR_INVALID_ARGUMENT;
  *device_error = 0;
  if (!w4_launched(false)) return MOE_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  static std::mutex one_reader;                    // g_w4_taken is its own until it has been copied
  std::lock_guard<std::mutex> lock(one_reader);
  int32_t v = 0;
  w4_take_error_kernel<<<1, 1, 0, s>>>();
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) e = cudaMemcpyFromSymbolAsync(&v, g_w4_taken, 4, 0, cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e != cudaSuccess) return cuda_status(e);
  *device_error = v;
  return v ? MOE_ERR_DEVICE_TIMEOUT : MOE_OK;
}

}  // extern "C"
