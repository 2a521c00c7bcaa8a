// Tokens sorted by expert and back: sort, dispatch (with its gradient) and
// weighted combine (with its gradients) for rows of any width and for fp32,
// fp16 and bf16.  The fused layer has these steps inside its own launches, on
// its own types and sizes (route_permute.cu).
//
// Pairs p = t * K + k are numbered over tokens and picks.  key(p) = id - first
// when the expert is on this shard, else E.  A stable counting sort by key gives
// every pair one of the T * K rows:
//   row(p) = #{q : key(q) < key(p)} + #{q < p : key(q) = key(p)}
// Rows of pairs that are not on the shard come last; inv_row holds -1 - row for
// them, so each output row is written by exactly one pair (the others' rows with
// zeros) and no pass has to clear a buffer first.
#include <cooperative_groups.h>

#include "rows.cuh"

namespace moe {
namespace {

namespace cg = cooperative_groups;

constexpr int kSortMaxExperts = 1024;
constexpr int kSortCluster = 8;

// --------------------------------------------------------------------------
// Sort: one launch of one cluster.  A few integers for each pair go in and out
// (12 bytes), so latency bounds it, not bandwidth: one launch with the counters
// in shared memory, instead of a histogram, a scan and a scatter launch with
// counters in global memory.  Each warp owns a run of consecutive pairs and one
// row of counters, so no order depends on atomics: counts per warp, then sums over
// warps, CTAs (distributed shared memory) and experts, then each warp walks its
// run again and hands out rows in order.
// --------------------------------------------------------------------------
__global__ void __launch_bounds__(1024)
sort_kernel(const int32_t* __restrict__ ids, int P, int K, int E, int first, int run,
            int32_t* __restrict__ offsets, int32_t* __restrict__ inv_row, int32_t* __restrict__ row_token) {
  extern __shared__ int s_mem[];
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int keys = E + 1;
  int* s_hist = s_mem;                        // [warps][keys]: counts, then next rows
  int* s_total = s_mem + (size_t)warps * keys;   // [keys]: this CTA's counts
  int* s_start = s_total + keys;              // [keys]: first row of each key
  int* s_before = s_start + keys;             // [keys]: counts of the CTAs before this one
  __shared__ int s_warp[32];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks();
  griddep_wait();
  griddep_launch_dependents();
  for (int i = threadIdx.x; i < warps * keys; i += blockDim.x) s_hist[i] = 0;
  __syncthreads();
  const int64_t begin64 = ((int64_t)rank * warps + warp) * run;
  const int begin = begin64 < P ? (int)begin64 : P;
  const int end = P - begin < run ? P : begin + run;
  int* mine = s_hist + (size_t)warp * keys;
  auto key_of = [&](int p) {
    const unsigned local = (unsigned)__ldg(ids + p) - (unsigned)first;   // wraps far above E when below first
    return local < (unsigned)E ? (int)local : E;
  };
  constexpr int kTogether = 4;                // ids on their way at a time
  for (int p0 = begin + lane; p0 < end; p0 += 32 * kTogether) {
    int key[kTogether];
#pragma unroll
    for (int i = 0; i < kTogether; ++i) key[i] = p0 + 32 * i < end ? key_of(p0 + 32 * i) : -1;
#pragma unroll
    for (int i = 0; i < kTogether; ++i)
      if (key[i] >= 0) atomicAdd(mine + key[i], 1);
  }
  __syncthreads();
  // Counts to offsets among this CTA's warps: 4 threads a key, a quarter of the warps each.
  for (int i = threadIdx.x; i < 4 * ((keys + 7) / 8 * 8); i += blockDim.x) {   // whole warps
    const int e = i >> 2, quarter = warps / 4, w0 = (i & 3) * quarter;
    int sum = 0;
    if (e < keys)
#pragma unroll 8
      for (int w = w0; w < w0 + quarter; ++w) {
        const int c = s_hist[w * keys + e];
        s_hist[w * keys + e] = sum;
        sum += c;
      }
    int incl = sum;
#pragma unroll
    for (int off = 1; off < 4; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, incl, off, 4);
      if ((i & 3) >= off) incl += o;
    }
    if (e < keys) {
      for (int w = w0; w < w0 + quarter; ++w) s_hist[w * keys + e] += incl - sum;
      if ((i & 3) == 3) s_total[e] = incl;
    }
  }
  if (ctas > 1) cluster.sync(); else __syncthreads();
  // Offsets among the CTAs and, warp by warp, among the keys.
  int carry = 0;                                           // of the keys of earlier rounds
  for (int e0 = 0; e0 < keys; e0 += blockDim.x) {
    const int e = e0 + (int)threadIdx.x;
    int before = 0, all = 0;
    if (e < keys)
#pragma unroll
      for (int c = 0; c < kSortCluster; ++c) {
        if (c >= ctas) break;
        const int v = ctas > 1 ? cluster.map_shared_rank(s_total, c)[e] : s_total[e];
        if (c < rank) before += v;
        all += v;
      }
    int incl = all;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += o;
    }
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    int base = carry;
    for (int w = 0; w < warps; ++w) {
      const int v = s_warp[w];
      if (w < warp) base += v;
      carry += v;
    }
    if (e < keys) {
      s_start[e] = base + incl - all;
      s_before[e] = before;
    }
    __syncthreads();
  }
  if (rank == 0)
    for (int e = threadIdx.x; e < keys; e += blockDim.x) offsets[e] = s_start[e];
  const int tail = s_start[E];
  for (int p0 = begin; p0 < end; p0 += 32 * kTogether) {
    int key[kTogether];
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      const int p = p0 + 32 * i + lane;
      key[i] = p < end ? key_of(p) : -1;
    }
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      const int p = p0 + 32 * i + lane;
      const unsigned same = __match_any_sync(0xffffffffu, key[i]);
      int* next = mine + (key[i] < 0 ? 0 : key[i]);
      const int at = *next;
      __syncwarp();
      if (key[i] >= 0) {
        const int row = s_start[key[i]] + s_before[key[i]] + at + __popc(same & ((1u << lane) - 1u));
        inv_row[p] = key[i] < E ? row : -1 - row;
        row_token[row] = row < tail ? p / K : -1;
        if (lane == __ffs(same) - 1) *next = at + __popc(same);
      }
      __syncwarp();
    }
  }
  if (ctas > 1) cluster.sync();   // no CTA leaves while another still reads its counts
}

// A CTA's threads cover `tx` consecutive vectors of blockDim.x / tx tokens.
struct Place {
  int t, v;   // token, vector of the row
};
__device__ __forceinline__ Place place_of(int chunks, int tx) {
  const int ty = (int)blockDim.x / tx;
  const int block_t = (int)blockIdx.x / chunks;
  return {block_t * ty + (int)threadIdx.x / tx, ((int)blockIdx.x - block_t * chunks) * tx + (int)threadIdx.x % tx};
}

// --------------------------------------------------------------------------
// Dispatch: each thread reads one vector of a token once and writes it to the
// token's K rows.  Bound by memory: T reads and T * K writes of a row.
// --------------------------------------------------------------------------
template <typename W>
__global__ void __launch_bounds__(256)
dispatch_kernel(const W* __restrict__ hidden, const int32_t* __restrict__ inv_row, int T, int K, int nvec,
                int chunks, int tx, W* __restrict__ rows) {
  griddep_wait();
  griddep_launch_dependents();
  const Place at = place_of(chunks, tx);
  if (at.t >= T || at.v >= nvec) return;
  const W x = __ldcs(hidden + (size_t)at.t * nvec + at.v);
  const W zero = {};
  const int32_t* inv = inv_row + (size_t)at.t * K;
  const unsigned R = (unsigned)(T * K);
#pragma unroll 8
  for (int k = 0; k < K; ++k) {
    const int r = __ldg(inv + k);
    const unsigned row = r >= 0 ? r : -1 - r;
    if (row < R) rows[(size_t)row * nvec + at.v] = r >= 0 ? x : zero;
  }
}

// --------------------------------------------------------------------------
// Combine: out[t] = sum_k w[t,k] * rows[inv_row[t,k]], in fp32, k ascending, one
// rounding.  WEIGHTED = false is dispatch's gradient (all weights 1).  Bound
// by memory: T * K reads and T writes of a row; eight row loads are in flight in
// each thread before the first is used.
// --------------------------------------------------------------------------
constexpr int kBatch = 8;   // picks of one token whose rows are loaded together

template <typename TRow, typename TOut, int N, bool WEIGHTED>
__global__ void __launch_bounds__(256)
combine_rows_kernel(const TRow* __restrict__ rows, const int32_t* __restrict__ inv_row,
                    const float* __restrict__ weights, int T, int K, int nvec, int chunks, int tx,
                    TOut* __restrict__ out) {
  griddep_wait();
  griddep_launch_dependents();
  const Place at = place_of(chunks, tx);
  if (at.t >= T || at.v >= nvec) return;
  const size_t H = (size_t)nvec * N;
  const unsigned R = (unsigned)(T * K);
  float acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  for (int k0 = 0; k0 < K; k0 += kBatch) {
    Pack<TRow, N> x[kBatch];
    float w[kBatch];
    bool here[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int k = k0 + j;
      const int r = k < K ? __ldg(inv_row + (size_t)at.t * K + k) : -1;
      here[j] = (unsigned)r < R;
      if (WEIGHTED) w[j] = k < K ? __ldg(weights + (size_t)at.t * K + k) : 0.f;
      if (here[j]) x[j] = load_stream<TRow, N>(rows + (size_t)r * H + (size_t)at.v * N);
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (!here[j]) continue;
#pragma unroll
      for (int i = 0; i < N; ++i)
        acc[i] = WEIGHTED ? fmaf(w[j], to_float(x[j].v[i]), acc[i]) : acc[i] + to_float(x[j].v[i]);
    }
  }
  Pack<TOut, N> o;
#pragma unroll
  for (int i = 0; i < N; ++i) o.v[i] = from_float<TOut>(acc[i]);
  store_wide<TOut, N>(out + (size_t)at.t * H + (size_t)at.v * N, o);
}

// --------------------------------------------------------------------------
// Combine's gradients: grad_rows[inv_row[t,k]] = w[t,k] * g[t] and
// grad_weights[t,k] = <g[t], rows[inv_row[t,k]]>, in one pass: GS threads share a
// token, hold a vector of g in registers and go over the token's K rows.  The
// dot products are added in a fixed order (a thread's vectors, then a tree over
// the GS threads).  Bound by memory: T + T * K reads and T * K writes of a row.
// --------------------------------------------------------------------------
template <typename TRow, typename TOut, int N, int GS>
__global__ void __launch_bounds__(GS < 128 ? 128 : GS)
combine_backward_kernel(const TOut* __restrict__ grad_out, const TRow* __restrict__ rows,
                        const int32_t* __restrict__ inv_row, const float* __restrict__ weights, int T, int K,
                        int nvec, TRow* __restrict__ grad_rows, float* __restrict__ grad_weights) {
  constexpr int kGroups = GS < 128 ? 128 / GS : 1;
  constexpr int kWarps = GS / 32;
  __shared__ float s_dot[kWarps > 1 ? kWarps : 1][kBatch];
  griddep_wait();
  griddep_launch_dependents();
  const int t = (int)blockIdx.x * kGroups + (int)threadIdx.x / GS, lane = (int)threadIdx.x % GS;
  if (t >= T) return;                       // whole groups leave, and only where a group is a warp
  const size_t H = (size_t)nvec * N;
  const unsigned R = (unsigned)(T * K);
  for (int k0 = 0; k0 < K; k0 += kBatch) {
    int r[kBatch];
    float w[kBatch], dot[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int k = k0 + j;
      r[j] = k < K ? __ldg(inv_row + (size_t)t * K + k) : INT_MIN;
      w[j] = k < K ? __ldg(weights + (size_t)t * K + k) : 0.f;
      dot[j] = 0.f;
    }
    for (int v = lane; v < nvec; v += GS) {
      const size_t col = (size_t)v * N;
      const Pack<TOut, N> g = K <= kBatch ? load_stream<TOut, N>(grad_out + (size_t)t * H + col)
                                          : load_cached<TOut, N>(grad_out + (size_t)t * H + col);
      Pack<TRow, N> x[kBatch];
      if (grad_weights) {
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
          if ((unsigned)r[j] < R) x[j] = load_stream<TRow, N>(rows + (size_t)r[j] * H + col);
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        if (grad_weights && (unsigned)r[j] < R) {
#pragma unroll
          for (int i = 0; i < N; ++i) dot[j] = fmaf(to_float(g.v[i]), to_float(x[j].v[i]), dot[j]);
        }
        if (grad_rows) {
          const unsigned row = r[j] >= 0 ? r[j] : -1 - r[j];
          if (row >= R) continue;
          Pack<TRow, N> o = zero_pack<TRow, N>();
          if (r[j] >= 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) o.v[i] = from_float<TRow>(w[j] * to_float(g.v[i]));
          }
          store_wide<TRow, N>(grad_rows + (size_t)row * H + col, o);
        }
      }
    }
    if (!grad_weights) continue;
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
#pragma unroll
      for (int off = 16; off; off >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], off);
    if (kWarps == 1) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (lane == j && k0 + j < K) grad_weights[(size_t)t * K + k0 + j] = dot[j];
    } else {
      const int warp = lane >> 5;
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if ((lane & 31) == j) s_dot[warp][j] = dot[j];
      __syncthreads();
      if (lane < kBatch && k0 + lane < K) {
        float sum = 0.f;
#pragma unroll
        for (int q = 0; q < kWarps; ++q) sum += s_dot[q][lane];
        grad_weights[(size_t)t * K + k0 + lane] = sum;
      }
      __syncthreads();
    }
  }
}

// --------------------------------------------------------------------------
// The two kernels above for rows of whole 16-byte pieces and at most 8 picks, where
// bandwidth counts.  With the rows in registers a thread needs 100 to 180 of them and too
// few threads fit to cover the memory's latency (4096 tokens x 8 x 7168 bf16: combine 127,
// its gradients 215 us; with these 84 us, 6.3 TB/s, and 161 us, 6.2 TB/s, call after call).  Here every
// thread copies its own pieces of the next tokens asynchronously into its own places in
// shared memory, two steps ahead of the sums: no registers, no barrier, and twice 256
// threads x 2 steps x 128 bytes on their way on an SM.  More than 8 picks stay with the
// kernels above (2048 tokens x 16 x 7168 bf16: 94 and 200 us, memory's floor 76 and 148;
// 3640 x 9 x 7168, a second batch for one pick: 149 and 270, floor 80 and 151).
// --------------------------------------------------------------------------
constexpr int kStreamThreads = 256, kSteps = 3;   // places for 3 steps: 2 ahead

template <typename TRow, typename TOut, bool WEIGHTED>
__global__ void __launch_bounds__(kStreamThreads, 2)
combine_stream_kernel(const TRow* __restrict__ rows, const int32_t* __restrict__ inv_row,
                      const float* __restrict__ weights, int T, int K, int nvec, TOut* __restrict__ out) {
  constexpr int N = 16 / (int)sizeof(TRow);
  extern __shared__ uint4 s_place[];               // [kSteps][kBatch][kStreamThreads]
  griddep_wait();
  griddep_launch_dependents();
  const size_t H = (size_t)nvec * N;
  const unsigned R = (unsigned)(T * K);
  // Pieces (token, vector) are numbered through; a thread takes every stride-th.
  const int stride = (int)gridDim.x * kStreamThreads, skip_t = stride / nvec, skip_v = stride - skip_t * nvec;
  struct At {
    int t, v;
  };
  auto next = [&](At& at) {
    at.t += skip_t;
    at.v += skip_v;
    if (at.v >= nvec) {
      at.v -= nvec;
      ++at.t;
    }
  };
  const int start = (int)blockIdx.x * kStreamThreads + (int)threadIdx.x;
  At ahead = {start / nvec, start - start / nvec * nvec}, at = ahead;
  int r[kBatch];                                   // of the next piece to copy
  auto look_up = [&]() {
#pragma unroll
    for (int j = 0; j < kBatch; ++j) r[j] = ahead.t < T && j < K ? __ldg(inv_row + (size_t)ahead.t * K + j) : -1;
  };
  unsigned here[kSteps];                           // which picks' pieces are in a place
  auto copy = [&](int place) {
    here[place] = 0;
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if ((unsigned)r[j] < R) {
        copy16(&s_place[(place * kBatch + j) * kStreamThreads + threadIdx.x], rows + (size_t)r[j] * H + (size_t)ahead.v * N);
        here[place] |= 1u << j;
      }
    copies_commit();
    next(ahead);
    look_up();
  };
  look_up();
#pragma unroll
  for (int i = 0; i < kSteps - 1; ++i) copy(i);
  while (at.t < T) {
#pragma unroll
    for (int place = 0; place < kSteps; ++place) {
      copy((place + kSteps - 1) % kSteps);
      if (at.t < T) {
        float w[kBatch];
        if (WEIGHTED) {
#pragma unroll
          for (int j = 0; j < kBatch; ++j) w[j] = j < K ? __ldg(weights + (size_t)at.t * K + j) : 0.f;
        }
        copies_wait<kSteps - 1>();
        float acc[N];
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = 0.f;
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          if (!(here[place] >> j & 1)) continue;
          const uint4 raw = s_place[(place * kBatch + j) * kStreamThreads + threadIdx.x];
          const Pack<TRow, N>& x = reinterpret_cast<const Pack<TRow, N>&>(raw);
#pragma unroll
          for (int i = 0; i < N; ++i)
            acc[i] = WEIGHTED ? fmaf(w[j], to_float(x.v[i]), acc[i]) : acc[i] + to_float(x.v[i]);
        }
        Pack<TOut, N> o;
#pragma unroll
        for (int i = 0; i < N; ++i) o.v[i] = from_float<TOut>(acc[i]);
        store_wide<TOut, N>(out + (size_t)at.t * H + (size_t)at.v * N, o);
      }
      next(at);
    }
  }
  copies_wait<0>();
}

// GS threads share a token and go over its vectors in steps.
template <typename TRow, typename TOut, int GS>
__global__ void __launch_bounds__(kStreamThreads, 2)
combine_backward_stream_kernel(const TOut* __restrict__ grad_out, const TRow* __restrict__ rows,
                               const int32_t* __restrict__ inv_row, const float* __restrict__ weights, int T, int K,
                               int nvec, TRow* __restrict__ grad_rows, float* __restrict__ grad_weights) {
  constexpr int N = 16 / (int)sizeof(TRow), kWarps = GS / 32, kGroups = kStreamThreads / GS;
  extern __shared__ uint4 s_place[];               // [kSteps][kBatch][kStreamThreads]
  __shared__ float s_dot[kGroups][kWarps][kBatch];
  griddep_wait();
  griddep_launch_dependents();
  const size_t H = (size_t)nvec * N;
  const unsigned R = (unsigned)(T * K);
  const int group = (int)threadIdx.x / GS, lane = (int)threadIdx.x % GS;
  const int first = (int)blockIdx.x * kGroups + group, stride = (int)gridDim.x * kGroups;
  const int steps = (nvec + GS - 1) / GS;
  struct At {
    int t, step;
  };
  auto next = [&](At& at) {
    if (++at.step < steps) return false;
    at.step = 0;
    at.t += stride;
    return true;
  };
  At ahead = {first, 0}, at = ahead;
  int r_ahead[kBatch], r[kBatch];
  auto look_up = [&](int t, int (&rr)[kBatch]) {
#pragma unroll
    for (int j = 0; j < kBatch; ++j) rr[j] = t < T && j < K ? __ldg(inv_row + (size_t)t * K + j) : INT_MIN;
  };
  Pack<TOut, N> g[kSteps];
  auto copy = [&](int place) {
    const int v = ahead.step * GS + lane;
    if (ahead.t < T && v < nvec) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if ((unsigned)r_ahead[j] < R)
          copy16(&s_place[(place * kBatch + j) * kStreamThreads + threadIdx.x],
                 rows + (size_t)r_ahead[j] * H + (size_t)v * N);
      g[place] = load_stream<TOut, N>(grad_out + (size_t)ahead.t * H + (size_t)v * N);
    }
    copies_commit();
    if (next(ahead)) look_up(ahead.t, r_ahead);
  };
  look_up(first, r_ahead);
  float w[kBatch], dot[kBatch];
  auto begin = [&]() {
    look_up(at.t, r);
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      w[j] = at.t < T && j < K ? __ldg(weights + (size_t)at.t * K + j) : 0.f;
      dot[j] = 0.f;
    }
  };
  begin();
#pragma unroll
  for (int i = 0; i < kSteps - 1; ++i) copy(i);
  while (at.t < T) {
#pragma unroll
    for (int place = 0; place < kSteps; ++place) {
      copy((place + kSteps - 1) % kSteps);
      copies_wait<kSteps - 1>();
      const int v = at.step * GS + lane;
      if (at.t < T && v < nvec) {
        float gf[N];
#pragma unroll
        for (int i = 0; i < N; ++i) gf[i] = to_float(g[place].v[i]);
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          const unsigned row = r[j] >= 0 ? r[j] : -1 - r[j];
          if (row >= R) continue;
          Pack<TRow, N> o = zero_pack<TRow, N>();
          if (r[j] >= 0) {
            const uint4 raw = s_place[(place * kBatch + j) * kStreamThreads + threadIdx.x];
            const Pack<TRow, N>& x = reinterpret_cast<const Pack<TRow, N>&>(raw);
#pragma unroll
            for (int i = 0; i < N; ++i) {
              dot[j] = fmaf(gf[i], to_float(x.v[i]), dot[j]);
              o.v[i] = from_float<TRow>(w[j] * gf[i]);
            }
          }
          if (grad_rows) store_wide<TRow, N>(grad_rows + (size_t)row * H + (size_t)v * N, o);
        }
      }
      const int t = at.t;
      if (!next(at)) continue;                     // the same for a group's threads
      // the token is done: its dot products over the group's threads
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
#pragma unroll
        for (int off = 16; off; off >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], off);
      float mine = 0.f;
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if ((lane & 31) == j) mine = dot[j];
      if (kWarps > 1) {
        if ((lane & 31) < kBatch) s_dot[group][lane >> 5][lane & 31] = mine;
        named_bar_sync(1 + group, GS);
        if (lane < kBatch) {
          mine = 0.f;
#pragma unroll
          for (int q = 0; q < kWarps; ++q) mine += s_dot[group][q][lane];
        }
        named_bar_sync(1 + group, GS);
      }
      if (t < T && lane < kBatch && lane < K) grad_weights[(size_t)t * K + lane] = mine;
      begin();
    }
  }
  copies_wait<0>();
}

// ---------------------------------------------------------------- host side
// How many threads of a CTA lie along a row: the most (up to 256) that leave
// the fewest lanes idle in the row's last chunk.
int row_threads(int nvec) {
  int best = 32;
  int64_t least = INT64_MAX;
  for (int tx = 256; tx >= 8; tx >>= 1) {
    const int64_t covered = ((int64_t)nvec + tx - 1) / tx * tx;
    if (covered < least) { least = covered; best = tx; }
  }
  return best;
}

struct Grid {
  int tx, chunks;
  int64_t blocks;
};
Grid row_grid(int T, int nvec) {
  Grid g;
  g.tx = row_threads(nvec);
  g.chunks = (nvec + g.tx - 1) / g.tx;
  const int ty = 256 / g.tx;
  g.blocks = ((int64_t)T + ty - 1) / ty * g.chunks;
  return g;
}

int check_sizes(int32_t T, int32_t K, int32_t H) {
  if (T < 0 || K < 1 || H < 1) return MOE_ERR_INVALID_ARGUMENT;
  if ((int64_t)T * K > INT32_MAX / 2) return MOE_ERR_TOO_LARGE;   // rows and -1 - row are int32
  return MOE_OK;
}

template <typename W>
int run_dispatch(const void* hidden, const int32_t* inv_row, int T, int K, int64_t nvec, void* rows, cudaStream_t s) {
  const Grid g = row_grid(T, (int)nvec);
  if (g.blocks > INT32_MAX) return MOE_ERR_TOO_LARGE;
  return cuda_status(launch_pdl(dispatch_kernel<W>, dim3((unsigned)g.blocks), dim3(256), 0, s,
                                static_cast<const W*>(hidden), inv_row, T, K, (int)nvec, g.chunks, g.tx,
                                static_cast<W*>(rows)));
}

template <typename TRow, typename TOut, int N>
int run_combine_n(const void* rows, const int32_t* inv_row, const float* w, int T, int K, int H, void* out,
                  cudaStream_t s) {
  const Grid g = row_grid(T, H / N);
  if (g.blocks > INT32_MAX) return MOE_ERR_TOO_LARGE;
  auto kern = w ? combine_rows_kernel<TRow, TOut, N, true> : combine_rows_kernel<TRow, TOut, N, false>;
  return cuda_status(launch_pdl(kern, dim3((unsigned)g.blocks), dim3(256), 0, s, static_cast<const TRow*>(rows),
                                inv_row, w, T, K, H / N, g.chunks, g.tx, static_cast<TOut*>(out)));
}

constexpr size_t kPlaceBytes = (size_t)kSteps * kBatch * kStreamThreads * 16;

// Two CTAs on each SM at most; fewer when there is less to do.
int stream_grid(int64_t ctas, int* grid) {
  int sms = 0;
  const int st = require_device(&sms);
  *grid = (int)(ctas < 2 * sms ? ctas : 2 * sms);
  return st;
}

template <typename Kern, typename... Args>
int launch_stream(std::atomic<void*>* seen, Kern kern, int grid, cudaStream_t s, Args... args) {
  const cudaError_t e = once_per_context(seen, [&] {
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kPlaceBytes);
  });
  if (e != cudaSuccess) return cuda_status(e);
  return cuda_status(launch_pdl(kern, dim3(grid), dim3(kStreamThreads), kPlaceBytes, s, args...));
}

template <typename TRow, typename TOut>
int run_combine_stream(const void* rows, const int32_t* inv_row, const float* w, int T, int K, int H, void* out,
                       cudaStream_t s) {
  static std::atomic<void*> seen[2][kMaxCachedDevices];
  const int nvec = H / (16 / (int)sizeof(TRow));
  int grid = 0;
  const int st = stream_grid(((int64_t)T * nvec + kStreamThreads - 1) / kStreamThreads, &grid);
  if (st != MOE_OK) return st;
  if (w)
    return launch_stream(seen[0], combine_stream_kernel<TRow, TOut, true>, grid, s, static_cast<const TRow*>(rows), inv_row,
                         w, T, K, nvec, static_cast<TOut*>(out));
  return launch_stream(seen[1], combine_stream_kernel<TRow, TOut, false>, grid, s, static_cast<const TRow*>(rows), inv_row, w,
                       T, K, nvec, static_cast<TOut*>(out));
}

template <typename TRow, typename TOut, int GS>
int run_backward_stream(const void* g, const void* rows, const int32_t* inv_row, const float* w, int T, int K, int H,
                        void* grad_rows, float* grad_w, cudaStream_t s) {
  static std::atomic<void*> seen[kMaxCachedDevices];
  constexpr int kGroups = kStreamThreads / GS;
  int grid = 0;
  const int st = stream_grid((T + kGroups - 1) / kGroups, &grid);
  if (st != MOE_OK) return st;
  return launch_stream(seen, combine_backward_stream_kernel<TRow, TOut, GS>, grid, s, static_cast<const TOut*>(g),
                       static_cast<const TRow*>(rows), inv_row, w, T, K, H / (16 / (int)sizeof(TRow)),
                       static_cast<TRow*>(grad_rows), grad_w);
}

template <typename TRow, typename TOut>
int run_combine(const void* rows, const int32_t* inv_row, const float* w, int T, int K, int H, void* out,
                cudaStream_t s) {
  constexpr int kMost = 16 / (int)sizeof(TRow);
  int n = vector_elements(H, sizeof(TRow), kMost, {rows});
  n = vector_elements(H, sizeof(TOut), n, {out});
  // From half a million pieces on the copies ahead pay (16-byte pieces of the output; bf16, 8 picks,
  // us with and without: 8192 x 512 26.7 and 26.7, 4096 x 2048 39 and 43, 4096 x 7168 98 and 127;
  // 64 x 1024 10.2 and 8.2).
  const int64_t pieces = (int64_t)T * (H / n);
  if (n == kMost && K <= kBatch && pieces >= 1 << 19 && pieces < INT32_MAX / 2)
    return run_combine_stream<TRow, TOut>(rows, inv_row, w, T, K, H, out, s);
  switch (n) {
    case 8: if constexpr (kMost >= 8) return run_combine_n<TRow, TOut, 8>(rows, inv_row, w, T, K, H, out, s);
    case 4: return run_combine_n<TRow, TOut, 4>(rows, inv_row, w, T, K, H, out, s);
    case 2: return run_combine_n<TRow, TOut, 2>(rows, inv_row, w, T, K, H, out, s);
    default: return run_combine_n<TRow, TOut, 1>(rows, inv_row, w, T, K, H, out, s);
  }
}

template <typename TRow, typename TOut, int N, int GS>
int run_backward_gs(const void* g, const void* rows, const int32_t* inv_row, const float* w, int T, int K, int H,
                    void* grad_rows, float* grad_w, cudaStream_t s) {
  constexpr int kGroups = GS < 128 ? 128 / GS : 1;
  return cuda_status(launch_pdl(combine_backward_kernel<TRow, TOut, N, GS>, dim3((T + kGroups - 1) / kGroups),
                                dim3(GS < 128 ? 128 : GS), 0, s, static_cast<const TOut*>(g),
                                static_cast<const TRow*>(rows), inv_row, w, T, K, H / N,
                                static_cast<TRow*>(grad_rows), grad_w));
}

template <typename TRow, typename TOut, int N>
int run_backward_n(const void* g, const void* rows, const int32_t* inv_row, const float* w, int T, int K, int H,
                   void* grad_rows, float* grad_w, cudaStream_t s) {
  if (H / N > 128)
    return run_backward_gs<TRow, TOut, N, 128>(g, rows, inv_row, w, T, K, H, grad_rows, grad_w, s);
  return run_backward_gs<TRow, TOut, N, 32>(g, rows, inv_row, w, T, K, H, grad_rows, grad_w, s);
}

template <typename TRow, typename TOut>
int run_backward(const void* g, const void* rows, const int32_t* inv_row, const float* w, int T, int K, int H,
                 void* grad_rows, float* grad_w, cudaStream_t s) {
  constexpr int kMost = 16 / (int)sizeof(TRow);
  int n = vector_elements(H, sizeof(TRow), kMost, {grad_w ? rows : nullptr, grad_rows});
  n = vector_elements(H, sizeof(TOut), n, {g});
  if (n == kMost && K <= kBatch && grad_w) {
    // A warp for each token needs no barriers, but its steps follow one another; so more threads for
    // longer rows and for few tokens (bf16, us with 32 / 128 / 256 threads: 8192 x 1024, 8 picks,
    // 59 / 67 / -, with 2 picks 33 / 45 / -; 2048 x 2048 33 / 35 / 39; 4096 x 7168 182 / 168 / 170;
    // 512 x 1024 16 / 14 / -; 64 x 7168 55 / 21 / 14).
    const int vectors = H / n;
    if (vectors > 128 && T <= 256) return run_backward_stream<TRow, TOut, 256>(g, rows, inv_row, w, T, K, H, grad_rows, grad_w, s);
    if (vectors > (T < 1024 ? 64 : 256))
      return run_backward_stream<TRow, TOut, 128>(g, rows, inv_row, w, T, K, H, grad_rows, grad_w, s);
    return run_backward_stream<TRow, TOut, 32>(g, rows, inv_row, w, T, K, H, grad_rows, grad_w, s);
  }
  switch (n) {
    case 8:
      if constexpr (kMost >= 8)
        return run_backward_n<TRow, TOut, 8>(g, rows, inv_row, w, T, K, H, grad_rows, grad_w, s);
    case 4: return run_backward_n<TRow, TOut, 4>(g, rows, inv_row, w, T, K, H, grad_rows, grad_w, s);
    case 2: return run_backward_n<TRow, TOut, 2>(g, rows, inv_row, w, T, K, H, grad_rows, grad_w, s);
    default: return run_backward_n<TRow, TOut, 1>(g, rows, inv_row, w, T, K, H, grad_rows, grad_w, s);
  }
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

MOE_API int moe_tokens_sort(const int32_t* topk_ids, int32_t num_tokens, int32_t top_k, int32_t num_local_experts,
                            int32_t local_expert_offset, int32_t* offsets, int32_t* inv_row, int32_t* row_token,
                            void* stream) {
  int st = check_sizes(num_tokens, top_k, 1);
  if (st != MOE_OK) return st;
  if (num_local_experts < 1 || local_expert_offset < 0 || !offsets) return MOE_ERR_INVALID_ARGUMENT;
  if (num_local_experts > kSortMaxExperts) return MOE_ERR_TOO_LARGE;
  if (local_expert_offset > INT32_MAX - num_local_experts) return MOE_ERR_TOO_LARGE;   // no id may wrap into the shard
  const int P = num_tokens * top_k;
  if (P > 0 && (!topk_ids || !inv_row || !row_token)) return MOE_ERR_INVALID_ARGUMENT;
  for (const void* p : {static_cast<const void*>(topk_ids), static_cast<const void*>(offsets),
                        static_cast<const void*>(inv_row), static_cast<const void*>(row_token)})
    if (!aligned_to(p, 4)) return MOE_ERR_MISALIGNED;
  if ((st = require_device(nullptr)) != MOE_OK) return st;
  // One CTA for small batches; eight, as a cluster, when each of its warps
  // would have more than 32 pairs (3885 pairs: 9.1 us with one, 7 with eight).
  const int ctas = P > 1024 ? kSortCluster : 1;
  int threads = (P + 31) / 32 * 32;
  threads = threads < 256 ? 256 : threads > 1024 ? 1024 : (threads + 127) / 128 * 128;   // 4 warps or a multiple
  const int warps = threads / 32 * ctas;
  const int run = (int)((((int64_t)P + warps - 1) / warps + 31) / 32 * 32);
  const size_t smem = ((size_t)(threads / 32) + 3) * (num_local_experts + 1) * sizeof(int);
  static std::atomic<void*> seen[kMaxCachedDevices];
  cudaError_t e = once_per_context(seen, [] {
    return cudaFuncSetAttribute(sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (32 + 3) * (kSortMaxExperts + 1) * (int)sizeof(int));
  });
  if (e != cudaSuccess) return cuda_status(e);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cuda_status(cudaLaunchKernelEx(&cfg, sort_kernel, topk_ids, P, (int)top_k, (int)num_local_experts,
                                        (int)local_expert_offset, run, offsets, inv_row, row_token));
}

MOE_API int moe_tokens_dispatch(const void* hidden, const int32_t* inv_row, int32_t num_tokens, int32_t top_k,
                                int32_t width, int32_t dtype, void* rows, void* stream) {
  int st = check_sizes(num_tokens, top_k, width);
  if (st != MOE_OK) return st;
  const int bytes = dtype_bytes(dtype);
  if (!bytes) return MOE_ERR_INVALID_ARGUMENT;
  if (num_tokens == 0) return MOE_OK;
  if (!hidden || !inv_row || !rows) return MOE_ERR_INVALID_ARGUMENT;
  if (!aligned_to(hidden, bytes) || !aligned_to(rows, bytes) || !aligned_to(inv_row, 4)) return MOE_ERR_MISALIGNED;
  if ((st = require_device(nullptr)) != MOE_OK) return st;
  const int n = vector_elements(width, bytes, 16 / bytes, {hidden, rows});
  const int64_t nvec = width / n;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (n * bytes) {   // the rows are copied, so only their size matters
    case 16: return run_dispatch<uint4>(hidden, inv_row, num_tokens, top_k, nvec, rows, s);
    case 8: return run_dispatch<uint2>(hidden, inv_row, num_tokens, top_k, nvec, rows, s);
    case 4: return run_dispatch<uint32_t>(hidden, inv_row, num_tokens, top_k, nvec, rows, s);
    default: return run_dispatch<uint16_t>(hidden, inv_row, num_tokens, top_k, nvec, rows, s);
  }
}

MOE_API int moe_tokens_combine(const void* rows, const int32_t* inv_row, const float* weights, int32_t num_tokens,
                               int32_t top_k, int32_t width, int32_t rows_dtype, int32_t out_dtype, void* out,
                               void* stream) {
  int st = check_sizes(num_tokens, top_k, width);
  if (st != MOE_OK) return st;
  if (!dtype_bytes(rows_dtype) || !dtype_bytes(out_dtype)) return MOE_ERR_INVALID_ARGUMENT;
  if (rows_dtype != out_dtype && rows_dtype != MOE_F32) return MOE_ERR_INVALID_ARGUMENT;
  if (num_tokens == 0) return MOE_OK;
  if (!rows || !inv_row || !out) return MOE_ERR_INVALID_ARGUMENT;
  if (!aligned_to(rows, dtype_bytes(rows_dtype)) || !aligned_to(out, dtype_bytes(out_dtype)) ||
      !aligned_to(inv_row, 4) || !aligned_to(weights, 4))
    return MOE_ERR_MISALIGNED;
  if ((st = require_device(nullptr)) != MOE_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define MOE_COMBINE(TRow, TOut) \
  return run_combine<TRow, TOut>(rows, inv_row, weights, num_tokens, top_k, width, out, s)
  if (rows_dtype == MOE_BF16) MOE_COMBINE(__nv_bfloat16, __nv_bfloat16);
  if (rows_dtype == MOE_F16) MOE_COMBINE(__half, __half);
  if (out_dtype == MOE_BF16) MOE_COMBINE(float, __nv_bfloat16);
  if (out_dtype == MOE_F16) MOE_COMBINE(float, __half);
  MOE_COMBINE(float, float);
#undef MOE_COMBINE
}

MOE_API int moe_tokens_combine_backward(const void* grad_out, const void* rows, const int32_t* inv_row,
                                        const float* weights, int32_t num_tokens, int32_t top_k, int32_t width,
                                        int32_t rows_dtype, int32_t out_dtype, void* grad_rows,
                                        float* grad_weights, void* stream) {
  int st = check_sizes(num_tokens, top_k, width);
  if (st != MOE_OK) return st;
  if (!dtype_bytes(rows_dtype) || !dtype_bytes(out_dtype)) return MOE_ERR_INVALID_ARGUMENT;
  if (rows_dtype != out_dtype && rows_dtype != MOE_F32) return MOE_ERR_INVALID_ARGUMENT;
  if (num_tokens == 0 || (!grad_rows && !grad_weights)) return MOE_OK;
  if (!grad_out || !inv_row || !weights || (grad_weights && !rows)) return MOE_ERR_INVALID_ARGUMENT;
  if (!aligned_to(grad_out, dtype_bytes(out_dtype)) || !aligned_to(rows, dtype_bytes(rows_dtype)) ||
      !aligned_to(grad_rows, dtype_bytes(rows_dtype)) || !aligned_to(inv_row, 4) || !aligned_to(weights, 4) ||
      !aligned_to(grad_weights, 4))
    return MOE_ERR_MISALIGNED;
  if ((st = require_device(nullptr)) != MOE_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define MOE_BACKWARD(TRow, TOut)                                                                             \
  return run_backward<TRow, TOut>(grad_out, rows, inv_row, weights, num_tokens, top_k, width, grad_rows,     \
                                  grad_weights, s)
  if (rows_dtype == MOE_BF16) MOE_BACKWARD(__nv_bfloat16, __nv_bfloat16);
  if (rows_dtype == MOE_F16) MOE_BACKWARD(__half, __half);
  if (out_dtype == MOE_BF16) MOE_BACKWARD(float, __nv_bfloat16);
  if (out_dtype == MOE_F16) MOE_BACKWARD(float, __half);
  MOE_BACKWARD(float, float);
#undef MOE_BACKWARD
}

}  // extern "C"
