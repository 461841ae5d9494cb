// Tokens sorted by expert and back, with the gradients of both moves.
//
// A pair is a token's k-th choice, numbered p = t * top_k + k.  sort: a stable counting sort of the pairs by local expert,
//   offsets[e] = align * sum_{e' < e} ceil(counts[e'] / align)
//   pos[t,k]   = offsets[e] + (pairs of the same expert e before p), -1 where the expert is not local
//   pair[pos[t,k]] = p, -1 in padding rows and behind the last segment
// permute: y[pos[t,k]] = x[t];  its gradient and the way back, unpermute: out[t] = sum_k w[t,k] y[pos[t,k]] (k ascending,
// fp32, rounded once);  gradient of that: dy[pos[t,k]] = w[t,k] dout[t], dw[t,k] = <dout[t], y[pos[t,k]]>.
//
// No atomics on anything that an order could change, so all results repeat bit for bit.  All but the sort is bound by HBM.
// Every pass walks tokens, not sorted rows: a token's row is then read (or written) once and its top_k sorted rows once.
#include "common.cuh"
#include "host.cuh"
#include "kernels.cuh"

namespace b200moe {

namespace {

constexpr int kMaxSortExperts = 1024;
constexpr int kMaxSortTopK = 32;                 // a token's positions are held by the lanes of a warp
constexpr int kSortWarps = 16;
constexpr int kSortThreads = 32 * kSortWarps;
constexpr int kSortCluster = 8;                  // CTAs that one launch sorts with
constexpr int kSortRounds = 4;                   // pairs of a thread
constexpr int kSortChunk = kSortThreads * kSortRounds;

struct SortParams {
  const void* ids;
  long long ids_stride;
  int pairs, top_k;
  int contiguous;                                // ids_stride == top_k
  int wide;                                      // int64 ids
  int vec_pair;                                  // what lies behind the last segment starts on 16 bytes of `pair`
  int local_off, e_local, align;
  int rows;                                      // length of `pair`
  int* counts;                                   // [e_local]
  int* offsets;                                  // [e_local + 1]
  int* pos;                                      // [pairs]
  int* pair;                                     // [rows]
  int* chunk_counts;                             // [chunks][e_local] of the kernel before; null: the chunks are one cluster
  int chunks;
  int scanned;                                   // chunk_counts [chunks + 1][e_local] holds the sums over the chunks before
};

__device__ __forceinline__ int local_expert(const SortParams& p, int i) {
  long long at = i;
  if (!p.contiguous) {
    const int t = i / p.top_k;
    at = t * p.ids_stride + (i - t * p.top_k);
  }
  const long long id = p.wide ? reinterpret_cast<const long long*>(p.ids)[at] : (long long)reinterpret_cast<const int*>(p.ids)[at];
  return id >= p.local_off && id < (long long)p.local_off + p.e_local ? (int)(id - p.local_off) : -1;
}

// Expert of each of a thread's pairs (-1: not local, or past the end): warp w of chunk c has the 32 x kSortRounds pairs from
// (c * kSortWarps + w) * 32 kSortRounds on, round r 32 of them.  All loads are in flight together.
__device__ __forceinline__ long long load_experts(const SortParams& p, int (&e)[kSortRounds]) {
  const long long first = ((long long)blockIdx.x * kSortWarps + (threadIdx.x >> 5)) * (32 * kSortRounds) + (threadIdx.x & 31);
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    const long long i = first + r * 32;
    e[r] = i < p.pairs ? local_expert(p, (int)i) : -1;
  }
  return first;
}

__global__ void __launch_bounds__(kSortThreads)
sort_count_kernel(const __grid_constant__ SortParams p) {
  extern __shared__ int s_cnt[];                 // [e_local]
  for (int e = threadIdx.x; e < p.e_local; e += kSortThreads) s_cnt[e] = 0;
  chain_wait();
  chain_release();
  int e[kSortRounds];
  load_experts(p, e);
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r)
    if (e[r] >= 0) atomicAdd(s_cnt + e[r], 1);
  __syncthreads();
  for (int x = threadIdx.x; x < p.e_local; x += kSortThreads) p.chunk_counts[(size_t)blockIdx.x * p.e_local + x] = s_cnt[x];
}

// The counts of many chunks become the sums over the chunks before, with the totals behind them: a warp takes 32 experts'
// neighbouring counters through a 32nd of the chunks, first for its sum and then for the sums before each chunk.
__global__ void __launch_bounds__(1024)
sort_scan_kernel(const __grid_constant__ SortParams p) {
  __shared__ int s_sum[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, E = p.e_local, x = (int)blockIdx.x * 32 + lane;
  const int per = (p.chunks + 31) / 32, c0 = warp * per, c1 = min(c0 + per, p.chunks);
  chain_wait();
  chain_release();
  int sum = 0;
  if (x < E) {
#pragma unroll 16
    for (int c = c0; c < c1; ++c) sum += p.chunk_counts[(size_t)c * E + x];
  }
  s_sum[warp][lane] = sum;
  __syncthreads();
  if (x >= E) return;
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < 32; ++w) {
    const int n = s_sum[w][lane];
    before += w < warp ? n : 0;
    total += n;
  }
  for (int c = c0; c < c1; c += 8) {
    int n[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) n[j] = c + j < c1 ? p.chunk_counts[(size_t)(c + j) * E + x] : 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (c + j < c1) p.chunk_counts[(size_t)(c + j) * E + x] = before;
      before += n[j];
    }
  }
  if (warp == 0) p.chunk_counts[(size_t)p.chunks * E + x] = total;
}

// Exclusive sum over the CTA's threads.
__device__ __forceinline__ int block_exclusive_sum(int v, int* s_warp, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int sum = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += up;
  }
  if (lane == 31) s_warp[warp] = sum;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSortWarps; ++w) {
    const int x = s_warp[w];
    before += w < warp ? x : 0;
    all += x;
  }
  *total = all;
  return sum - v + before;
}

__device__ __forceinline__ int ld_cluster_s32(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// Places the pairs of a CTA's chunk.  Each warp owns a run of the chunk and a row of counters; a pair's place among its warp's
// pairs of the same expert is the counter plus its rank in a match of the expert over the warp, a warp's first place the sum over
// the warps before it.  What the other chunks hold comes out of their shared memory (the chunks are one cluster: one launch),
// or out of the kernel before.  What this takes is latency: no loop over anything but rounds, warps and chunks.
__global__ void __launch_bounds__(kSortThreads)
sort_place_kernel(const __grid_constant__ SortParams p) {
  extern __shared__ __align__(16) int smem[];
  const int E = p.e_local;
  int* s_cnt = smem;                             // [kSortWarps][E]
  int* s_total = s_cnt + kSortWarps * E;         // [E] pairs of all chunks
  int* s_before = s_total + E;                   // [E] pairs of the chunks before this one
  int* s_chunk = s_before + E;                   // [E] pairs of this chunk
  int* s_first = s_chunk + E;                    // [E + 1]
  __shared__ int s_warp[kSortWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < (kSortWarps + 2) * E; i += kSortThreads) smem[i] = 0;
  chain_wait();
  chain_release();
  int e[kSortRounds], rank[kSortRounds];
  const long long first_pair = load_experts(p, e);
  __syncthreads();
  int* mine = s_cnt + warp * E;
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    const unsigned same = __match_any_sync(0xffffffffu, e[r]);
    const int before = e[r] >= 0 ? mine[e[r]] : 0;
    rank[r] = before + __popc(same & ((1u << lane) - 1u));
    __syncwarp();
    if (e[r] >= 0 && lane == 31 - __clz(same)) mine[e[r]] = rank[r] + 1;
    __syncwarp();
  }
  __syncthreads();
  for (int x = threadIdx.x; x < E; x += kSortThreads) {
    int n[kSortWarps], sum = 0;
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) n[w] = s_cnt[w * E + x];
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      s_cnt[w * E + x] = sum;
      sum += n[w];
    }
    s_chunk[x] = sum;
  }
  const bool cluster = p.chunks > 1 && !p.chunk_counts;
  if (cluster) {
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    for (int x = threadIdx.x; x < E; x += kSortThreads) {
      const uint32_t addr = smem_u32(s_chunk + x);
      int n[kSortCluster];
#pragma unroll
      for (int c = 0; c < kSortCluster; ++c) n[c] = c < p.chunks ? ld_cluster_s32(map_to_rank(addr, c)) : 0;
      int total = 0, before = 0;
#pragma unroll
      for (int c = 0; c < kSortCluster; ++c) {
        total += n[c];
        before += c < (int)blockIdx.x ? n[c] : 0;
      }
      s_total[x] = total;
      s_before[x] = before;
    }
    __syncwarp();
    cluster_arrive();                            // waited for at the end: peers may still read this CTA's counts
  } else if (p.scanned) {
    for (int x = threadIdx.x; x < E; x += kSortThreads) {
      s_total[x] = p.chunk_counts[(size_t)p.chunks * E + x];
      s_before[x] = p.chunk_counts[(size_t)blockIdx.x * E + x];
    }
  } else if (p.chunk_counts) {
    const int parts = E < kSortThreads ? kSortThreads / E : 1;
    const int per = (p.chunks + parts - 1) / parts;
    for (int i = threadIdx.x; i < parts * E; i += kSortThreads) {
      const int x = i % E, c0 = i / E * per, c1 = min(c0 + per, p.chunks);
      int total = 0, before = 0;
#pragma unroll 16
      for (int c = c0; c < c1; ++c) {
        const int n = p.chunk_counts[(size_t)c * E + x];
        total += n;
        before += c < (int)blockIdx.x ? n : 0;
      }
      atomicAdd(s_total + x, total);
      atomicAdd(s_before + x, before);
    }
    __syncthreads();
  } else {
    for (int x = threadIdx.x; x < E; x += kSortThreads) s_total[x] = s_chunk[x];
  }
  // first rows: a thread has the experts [per x thread, + per); up to kSortThreads experts each has those that it wrote above
  if (E > kSortThreads) __syncthreads();
  const int per = (E + kSortThreads - 1) / kSortThreads, x0 = threadIdx.x * per;
  int padded[kMaxSortExperts / kSortThreads], sum = 0;
#pragma unroll
  for (int j = 0; j < kMaxSortExperts / kSortThreads; ++j) {
    padded[j] = j < per && x0 + j < E ? (s_total[x0 + j] + p.align - 1) / p.align * p.align : 0;
    sum += padded[j];
  }
  int used;
  int first = block_exclusive_sum(sum, s_warp, &used);
#pragma unroll
  for (int j = 0; j < kMaxSortExperts / kSortThreads; ++j) {
    if (j >= per || x0 + j >= E) break;
    s_first[x0 + j] = first;
    if (blockIdx.x == 0) {
      p.counts[x0 + j] = s_total[x0 + j];
      p.offsets[x0 + j] = first;
    }
    first += padded[j];
  }
  if (threadIdx.x == 0) {
    s_first[E] = used;
    if (blockIdx.x == 0) p.offsets[E] = used;
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    const long long i = first_pair + r * 32;
    const int row = e[r] >= 0 ? s_first[e[r]] + s_before[e[r]] + mine[e[r]] + rank[r] : -1;
    if (i < p.pairs) p.pos[i] = row;
    if (row >= 0) p.pair[row] = (int)i;
  }
  // rows that no pair takes: the padding of every chunks-th expert, and a share of what lies behind the last segment
  if (p.align > 1)
    for (int x = (int)blockIdx.x + warp * (int)gridDim.x; x < E; x += (int)gridDim.x * kSortWarps)
      for (int r = s_first[x] + s_total[x] + lane; r < s_first[x + 1]; r += 32) p.pair[r] = -1;
  long long tail = used;
  if (p.vec_pair) {                              // (`used` and `rows` are multiples of align, a multiple of four)
    for (long long r = (long long)used / 4 + (long long)blockIdx.x * kSortThreads + threadIdx.x; r < p.rows / 4; r += (long long)gridDim.x * kSortThreads)
      reinterpret_cast<int4*>(p.pair)[r] = make_int4(-1, -1, -1, -1);
    tail = p.rows / 4 * 4;
  }
  for (long long r = tail + (long long)blockIdx.x * kSortThreads + threadIdx.x; r < p.rows; r += (long long)gridDim.x * kSortThreads)
    p.pair[r] = -1;
  __syncwarp();
  if (cluster) cluster_wait();
}

size_t sort_place_smem(int e_local) { return ((size_t)(kSortWarps + 4) * e_local + 1) * 4; }

// How a number of pairs is sorted: chunks of kSortChunk pairs, in one launch (of one cluster) or in two.  (Four times as many pairs
// a thread took longer at every size: 28 us instead of 19 for 2^19 pairs of 256 experts.)
struct SortPlan {
  int chunks;
  bool one_launch;
};
SortPlan sort_plan(long long pairs, long long rows) {
  SortPlan s;
  s.one_launch = pairs <= (long long)kSortCluster * kSortChunk;
  s.chunks = pairs > 0 ? (int)((pairs + kSortChunk - 1) / kSortChunk) : 1;
  if (s.one_launch) {
    // clusters of 1, 2, 4, 8; CTAs without pairs where many empty rows are to be marked (16 tokens of 256 experts whose segments
    // start on multiples of 128: 32640 rows)
    while (s.chunks < kSortCluster && rows > (long long)s.chunks * 4096) ++s.chunks;
    while (s.chunks & (s.chunks - 1)) ++s.chunks;
  }
  return s;
}
// Every chunk adds up what the others have of each expert, which goes with the square of the chunks; from this many counters
// on a launch of its own makes running sums of them.  us without / with (experts x chunks): 8 x 256 9.0 / 12.6; 256 x 64 10.0 /
// 12.1, x 128 17.3 / 13.2, x 1024 72 / 47; 1024 x 32 12.6 / 12.8, x 64 15.8 / 13.2, x 256 52.6 / 19.9.
constexpr long long kSortScanCounters = 24576;

cudaError_t launch_sort(const SortParams& p, const SortPlan& plan, cudaStream_t stream) {
  if (!plan.one_launch) {
    cudaError_t e = launch_chained(sort_count_kernel, dim3(plan.chunks), dim3(kSortThreads), (size_t)p.e_local * 4, stream, p);
    if (e == cudaSuccess && p.scanned) e = launch_chained(sort_scan_kernel, dim3((p.e_local + 31) / 32), dim3(1024), 0, stream, p);
    if (e != cudaSuccess) return e;
  }
  return launch_chained_cluster(sort_place_kernel, dim3(plan.chunks), dim3(kSortThreads), sort_place_smem(p.e_local), stream,
                                plan.one_launch ? plan.chunks : 1, p);
}

// ---- moving rows ----

// V: what a lane moves at once (16 bytes, or one element where a row does not start on such a boundary).
struct RowMove {
  const uint8_t* src;
  long long src_stride;                          // bytes
  uint8_t* dst;
  long long dst_stride;
  const int* pos;
  const int* pair;
  const int* used_rows;                          // device: rows of all segments
  long long tokens, rows;
  int top_k;
  int row_vecs;                                  // V's of a row
  int zero_tail;                                 // rows behind the last segment are zeroed too
};

constexpr int kMoveThreads = 128;

// Rows of `dst` without a pair become zero; `item` counts groups of `zero_rows` (at most 32) rows.
template <typename V>
__device__ __forceinline__ void zero_empty_rows(const int* pair, const int* used_rows, long long rows, int zero_tail, uint8_t* dst,
                                                long long dst_stride, int row_vecs, int zero_rows, long long item, int lane) {
  const long long r0 = item * zero_rows;
  const long long limit = zero_tail ? rows : (long long)*used_rows;
  bool empty = false;
  if (lane < zero_rows && r0 + lane < rows && r0 + lane < limit) empty = pair[r0 + lane] < 0;
  unsigned todo = __ballot_sync(0xffffffffu, empty);
  while (todo) {
    const int j = __ffs(todo) - 1;
    todo &= todo - 1;
    V* d = reinterpret_cast<V*>(dst + (r0 + j) * dst_stride);
    for (int v = lane; v < row_vecs; v += 32) d[v] = V{};
  }
}

// Sorted rows that a warp looks at for empty ones: some 28 KB, so that those that are empty do not make a warp's work much longer than
// a token's, and a look without one is a small part of what it goes with.
int zero_rows_of(long long row_bytes) { return (int)(row_bytes >= 28672 ? 1 : row_bytes * 32 <= 28672 ? 32 : 28672 / row_bytes); }

// A warp takes U x 32 vectors of one token's row into registers and stores them to the token's sorted rows, or looks at sorted rows
// for empty ones.  One small piece of work a warp, and as many CTAs as that takes: 4096 tokens of 14 KB to 65280 rows of which half are
// empty take 153 us (6.5 TB/s); with four rows to look at, 512 bytes of a token and 64 CTAs an SM that took several pieces each, 174.
template <typename V, int U>
__global__ void __launch_bounds__(kMoveThreads)
permute_kernel(const __grid_constant__ RowMove p, int segments, int segment_vecs, int zero_rows, long long move_items, long long items) {
  chain_wait();
  chain_release();
  const int lane = threadIdx.x & 31;
  const long long step = (long long)gridDim.x * (kMoveThreads / 32);
  for (long long w = (long long)blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5); w < items; w += step) {
    if (w >= move_items) {
      zero_empty_rows<V>(p.pair, p.used_rows, p.rows, p.zero_tail, p.dst, p.dst_stride, p.row_vecs, zero_rows, w - move_items, lane);
      continue;
    }
    const long long t = w / segments;
    const int v_begin = (int)(w - t * segments) * segment_vecs, v_end = min(v_begin + segment_vecs, p.row_vecs), v0 = v_begin + lane;
    const int mine = lane < p.top_k ? p.pos[t * p.top_k + lane] : -1;
    const V* src = reinterpret_cast<const V*>(p.src + t * p.src_stride);
    V x[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v0 + u * 32 < v_end) x[u] = ld_chained(src + v0 + u * 32);
    for (int k = 0; k < p.top_k; ++k) {
      const int row = __shfl_sync(0xffffffffu, mine, k);
      if (row < 0) continue;
      V* dst = reinterpret_cast<V*>(p.dst + row * p.dst_stride);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (v0 + u * 32 < v_end) dst[v0 + u * 32] = x[u];
    }
  }
}

// ---- sums over a token's rows ----

template <typename T, int N> struct alignas(sizeof(T) * N) Pack { T v[N]; };

template <typename T> struct is_bf16 { static constexpr bool value = false; };
template <> struct is_bf16<__nv_bfloat16> { static constexpr bool value = true; };
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
// Element i of a pack; bf16 out of whole words, one instruction each.  (By single elements the gradient of 4096 tokens of 2048 takes
// 54 us instead of 47, of 16384 of 512 71 instead of 53.)
template <typename T, int N>
__device__ __forceinline__ float elem(const Pack<T, N>& p, int i) {
  if constexpr (N % 2 == 0 && sizeof(T) == 2 && is_bf16<T>::value) {
    uint32_t w;
    memcpy(&w, p.v + (i & ~1), 4);
    return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
  } else {
    return to_float(p.v[i]);
  }
}
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename P>
__device__ __forceinline__ P load_pack(const P* p) {
  P r;
  if constexpr (sizeof(P) == 16) {
    const uint4 u = ld_chained(reinterpret_cast<const uint4*>(p));
    memcpy(&r, &u, 16);
  } else {
    r = *p;
  }
  return r;
}
template <typename P>
__device__ __forceinline__ void store_pack(P* p, const P& v) {
  if constexpr (sizeof(P) == 16) {
    uint4 u;
    memcpy(&u, &v, 16);
    *reinterpret_cast<uint4*>(p) = u;
  } else {
    *p = v;
  }
}

constexpr int kSumBatch = 8;                     // rows of a token in flight together

// A GROUP of threads takes a token's output row, or one of `segments` parts of it: the rows' addresses are then known for the whole
// row, and eight loads a thread are in flight (U times as many where a load brings less than 16 bytes).  (A warp for each 512 bytes
// of an output row, which has to fetch the positions first, reached 3.5 TB/s of 14 KB rows, this 6.)  AHEAD: four CTAs an SM take
// one row after another, with the next one's positions on their way meanwhile.  us, without / with: 8192 rows of 2048 bf16 62 /
// 53, 4096 of 7168 89 / 84; 4097 of 2048 fp32 47 / 57, of 7168 153 / 184: fp32, whose sums take fewer registers, has six CTAs on an SM
// without it (with four of them 58 us).
template <typename T, int N, int U, int GROUP, bool AHEAD>
__global__ void __launch_bounds__(kMoveThreads, AHEAD ? 4 : 6)
unpermute_kernel(const T* y, long long y_stride, const int* pos, const float* weights, long long w_stride, T* __restrict__ out,
                 long long out_stride, int items, int top_k, int row_vecs, int segments, int segment_vecs) {
  using P = Pack<T, N>;
  chain_wait();
  chain_release();
  int row[kSumBatch];
  float w[kSumBatch];
  auto fetch = [&](int t, int k0) {
    const int* at = pos + (size_t)t * top_k + k0;
#pragma unroll
    for (int j = 0; j < kSumBatch; ++j) {
      row[j] = k0 + j < top_k ? ld_chained(at + j) : -1;
      w[j] = weights && k0 + j < top_k ? ld_chained(weights + (size_t)t * w_stride + k0 + j) : 1.f;
    }
  };
  const int lane = threadIdx.x % GROUP;
  int item = blockIdx.x * (kMoveThreads / GROUP) + threadIdx.x / GROUP;
  if (item >= items) return;
  fetch(item / segments, 0);
  do {
    const int t = item / segments, v_begin = (item - t * segments) * segment_vecs, v_end = min(v_begin + segment_vecs, row_vecs);
    P* dst = reinterpret_cast<P*>(out + (size_t)t * out_stride);
    const P* src[kSumBatch];
    float weight[kSumBatch];
    auto use = [&] {
#pragma unroll
      for (int j = 0; j < kSumBatch; ++j) {
        src[j] = row[j] >= 0 ? reinterpret_cast<const P*>(y + row[j] * y_stride) : nullptr;
        weight[j] = w[j];
      }
    };
    use();
    item += gridDim.x * (kMoveThreads / GROUP);
    if (AHEAD && top_k <= kSumBatch && item < items) fetch(item / segments, 0);
    for (int v = v_begin + lane; v < v_end; v += U * GROUP) {
      float acc[U][N];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < N; ++i) acc[u][i] = 0.f;
      int at[U];                                   // (loads behind the end repeat the last: one that only some threads make waits alone)
#pragma unroll
      for (int u = 0; u < U; ++u) at[u] = U == 1 ? v : min(v + u * GROUP, v_end - 1);
      for (int k0 = 0;;) {
        P x[kSumBatch][U];
#pragma unroll
        for (int j = 0; j < kSumBatch; ++j)
          if (src[j]) {
#pragma unroll
            for (int u = 0; u < U; ++u) x[j][u] = load_pack(src[j] + at[u]);
          }
#pragma unroll
        for (int j = 0; j < kSumBatch; ++j)
          if (src[j]) {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
              for (int i = 0; i < N; ++i) acc[u][i] = fmaf(weight[j], elem(x[j][u], i), acc[u][i]);
          }
        if (top_k <= kSumBatch) break;
        k0 = k0 + kSumBatch < top_k ? k0 + kSumBatch : 0;   // (more choices: the next eight, and the first again for the next v)
        fetch(t, k0);
        use();
        if (k0 == 0) break;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        P r;
#pragma unroll
        for (int i = 0; i < N; ++i) r.v[i] = from_float<T>(acc[u][i]);
        if (U == 1 || v + u * GROUP < v_end) store_pack(dst + v + u * GROUP, r);
      }
    }
    if (AHEAD && top_k > kSumBatch && item < items) fetch(item / segments, 0);
  } while (AHEAD && item < items);
}

template <typename T>
struct UnpermuteGrad {
  const T* dout;
  long long dout_stride;
  const T* y;
  long long y_stride;
  const float* weights;                          // null: ones
  long long w_stride;
  const int* pos;
  const int* pair;
  const int* used_rows;
  T* dy;                                         // null: not wanted
  long long dy_stride;
  float* dw;                                     // [tokens][top_k], null: not wanted
  long long tokens, rows;
  int top_k, row_vecs;
};

// A GROUP of threads per token: its row of dout is read once (top_k <= 8), each sorted row of y read and of dy written once; the
// dots are summed by shuffles and over the group's warps in a fixed order.
template <typename T, int N, int U, int GROUP>
__global__ void __launch_bounds__(kMoveThreads, U > 1 ? 4 : 5)
unpermute_grad_kernel(const __grid_constant__ UnpermuteGrad<T> p, int zero_rows, long long items) {
  using P = Pack<T, N>;
  constexpr int kWarps = GROUP / 32, kGroups = kMoveThreads / GROUP;
  __shared__ float s_dot[kWarps][kSumBatch];
  chain_wait();
  chain_release();
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32 % kWarps, thread = threadIdx.x % GROUP;
  for (long long t = (long long)blockIdx.x * kGroups + threadIdx.x / GROUP; t < items; t += (long long)gridDim.x * kGroups) {
    if (t >= p.tokens) {
      zero_empty_rows<P>(p.pair, p.used_rows, p.rows, 1, reinterpret_cast<uint8_t*>(p.dy), p.dy_stride * (long long)sizeof(T),
                         p.row_vecs, zero_rows, (t - p.tokens) * kWarps + warp, lane);
      continue;
    }
    const P* dout = reinterpret_cast<const P*>(p.dout + t * p.dout_stride);
    for (int k0 = 0; k0 < p.top_k; k0 += kSumBatch) {
      int row[kSumBatch];
      float wt[kSumBatch], dot[kSumBatch];
#pragma unroll
      for (int j = 0; j < kSumBatch; ++j) {
        const bool there = k0 + j < p.top_k;
        row[j] = there ? p.pos[t * p.top_k + k0 + j] : -1;
        wt[j] = there && p.weights ? p.weights[t * p.w_stride + k0 + j] : 1.f;
        dot[j] = 0.f;
      }
      for (int v = thread; v < p.row_vecs; v += U * GROUP) {
        // (loads behind the end repeat the last vector; neither stored nor summed)
        int at[U];
        bool there[U];
        P d[U], x[kSumBatch][U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          at[u] = U == 1 ? v : min(v + u * GROUP, p.row_vecs - 1);
          there[u] = U == 1 || v + u * GROUP < p.row_vecs;
          d[u] = load_pack(dout + at[u]);
        }
        if (p.dw) {
#pragma unroll
          for (int j = 0; j < kSumBatch; ++j)
            if (row[j] >= 0) {
#pragma unroll
              for (int u = 0; u < U; ++u) x[j][u] = load_pack(reinterpret_cast<const P*>(p.y + row[j] * p.y_stride) + at[u]);
            }
        }
#pragma unroll
        for (int j = 0; j < kSumBatch; ++j) {
          if (row[j] < 0) continue;
#pragma unroll
          for (int u = 0; u < U; ++u) {
            if (p.dw && there[u]) {
#pragma unroll
              for (int i = 0; i < N; ++i) dot[j] = fmaf(elem(d[u], i), elem(x[j][u], i), dot[j]);
            }
            if (p.dy && there[u]) {
              P r;
#pragma unroll
              for (int i = 0; i < N; ++i) r.v[i] = from_float<T>(wt[j] * elem(d[u], i));
              store_pack(reinterpret_cast<P*>(p.dy + row[j] * p.dy_stride) + at[u], r);
            }
          }
        }
      }
      if (p.dw) {
        float* dw = p.dw + t * p.top_k + k0;
#pragma unroll
        for (int j = 0; j < kSumBatch; ++j) {
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], o);
          if (kWarps > 1 && lane == 0) s_dot[warp][j] = dot[j];
          if (kWarps == 1 && lane == j && k0 + j < p.top_k) dw[j] = dot[j];
        }
        if (kWarps > 1) {
          __syncthreads();
          if (thread < kSumBatch && k0 + thread < p.top_k) {
            float sum = 0.f;
            for (int w = 0; w < kWarps; ++w) sum += s_dot[w][thread];
            dw[thread] = sum;
          }
          __syncthreads();
        }
      }
    }
  }
}

unsigned grid_for(long long items, long long most) { return (unsigned)(items < most ? items : most); }

template <typename V, int U>
cudaError_t launch_permute_rows(const RowMove& p, cudaStream_t stream) {
  const int pieces = (p.row_vecs + 31) / 32, segments = (pieces + U - 1) / U, segment_vecs = (pieces + segments - 1) / segments * 32;
  const int zero_rows = zero_rows_of((long long)p.row_vecs * (long long)sizeof(V));
  const long long move_items = p.tokens * segments;
  const long long items = move_items + (p.rows + zero_rows - 1) / zero_rows;
  constexpr int kWarps = kMoveThreads / 32;
  return launch_chained(permute_kernel<V, U>, dim3(grid_for((items + kWarps - 1) / kWarps, 0x7fffffffll)), dim3(kMoveThreads), 0, stream, p,
                        segments, segment_vecs, zero_rows, move_items, items);
}

template <typename T, int N, int U, int GROUP>
cudaError_t launch_unpermute_group(const void* y, long long y_stride, const int* pos, const float* weights, long long w_stride, void* out,
                                   long long out_stride, int tokens, int top_k, int row_vecs, int num_sms, cudaStream_t stream) {
  constexpr bool kAhead = sizeof(T) == 2;
  constexpr int kGroups = kMoveThreads / GROUP;
  // one group a token, more where that leaves SMs without one
  const int pieces = (row_vecs + GROUP - 1) / GROUP;
  int segments = (int)(((kAhead ? 4ll : 8ll) * kGroups * num_sms + tokens - 1) / tokens);
  if (segments > pieces) segments = pieces;
  const int segment_vecs = (pieces + segments - 1) / segments * GROUP;
  segments = (row_vecs + segment_vecs - 1) / segment_vecs;
  const long long items = (long long)tokens * segments;
  if (items > 0x7fffffffll - 32ll * num_sms) return cudaErrorInvalidValue;   // (a token in parts: few tokens)
  return launch_chained(unpermute_kernel<T, N, U, GROUP, kAhead>, dim3(grid_for((items + kGroups - 1) / kGroups, kAhead ? 4ll * num_sms : items)),
                        dim3(kMoveThreads), 0, stream, reinterpret_cast<const T*>(y), y_stride, pos, weights, w_stride,
                        reinterpret_cast<T*>(out), out_stride, (int)items, top_k, row_vecs, segments, segment_vecs);
}

template <typename T, int N>
cudaError_t launch_unpermute(const void* y, long long y_stride, const int* pos, const float* weights, long long w_stride, void* out,
                             long long out_stride, int tokens, int top_k, int hidden, int num_sms, cudaStream_t stream) {
  // loads of fewer bytes: more of them in flight (as many as leave the registers without spills)
  constexpr int U = sizeof(T) * N == 16 ? 1 : sizeof(T) == 4 ? 2 : N == 2 ? 3 : 4;
  const int row_vecs = hidden / N;
  // Short rows leave threads of a group of 128 idle.  us, groups of 32 / of 128: bf16 16384 rows of 512 27 / 47, 8192 of 1536 41 / 47, of
  // 2048 54 / 52, 4096 of 602 11 / 14, of 7168 91 / 86; fp32 16384 rows of 512, two choices 22 / 31, 8192 of 1024 52 / 46.
  const bool small = sizeof(T) == 2 ? row_vecs < 2 * U * kMoveThreads : row_vecs <= U * kMoveThreads;
  auto go = small ? launch_unpermute_group<T, N, U, 32> : launch_unpermute_group<T, N, U, kMoveThreads>;
  return go(y, y_stride, pos, weights, w_stride, out, out_stride, tokens, top_k, row_vecs, num_sms, stream);
}

// elements of a vector: 16 bytes, 4 bytes or one element, as far as all rows start on such a boundary (`bits`: addresses
// and pitches in bytes, or'ed)
template <typename T> int vector_elems(int hidden, uintptr_t bits) {
  const uintptr_t row = (uintptr_t)hidden * sizeof(T) | bits;
  return row % 16 == 0 ? 16 / (int)sizeof(T) : row % 4 == 0 ? 4 / (int)sizeof(T) : 1;
}

template <typename T>
cudaError_t unpermute_type(const void* y, long long y_stride, const int* pos, const float* weights, long long w_stride, void* out,
                           long long out_stride, int tokens, int top_k, int hidden, int num_sms, cudaStream_t stream) {
  constexpr int N16 = 16 / sizeof(T), N4 = 4 / sizeof(T);
  const int n = vector_elems<T>(hidden, reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(out) |
                                            (uintptr_t)(y_stride * sizeof(T)) | (uintptr_t)(out_stride * sizeof(T)));
  auto go = n == N16 ? launch_unpermute<T, N16> : n == N4 ? launch_unpermute<T, N4> : launch_unpermute<T, 1>;
  return go(y, y_stride, pos, weights, w_stride, out, out_stride, tokens, top_k, hidden, num_sms, stream);
}

template <typename T, int N, int U, int GROUP>
cudaError_t launch_unpermute_grad_group(const UnpermuteGrad<T>& p, int num_sms, cudaStream_t stream) {
  constexpr int kWarps = GROUP / 32, kGroups = kMoveThreads / GROUP;
  const int zero_rows = zero_rows_of((long long)p.row_vecs * N * (long long)sizeof(T));
  const long long items = p.tokens + (p.dy ? (p.rows + zero_rows * kWarps - 1) / (zero_rows * kWarps) : 0);
  if (items == 0) return cudaSuccess;
  return launch_chained(unpermute_grad_kernel<T, N, U, GROUP>, dim3(grid_for((items + kGroups - 1) / kGroups, 64ll * num_sms)),
                        dim3(kMoveThreads), 0, stream, p, zero_rows, items);
}

template <typename T, int N>
cudaError_t launch_unpermute_grad(UnpermuteGrad<T> p, int hidden, int num_sms, cudaStream_t stream) {
  // single elements: more loads in flight.  us, one at a time / four: 2048 tokens x 8 of 4097 bf16 104 / 80, fp32 132 / 108; pairs of
  // 16-bit elements gain nothing
  constexpr int U = N == 1 ? 4 : 1;
  p.row_vecs = hidden / N;
  // Many short rows by single warps.  us, groups of 32 / of 128, eight choices: bf16 16384 tokens of 512 71 / 98, 8192 of 1024 64 / 62,
  // 4097 of 601 21 / 31, 100 of 2048 16 / 5 (with elements one by one, see elem); fp32 16384 of 256 51 / 70, of
  // 512 with two choices 38 / 51, 8192 of 1024 93 / 88.
  const bool small = p.row_vecs < (U > 1 ? 2 : 1) * U * kMoveThreads + (sizeof(T) == 4) && p.tokens >= 4ll * num_sms;
  return small ? launch_unpermute_grad_group<T, N, U, 32>(p, num_sms, stream)
               : launch_unpermute_grad_group<T, N, U, kMoveThreads>(p, num_sms, stream);
}

template <typename T>
cudaError_t unpermute_grad_type(const void* dout, long long dout_stride, const void* y, long long y_stride, const float* weights,
                                long long w_stride, const int* pos, const int* pair, const int* used_rows, void* dy,
                                long long dy_stride, float* dw, long long tokens, long long rows, int top_k, int hidden,
                                int num_sms, cudaStream_t stream) {
  UnpermuteGrad<T> p;
  p.dout = reinterpret_cast<const T*>(dout);
  p.dout_stride = dout_stride;
  p.y = reinterpret_cast<const T*>(y);
  p.y_stride = y_stride;
  p.weights = weights;
  p.w_stride = w_stride;
  p.pos = pos;
  p.pair = pair;
  p.used_rows = used_rows;
  p.dy = reinterpret_cast<T*>(dy);
  p.dy_stride = dy_stride;
  p.dw = dw;
  p.tokens = tokens;
  p.rows = rows;
  p.top_k = top_k;
  p.row_vecs = 0;
  constexpr int N16 = 16 / sizeof(T), N4 = 4 / sizeof(T);
  uintptr_t bits = reinterpret_cast<uintptr_t>(dout) | (uintptr_t)(dout_stride * sizeof(T));
  if (dw) bits |= reinterpret_cast<uintptr_t>(y) | (uintptr_t)(y_stride * sizeof(T));
  if (dy) bits |= reinterpret_cast<uintptr_t>(dy) | (uintptr_t)(dy_stride * sizeof(T));
  const int n = vector_elems<T>(hidden, bits);
  auto go = n == N16 ? launch_unpermute_grad<T, N16> : n == N4 ? launch_unpermute_grad<T, N4> : launch_unpermute_grad<T, 1>;
  return go(p, hidden, num_sms, stream);
}

// tokens x top_k pairs and `rows` sorted rows that int32 tables can name
int order_ok(int64_t tokens, int top_k, int64_t rows) {
  if (tokens < 0 || top_k < 1 || rows < 0) return B200MOE_ERR_INVALID_ARGUMENT;
  if (top_k > kMaxSortTopK || tokens > 0x7fffffffll / top_k || rows > 0x7fffffffll) return B200MOE_ERR_UNSUPPORTED_SHAPE;
  return B200MOE_OK;
}

}  // namespace

cudaError_t configure_sort_rows() {
  return cudaFuncSetAttribute(sort_place_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sort_place_smem(kMaxSortExperts));
}

}  // namespace b200moe

using namespace b200moe;

extern "C" {

int64_t b200moe_sort_rows(int64_t tokens, int top_k, int e_local, int align) {
  if (order_ok(tokens, top_k, 0) != B200MOE_OK || e_local < 1 || e_local > kMaxSortExperts || align < 1 || align > 65536)
    return B200MOE_ERR_INVALID_ARGUMENT;
  const int64_t pairs = tokens * top_k;
  const int64_t rows = pairs + (int64_t)(align - 1) * (pairs < e_local ? pairs : e_local);
  return (rows + align - 1) / align * align;
}

int64_t b200moe_sort_workspace_bytes(int64_t tokens, int top_k, int e_local) {
  if (order_ok(tokens, top_k, 0) != B200MOE_OK || e_local < 1 || e_local > kMaxSortExperts) return B200MOE_ERR_INVALID_ARGUMENT;
  const SortPlan plan = sort_plan(tokens * top_k, 0);
  return plan.one_launch ? 0 : (int64_t)(plan.chunks + 1) * e_local * 4;
}

int b200moe_sort_tokens(const void* topk_ids, int ids_bits, int64_t ids_row_stride, int64_t tokens, int top_k, int e_local,
                        int local_expert_offset, int align, int32_t* counts, int32_t* offsets, int32_t* pos, int32_t* pair,
                        int64_t rows, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = order_ok(tokens, top_k, rows);
  if (rc != B200MOE_OK) return rc;
  if (!counts || !offsets || e_local < 1 || align < 1 || local_expert_offset < 0 || (ids_bits != 32 && ids_bits != 64))
    return B200MOE_ERR_INVALID_ARGUMENT;
  if (e_local > kMaxSortExperts || align > 65536) return B200MOE_ERR_UNSUPPORTED_SHAPE;
  if (tokens > 0 && (!topk_ids || !pos || !pair || ids_row_stride < top_k)) return B200MOE_ERR_INVALID_ARGUMENT;
  const int64_t need = b200moe_sort_rows(tokens, top_k, e_local, align);
  if (rows < need || need > 0x7fffffffll) return B200MOE_ERR_UNSUPPORTED_SHAPE;
  if (rows > 0 && !pair) return B200MOE_ERR_INVALID_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(topk_ids) % (ids_bits / 8) != 0 || reinterpret_cast<uintptr_t>(workspace) % 4 != 0 ||
      !words_aligned(counts, offsets, pos, pair))
    return B200MOE_ERR_MISALIGNED;
  const SortPlan plan = sort_plan(tokens * top_k, rows);
  if (!plan.one_launch) {
    if (!workspace) return B200MOE_ERR_INVALID_ARGUMENT;
    if (workspace_bytes < (size_t)(plan.chunks + 1) * e_local * 4) return B200MOE_ERR_WORKSPACE_TOO_SMALL;
  }
  int num_sms = 0;
  if ((rc = ensure_device(&num_sms)) != B200MOE_OK) return rc;
  SortParams p;
  p.ids = topk_ids;
  p.ids_stride = ids_row_stride;
  p.pairs = (int)(tokens * top_k);
  p.top_k = top_k;
  p.contiguous = ids_row_stride == top_k || tokens <= 1;
  p.wide = ids_bits == 64;
  p.vec_pair = align % 4 == 0 && reinterpret_cast<uintptr_t>(pair) % 16 == 0;
  p.local_off = local_expert_offset;
  p.e_local = e_local;
  p.align = align;
  p.rows = (int)rows;
  p.counts = counts;
  p.offsets = offsets;
  p.pos = pos;
  p.pair = pair;
  p.chunks = plan.chunks;
  p.scanned = !plan.one_launch && (long long)plan.chunks * e_local > kSortScanCounters;
  p.chunk_counts = plan.one_launch ? nullptr : reinterpret_cast<int*>(workspace);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  CUDA_TRY(launch_sort(p, plan, st));
  return B200MOE_OK;
}

int b200moe_permute_rows(const void* x, int64_t x_row_bytes, int64_t row_bytes, int elem_bytes, int64_t tokens, int top_k,
                         const int32_t* pos, const int32_t* pair, const int32_t* offsets, int e_local, int64_t rows, void* y,
                         int64_t y_row_bytes, int zero_tail, void* stream) {
  int rc = order_ok(tokens, top_k, rows);
  if (rc != B200MOE_OK) return rc;
  if ((elem_bytes != 1 && elem_bytes != 2 && elem_bytes != 4) || row_bytes < 0 || row_bytes % elem_bytes != 0 || e_local < 1)
    return B200MOE_ERR_INVALID_ARGUMENT;
  if (row_bytes > 0x3fffffff) return B200MOE_ERR_UNSUPPORTED_SHAPE;
  if (rows == 0 || row_bytes == 0) return B200MOE_OK;
  if (!pair || !offsets || !y || y_row_bytes < row_bytes || (tokens > 0 && (!x || !pos || x_row_bytes < row_bytes)))
    return B200MOE_ERR_INVALID_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(x) | (uintptr_t)x_row_bytes | reinterpret_cast<uintptr_t>(y) | (uintptr_t)y_row_bytes) % elem_bytes != 0 ||
      !words_aligned(pos, pair, offsets))
    return B200MOE_ERR_MISALIGNED;
  int num_sms = 0;
  if ((rc = ensure_device(&num_sms)) != B200MOE_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  RowMove p;
  p.src = reinterpret_cast<const uint8_t*>(x);
  p.src_stride = x_row_bytes;
  p.dst = reinterpret_cast<uint8_t*>(y);
  p.dst_stride = y_row_bytes;
  p.pos = pos;
  p.pair = pair;
  p.used_rows = offsets + e_local;
  p.tokens = tokens;
  p.rows = rows;
  p.top_k = top_k;
  p.zero_tail = zero_tail != 0;
  // what a lane moves at once: 16 bytes, or the largest smaller part on whose boundaries all rows start
  const uintptr_t bits = reinterpret_cast<uintptr_t>(x) | (uintptr_t)x_row_bytes | reinterpret_cast<uintptr_t>(y) |
                         (uintptr_t)y_row_bytes | (uintptr_t)row_bytes;
  const int vec = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : bits % 2 == 0 ? 2 : 1;
  p.row_vecs = (int)(row_bytes / vec);
  if (vec == 16)
    CUDA_TRY((launch_permute_rows<uint4, 2>(p, st)));
  else if (vec == 4)
    CUDA_TRY((launch_permute_rows<uint32_t, 4>(p, st)));
  else if (vec == 2)
    CUDA_TRY((launch_permute_rows<uint16_t, 8>(p, st)));
  else
    CUDA_TRY((launch_permute_rows<uint8_t, 8>(p, st)));
  return B200MOE_OK;
}

int b200moe_unpermute_rows(const void* y, int dtype, int64_t y_row_stride, const int32_t* pos, const float* weights,
                           int64_t w_row_stride, int64_t tokens, int top_k, int hidden, void* out, int64_t out_row_stride,
                           void* stream) {
  int rc = order_ok(tokens, top_k, 0);
  if (rc != B200MOE_OK) return rc;
  if (hidden < 0 || (dtype != B200MOE_F32 && dtype != B200MOE_BF16 && dtype != B200MOE_F16)) return B200MOE_ERR_INVALID_ARGUMENT;
  if (tokens == 0 || hidden == 0) return B200MOE_OK;
  if (!y || !pos || !out || y_row_stride < hidden || out_row_stride < hidden || (weights && w_row_stride < top_k))
    return B200MOE_ERR_INVALID_ARGUMENT;
  const uintptr_t size = dtype == B200MOE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(y) % size != 0 || reinterpret_cast<uintptr_t>(out) % size != 0 || !words_aligned(pos, weights))
    return B200MOE_ERR_MISALIGNED;
  int num_sms = 0;
  if ((rc = ensure_device(&num_sms)) != B200MOE_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  auto go = dtype == B200MOE_F32 ? unpermute_type<float> : dtype == B200MOE_BF16 ? unpermute_type<__nv_bfloat16> : unpermute_type<__half>;
  CUDA_TRY(go(y, y_row_stride, pos, weights, w_row_stride, out, out_row_stride, (int)tokens, top_k, hidden, num_sms, st));
  return B200MOE_OK;
}

int b200moe_unpermute_grad(const void* dout, int dtype, int64_t dout_row_stride, const void* y, int64_t y_row_stride,
                           const float* weights, int64_t w_row_stride, const int32_t* pos, const int32_t* pair,
                           const int32_t* offsets, int e_local, int64_t tokens, int top_k, int hidden, int64_t rows, void* dy,
                           int64_t dy_row_stride, float* dw, void* stream) {
  int rc = order_ok(tokens, top_k, rows);
  if (rc != B200MOE_OK) return rc;
  if (hidden < 0 || e_local < 1 || (dtype != B200MOE_F32 && dtype != B200MOE_BF16 && dtype != B200MOE_F16))
    return B200MOE_ERR_INVALID_ARGUMENT;
  if (!dy && !dw) return B200MOE_OK;
  if (rows == 0) dy = nullptr;
  if (tokens > 0 && (!pos || (hidden > 0 && (!dout || dout_row_stride < hidden)) || (weights && w_row_stride < top_k)))
    return B200MOE_ERR_INVALID_ARGUMENT;
  if ((dy && hidden > 0 && (dy_row_stride < hidden || !pair || !offsets)) ||
      (dw && hidden > 0 && rows > 0 && tokens > 0 && (!y || y_row_stride < hidden)))
    return B200MOE_ERR_INVALID_ARGUMENT;
  const uintptr_t size = dtype == B200MOE_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(dout) | reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(dy)) % size != 0 ||
      !words_aligned(pos, pair, offsets, weights, dw))
    return B200MOE_ERR_MISALIGNED;
  int num_sms = 0;
  if ((rc = ensure_device(&num_sms)) != B200MOE_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  auto go = dtype == B200MOE_F32 ? unpermute_grad_type<float>
                                 : dtype == B200MOE_BF16 ? unpermute_grad_type<__nv_bfloat16> : unpermute_grad_type<__half>;
  CUDA_TRY(go(dout, dout_row_stride, y, y_row_stride, weights, w_row_stride, pos, pair, offsets ? offsets + e_local : nullptr, dy,
              dy_row_stride, dw, tokens, rows, top_k, hidden, num_sms, st));
  return B200MOE_OK;
}

}  // extern "C"
