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
constexpr int kSortThreads = 1024;
constexpr int kSortChunk = 4096;                 // pairs of a CTA, until there is one for each SM
constexpr int kSortOneBlock = 8192;              // up to so many pairs one CTA sorts alone, in one launch

struct SortParams {
  const void* ids;
  long long ids_stride;
  long long pairs;
  int top_k;
  int wide;                                      // int64 ids
  int local_off, e_local, align;
  long long rows;                                // length of `pair`
  int* counts;                                   // [e_local]
  int* offsets;                                  // [e_local + 1]
  int* pos;                                      // [pairs]
  int* pair;                                     // [rows]
  int* chunk_counts;                             // [chunks][e_local]
  long long chunk;                               // pairs of a CTA
  int chunks;
};

__device__ __forceinline__ int local_expert(const SortParams& p, long long i) {
  const long long t = i / p.top_k;
  const long long at = t * p.ids_stride + (i - t * p.top_k);
  const long long id = p.wide ? reinterpret_cast<const long long*>(p.ids)[at] : (long long)reinterpret_cast<const int*>(p.ids)[at];
  return id >= p.local_off && id < (long long)p.local_off + p.e_local ? (int)(id - p.local_off) : -1;
}

// Pairs [begin, end) of one warp, counted per expert into its own row of shared counters.
__device__ __forceinline__ void count_range(const SortParams& p, long long begin, long long end, int lane, int* cnt) {
  for (long long i = begin + lane; i < end; i += 32) {
    const int e = local_expert(p, i);
    if (e >= 0) atomicAdd(cnt + e, 1);
  }
}

__device__ __forceinline__ void warp_range(const SortParams& p, int warp, int warps, long long* begin, long long* end) {
  const long long first = (long long)blockIdx.x * p.chunk, last = min(first + p.chunk, p.pairs);
  const long long share = ((last - first + warps - 1) / warps + 31) / 32 * 32;
  *begin = min(first + warp * share, last);
  *end = min(*begin + share, last);
}

__global__ void __launch_bounds__(kSortThreads)
sort_count_kernel(const __grid_constant__ SortParams p) {
  extern __shared__ int s_cnt[];                 // [e_local]
  for (int e = threadIdx.x; e < p.e_local; e += blockDim.x) s_cnt[e] = 0;
  __syncthreads();
  chain_wait();
  chain_release();
  long long begin, end;
  warp_range(p, threadIdx.x >> 5, blockDim.x >> 5, &begin, &end);
  count_range(p, begin, end, threadIdx.x & 31, s_cnt);
  __syncthreads();
  for (int e = threadIdx.x; e < p.e_local; e += blockDim.x) p.chunk_counts[(size_t)blockIdx.x * p.e_local + e] = s_cnt[e];
}

// Exclusive sum over the CTA's 1024 threads.
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
  if (warp == 0) {
    int w = s_warp[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += up;
    }
    s_warp[lane] = w;
  }
  __syncthreads();
  *total = s_warp[31];
  return sum - v + (warp > 0 ? s_warp[warp - 1] : 0);
}

// Places the pairs of a CTA's chunk.  Each warp owns a run of the chunk and a row of counters: counted once, turned into
// first rows by a sum over the warps, then walked again, 32 pairs at a time, a pair's place among its warp's by a match of the
// expert.  A call of one chunk needs no kernel before it.
__global__ void __launch_bounds__(kSortThreads)
sort_place_kernel(const __grid_constant__ SortParams p, int warps) {
  extern __shared__ int smem[];
  int* s_next = smem;                            // [warps][e_local]
  int* s_total = s_next + warps * p.e_local;     // [e_local] pairs of all chunks
  int* s_before = s_total + p.e_local;           // [e_local] pairs of the chunks before this one
  int* s_first = s_before + p.e_local;           // [e_local + 1]
  int* s_warp = s_first + p.e_local + 1;         // [32]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, E = p.e_local;
  for (int i = threadIdx.x; i < (warps + 2) * E; i += blockDim.x) smem[i] = 0;
  __syncthreads();
  chain_wait();
  chain_release();
  long long begin = 0, end = 0;
  if (warp < warps) {
    warp_range(p, warp, warps, &begin, &end);
    count_range(p, begin, end, lane, s_next + warp * E);
  }
  if (p.chunks > 1) {                            // all threads: parts of the columns of the chunk counts
    const int parts = blockDim.x / E > 0 ? blockDim.x / E : 1;
    const int per = (p.chunks + parts - 1) / parts;
    for (int i = threadIdx.x; i < parts * E; i += blockDim.x) {
      const int e = i % E, c0 = i / E * per, c1 = min(c0 + per, p.chunks);
      int total = 0, before = 0;
#pragma unroll 8
      for (int c = c0; c < c1; ++c) {
        const int n = p.chunk_counts[(size_t)c * E + e];
        total += n;
        before += c < (int)blockIdx.x ? n : 0;
      }
      atomicAdd(s_total + e, total);
      atomicAdd(s_before + e, before);
    }
  }
  __syncthreads();
  int total = 0;
  if (threadIdx.x < E) {
    int sum = 0;                                 // counters of a warp become the number of pairs in the warps before it
    for (int w = 0; w < warps; ++w) {
      const int n = s_next[w * E + threadIdx.x];
      s_next[w * E + threadIdx.x] = sum;
      sum += n;
    }
    total = p.chunks > 1 ? s_total[threadIdx.x] : sum;
  }
  const int padded = (int)(((long long)total + p.align - 1) / p.align * p.align);
  int used;
  const int first = block_exclusive_sum(padded, s_warp, &used);
  if (threadIdx.x < E) {
    s_total[threadIdx.x] = total;
    s_first[threadIdx.x] = first;
    const int base = first + s_before[threadIdx.x];
    for (int w = 0; w < warps; ++w) s_next[w * E + threadIdx.x] += base;
    if (blockIdx.x == 0) {
      p.counts[threadIdx.x] = total;
      p.offsets[threadIdx.x] = first;
    }
  }
  if (threadIdx.x == 0) {
    s_first[E] = used;
    if (blockIdx.x == 0) p.offsets[E] = used;
  }
  __syncthreads();
  if (warp < warps) {
    int* next = s_next + warp * E;
    for (long long i0 = begin; i0 < end; i0 += 32) {
      const long long i = i0 + lane;
      const int e = i < end ? local_expert(p, i) : -1;
      const unsigned same = __match_any_sync(0xffffffffu, e);
      int row = -1;
      if (e >= 0) row = next[e] + __popc(same & ((1u << lane) - 1u));
      __syncwarp();
      if (e >= 0 && lane == 31 - __clz(same)) next[e] = row + 1;
      __syncwarp();
      if (i < end) p.pos[i] = row;
      if (row >= 0) p.pair[row] = (int)i;
    }
  }
  // rows that no pair takes: the padding of every chunks-th expert, and a share of what lies behind the last segment
  for (int e = (int)blockIdx.x + warp * p.chunks; e < E; e += p.chunks * (blockDim.x >> 5))
    for (int r = s_first[e] + s_total[e] + lane; r < s_first[e + 1]; r += 32) p.pair[r] = -1;
  for (long long r = s_first[E] + (long long)blockIdx.x * blockDim.x + threadIdx.x; r < p.rows; r += (long long)p.chunks * blockDim.x)
    p.pair[r] = -1;
}

int sort_warps(int e_local) { return e_local <= 256 ? 32 : 16; }
size_t sort_place_smem(int e_local) { return ((size_t)(sort_warps(e_local) + 3) * e_local + 1 + 32) * 4; }

// One CTA up to kSortOneBlock pairs, else chunks of kSortChunk pairs, larger ones where that makes more CTAs than SMs (every CTA
// reads the counts of all).
void sort_chunks(long long pairs, int num_sms, long long* chunk, int* chunks) {
  if (pairs <= kSortOneBlock) {
    *chunk = pairs;
    *chunks = 1;
    return;
  }
  long long c = (pairs + num_sms - 1) / num_sms;
  c = c < kSortChunk ? kSortChunk : (c + 31) / 32 * 32;
  *chunk = c;
  *chunks = (int)((pairs + c - 1) / c);
}
constexpr int kSortMaxChunks = 256;              // more than any sm_100 part has SMs

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
constexpr int kZeroRows = 4;                     // sorted rows that a warp looks at for empty ones

// Rows of `dst` without a pair become zero; `item` counts groups of kZeroRows rows.
template <typename V>
__device__ __forceinline__ void zero_empty_rows(const int* pair, const int* used_rows, long long rows, int zero_tail, uint8_t* dst,
                                                long long dst_stride, int row_vecs, long long item, int lane) {
  const long long r0 = item * kZeroRows;
  const long long limit = zero_tail ? rows : (long long)*used_rows;
  bool empty = false;
  if (lane < kZeroRows && r0 + lane < rows && r0 + lane < limit) empty = pair[r0 + lane] < 0;
  unsigned todo = __ballot_sync(0xffffffffu, empty);
  while (todo) {
    const int j = __ffs(todo) - 1;
    todo &= todo - 1;
    V* d = reinterpret_cast<V*>(dst + (r0 + j) * dst_stride);
    for (int v = lane; v < row_vecs; v += 32) d[v] = V{};
  }
}

// A warp takes U x 32 vectors of one token's row into registers and stores them to the token's sorted rows.
template <typename V, int U>
__global__ void __launch_bounds__(kMoveThreads)
permute_kernel(const __grid_constant__ RowMove p, int segments, long long move_items, long long items) {
  chain_wait();
  chain_release();
  const int lane = threadIdx.x & 31;
  const long long step = (long long)gridDim.x * (kMoveThreads / 32);
  for (long long w = (long long)blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5); w < items; w += step) {
    if (w >= move_items) {
      zero_empty_rows<V>(p.pair, p.used_rows, p.rows, p.zero_tail, p.dst, p.dst_stride, p.row_vecs, w - move_items, lane);
      continue;
    }
    const long long t = w / segments;
    const int v0 = (int)(w - t * segments) * (U * 32) + lane;
    const int mine = lane < p.top_k ? p.pos[t * p.top_k + lane] : -1;
    const V* src = reinterpret_cast<const V*>(p.src + t * p.src_stride);
    V x[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v0 + u * 32 < p.row_vecs) x[u] = __ldg(src + v0 + u * 32);
    for (int k = 0; k < p.top_k; ++k) {
      const int row = __shfl_sync(0xffffffffu, mine, k);
      if (row < 0) continue;
      V* dst = reinterpret_cast<V*>(p.dst + row * p.dst_stride);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (v0 + u * 32 < p.row_vecs) dst[v0 + u * 32] = x[u];
    }
  }
}

// ---- sums over a token's rows ----

template <typename T, int N> struct alignas(sizeof(T) * N) Pack { T v[N]; };

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename P>
__device__ __forceinline__ P load_pack(const P* p) {
  P r;
  if constexpr (sizeof(P) == 16) {
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
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

// A warp takes 32 vectors of one token's output row.
template <typename T, int N>
__global__ void __launch_bounds__(kMoveThreads)
unpermute_kernel(const T* __restrict__ y, long long y_stride, const int* __restrict__ pos, const float* __restrict__ weights,
                 long long w_stride, T* __restrict__ out, long long out_stride, long long tokens, int top_k, int row_vecs,
                 int segments) {
  using P = Pack<T, N>;
  chain_wait();
  chain_release();
  const int lane = threadIdx.x & 31;
  const long long items = tokens * segments, step = (long long)gridDim.x * (kMoveThreads / 32);
  for (long long w = (long long)blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5); w < items; w += step) {
    const long long t = w / segments;
    const int v = (int)(w - t * segments) * 32 + lane;
    const int row_k = lane < top_k ? pos[t * top_k + lane] : -1;
    const float w_k = weights && lane < top_k ? weights[t * w_stride + lane] : 1.f;
    float acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
    for (int k0 = 0; k0 < top_k; k0 += kSumBatch) {
      P x[kSumBatch];
#pragma unroll
      for (int j = 0; j < kSumBatch; ++j) {
        const int row = __shfl_sync(0xffffffffu, row_k, (k0 + j) & 31);
        if (k0 + j < top_k && row >= 0 && v < row_vecs)
          x[j] = load_pack(reinterpret_cast<const P*>(y + (long long)row * y_stride) + v);
      }
#pragma unroll
      for (int j = 0; j < kSumBatch; ++j) {
        const int row = __shfl_sync(0xffffffffu, row_k, (k0 + j) & 31);
        const float wt = __shfl_sync(0xffffffffu, w_k, (k0 + j) & 31);
        if (k0 + j < top_k && row >= 0) {
#pragma unroll
          for (int i = 0; i < N; ++i) acc[i] = fmaf(wt, to_float(x[j].v[i]), acc[i]);
        }
      }
    }
    if (v < row_vecs) {
      P r;
#pragma unroll
      for (int i = 0; i < N; ++i) r.v[i] = from_float<T>(acc[i]);
      store_pack(reinterpret_cast<P*>(out + t * out_stride) + v, r);
    }
  }
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

// One CTA per token: its row of dout is read once (top_k <= 8), each sorted row of y read and of dy written once; the dots are
// summed by shuffles and over the four warps in a fixed order.
template <typename T, int N>
__global__ void __launch_bounds__(kMoveThreads)
unpermute_grad_kernel(const __grid_constant__ UnpermuteGrad<T> p, long long items) {
  using P = Pack<T, N>;
  constexpr int kWarps = kMoveThreads / 32;
  __shared__ float s_dot[kWarps][kSumBatch];
  chain_wait();
  chain_release();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (long long t = blockIdx.x; t < items; t += gridDim.x) {
    if (t >= p.tokens) {
      zero_empty_rows<P>(p.pair, p.used_rows, p.rows, 1, reinterpret_cast<uint8_t*>(p.dy), p.dy_stride * (long long)sizeof(T),
                         p.row_vecs, (t - p.tokens) * kWarps + warp, lane);
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
      for (int v = threadIdx.x; v < p.row_vecs; v += kMoveThreads) {
        const P d = load_pack(dout + v);
        P x[kSumBatch];
        if (p.dw) {
#pragma unroll
          for (int j = 0; j < kSumBatch; ++j)
            if (row[j] >= 0) x[j] = load_pack(reinterpret_cast<const P*>(p.y + row[j] * p.y_stride) + v);
        }
#pragma unroll
        for (int j = 0; j < kSumBatch; ++j) {
          if (row[j] < 0) continue;
          if (p.dw) {
#pragma unroll
            for (int i = 0; i < N; ++i) dot[j] = fmaf(to_float(d.v[i]), to_float(x[j].v[i]), dot[j]);
          }
          if (p.dy) {
            P r;
#pragma unroll
            for (int i = 0; i < N; ++i) r.v[i] = from_float<T>(wt[j] * to_float(d.v[i]));
            store_pack(reinterpret_cast<P*>(p.dy + row[j] * p.dy_stride) + v, r);
          }
        }
      }
      if (p.dw) {
#pragma unroll
        for (int j = 0; j < kSumBatch; ++j) {
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], o);
          if (lane == 0) s_dot[warp][j] = dot[j];
        }
        __syncthreads();
        if (threadIdx.x < kSumBatch && k0 + threadIdx.x < p.top_k) {
          float sum = 0.f;
          for (int w = 0; w < kWarps; ++w) sum += s_dot[w][threadIdx.x];
          p.dw[t * p.top_k + k0 + threadIdx.x] = sum;
        }
        __syncthreads();
      }
    }
  }
}

bool aligned16(const void* p, long long stride_bytes) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride_bytes % 16 == 0;
}

unsigned grid_for(long long items, long long most) { return (unsigned)(items < most ? items : most); }

template <typename V, int U>
cudaError_t launch_permute_rows(const RowMove& p, bool zero, int num_sms, cudaStream_t stream) {
  const int segments = (p.row_vecs + U * 32 - 1) / (U * 32);
  const long long move_items = p.tokens * segments;
  const long long items = move_items + (zero ? (p.rows + kZeroRows - 1) / kZeroRows : 0);
  if (items == 0) return cudaSuccess;
  constexpr int kWarps = kMoveThreads / 32;
  return launch_chained(permute_kernel<V, U>, dim3(grid_for((items + kWarps - 1) / kWarps, 64ll * num_sms)), dim3(kMoveThreads), 0,
                        stream, p, segments, move_items, items);
}

template <typename T, int N>
cudaError_t launch_unpermute(const void* y, long long y_stride, const int* pos, const float* weights, long long w_stride, void* out,
                             long long out_stride, long long tokens, int top_k, int hidden, int num_sms, cudaStream_t stream) {
  const int row_vecs = hidden / N, segments = (row_vecs + 31) / 32;
  constexpr int kWarps = kMoveThreads / 32;
  const long long blocks = (tokens * segments + kWarps - 1) / kWarps;
  return launch_chained(unpermute_kernel<T, N>, dim3(grid_for(blocks, 64ll * num_sms)), dim3(kMoveThreads), 0, stream,
                        reinterpret_cast<const T*>(y), y_stride, pos, weights, w_stride, reinterpret_cast<T*>(out), out_stride,
                        tokens, top_k, row_vecs, segments);
}

template <typename T>
cudaError_t unpermute_type(const void* y, long long y_stride, const int* pos, const float* weights, long long w_stride, void* out,
                           long long out_stride, long long tokens, int top_k, int hidden, int num_sms, cudaStream_t stream) {
  constexpr int N = 16 / sizeof(T);
  const bool vec = hidden % N == 0 && aligned16(y, y_stride * (long long)sizeof(T)) && aligned16(out, out_stride * (long long)sizeof(T));
  return vec ? launch_unpermute<T, N>(y, y_stride, pos, weights, w_stride, out, out_stride, tokens, top_k, hidden, num_sms, stream)
             : launch_unpermute<T, 1>(y, y_stride, pos, weights, w_stride, out, out_stride, tokens, top_k, hidden, num_sms, stream);
}

template <typename T, int N>
cudaError_t launch_unpermute_grad(UnpermuteGrad<T> p, int hidden, int num_sms, cudaStream_t stream) {
  p.row_vecs = hidden / N;
  constexpr int kWarps = kMoveThreads / 32;
  const long long items = p.tokens + (p.dy ? (p.rows + kZeroRows * kWarps - 1) / (kZeroRows * kWarps) : 0);
  if (items == 0) return cudaSuccess;
  return launch_chained(unpermute_grad_kernel<T, N>, dim3(grid_for(items, 64ll * num_sms)), dim3(kMoveThreads), 0, stream, p, items);
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
  constexpr int N = 16 / sizeof(T);
  const long long b = sizeof(T);
  const bool vec = hidden % N == 0 && aligned16(dout, dout_stride * b) && (!dw || aligned16(y, y_stride * b)) &&
                   (!dy || aligned16(dy, dy_stride * b));
  return vec ? launch_unpermute_grad<T, N>(p, hidden, num_sms, stream) : launch_unpermute_grad<T, 1>(p, hidden, num_sms, stream);
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

int64_t b200moe_sort_workspace_bytes(int e_local) {
  if (e_local < 1 || e_local > kMaxSortExperts) return B200MOE_ERR_INVALID_ARGUMENT;
  return (int64_t)kSortMaxChunks * e_local * 4;
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
  if (reinterpret_cast<uintptr_t>(topk_ids) % (ids_bits / 8) != 0 || reinterpret_cast<uintptr_t>(workspace) % 4 != 0)
    return B200MOE_ERR_MISALIGNED;
  int num_sms = 0;
  if ((rc = ensure_device(&num_sms)) != B200MOE_OK) return rc;
  SortParams p;
  p.ids = topk_ids;
  p.ids_stride = ids_row_stride;
  p.pairs = tokens * top_k;
  p.top_k = top_k;
  p.wide = ids_bits == 64;
  p.local_off = local_expert_offset;
  p.e_local = e_local;
  p.align = align;
  p.rows = rows;
  p.counts = counts;
  p.offsets = offsets;
  p.pos = pos;
  p.pair = pair;
  p.chunk_counts = reinterpret_cast<int*>(workspace);
  sort_chunks(p.pairs, num_sms < kSortMaxChunks ? num_sms : kSortMaxChunks, &p.chunk, &p.chunks);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (p.chunks > 1) {
    if (!workspace) return B200MOE_ERR_INVALID_ARGUMENT;
    if (workspace_bytes < (size_t)p.chunks * e_local * 4) return B200MOE_ERR_WORKSPACE_TOO_SMALL;
    CUDA_TRY(launch_chained(sort_count_kernel, dim3(p.chunks), dim3(kSortThreads), (size_t)e_local * 4, st, p));
  }
  CUDA_TRY(launch_chained(sort_place_kernel, dim3(p.chunks), dim3(kSortThreads), sort_place_smem(e_local), st, p,
                          sort_warps(e_local)));
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
  if ((reinterpret_cast<uintptr_t>(x) | (uintptr_t)x_row_bytes | reinterpret_cast<uintptr_t>(y) | (uintptr_t)y_row_bytes) % elem_bytes != 0)
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
  const bool vec = row_bytes % 16 == 0 && aligned16(x, x_row_bytes) && aligned16(y, y_row_bytes);
  p.row_vecs = (int)(row_bytes / (vec ? 16 : elem_bytes));
  if (vec)
    CUDA_TRY((launch_permute_rows<uint4, 1>(p, true, num_sms, st)));
  else if (elem_bytes == 4)
    CUDA_TRY((launch_permute_rows<uint32_t, 4>(p, true, num_sms, st)));
  else if (elem_bytes == 2)
    CUDA_TRY((launch_permute_rows<uint16_t, 4>(p, true, num_sms, st)));
  else
    CUDA_TRY((launch_permute_rows<uint8_t, 4>(p, true, num_sms, st)));
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
  if (reinterpret_cast<uintptr_t>(y) % size != 0 || reinterpret_cast<uintptr_t>(out) % size != 0) return B200MOE_ERR_MISALIGNED;
  int num_sms = 0;
  if ((rc = ensure_device(&num_sms)) != B200MOE_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  auto go = dtype == B200MOE_F32 ? unpermute_type<float> : dtype == B200MOE_BF16 ? unpermute_type<__nv_bfloat16> : unpermute_type<__half>;
  CUDA_TRY(go(y, y_row_stride, pos, weights, w_row_stride, out, out_row_stride, tokens, top_k, hidden, num_sms, st));
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
  if ((reinterpret_cast<uintptr_t>(dout) | reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(dy)) % size != 0)
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
