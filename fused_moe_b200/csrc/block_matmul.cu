// Dense product of e4m3 matrices with block scales on tcgen05 tensor cores.
//
//   out[m,n] = sum_b sa[m,b] sb[n/128,b] * ( sum_{k in block b} a[m,k] b[n,k] ),   blocks of 128 along K
//
// The scales are arbitrary fp32 numbers, so they cannot ride on the MMA: a K block's raw dot products are made in tensor
// memory from zero, read back and folded into fp32 registers with one FMA each, the factor being one number per row (= TMEM
// lane = thread) and 128-column slab.
//
// Two kernels: 128 x 128 tiles, one CTA on an SM with four accumulators or two with two each, the K blocks of a tile divided over a
// cluster where tiles are few; and 256 x 256 tiles of a CTA pair (cta_group::2) where there are enough of them.
//
// Few rows are bound by the weights' bytes and, below some 30 MB of them, by latency: one row through 4096 x 7168 takes 9.5 us from
// HBM (29 MB, 4.5 us at the copy rate; 8.2 us from L2), through 7168 x 16384 24.7 us (117 MB, 17.9).  Many rows are bound by the
// hand-offs between tensor cores and promotion: 8192 x 4096 x 7168 takes 203 to 222 us in a burst (by data and clock; 254 repeated, at
// the power limit), 2.2 to 2.4 PFLOP/s, some 1000 cycles for a K block of a pair's tile whose MMAs take 512.  An accumulator's way
// round - issue 200 cycles, MMAs 260 to 510, the look at the barrier 200 to 300, read-back 250 to 300, the counter's way back 200 and
// more - is longer than the MMAs of the other one, and a pair's two of 256 x 256 leave no room in tensor memory for a third.
#include "common.cuh"
#include "host.cuh"
#include "kernels.cuh"

namespace b200moe {

namespace {

constexpr int kTile = 128;
constexpr int kOperandBytes = kTile * kBlockK;   // 16 KiB
constexpr int kStageBytes = 2 * kOperandBytes;
constexpr int kMaxSplit = 8;
// What a row becomes whose sum a bounded wait cut short: nothing that could pass for a result.
constexpr float kGivenUp = __builtin_nanf("");

struct MatmulParams {
  CUtensorMap tmap_a, tmap_b;
  const float* a_scale;
  const float* b_scale;
  long long as_m, as_kb, bs_n, bs_kb;
  int M, N, kblocks;
  int m_tiles, n_tiles;
  int split;                                     // CTAs of a cluster, each with a part of the K blocks
  int box_rows;                                  // 128 x 128 tiles: rows of A that a copy brings
  void* out;
  int out_dtype;
  long long out_stride;
  int vec_out;                                   // rows of `out` start on 32-byte (2) or 16-byte (1) boundaries, or neither (0)
  int* status;                                   // device-accessible int32[2], or null
};

__device__ __forceinline__ void st_cluster_v4(uint32_t addr, float a, float b, float c, float d) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}
__device__ __forceinline__ void st_cluster_s32(uint32_t addr, int v) {
  asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ float4 ld_shared_v4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cta.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ uint32_t pack16(int dtype, float x, float y) {
  uint32_t w;
  if (dtype == B200MOE_BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    memcpy(&w, &h, 4);
  } else {
    const __half2 h = __floats2half2_rn(x, y);
    memcpy(&w, &h, 4);
  }
  return w;
}

// Columns [n, n + 4) of row m, of which those below N exist.
__device__ __forceinline__ void store4(const MatmulParams& p, int m, int n, float4 v) {
  if (m >= p.M || n >= p.N) return;
  const bool whole = p.vec_out && n + 4 <= p.N;
  if (p.out_dtype == B200MOE_F32) {
    float* dst = reinterpret_cast<float*>(p.out) + (size_t)m * p.out_stride + n;
    if (whole) {
      *reinterpret_cast<float4*>(dst) = v;
    } else {
      dst[0] = v.x;
      if (n + 1 < p.N) dst[1] = v.y;
      if (n + 2 < p.N) dst[2] = v.z;
      if (n + 3 < p.N) dst[3] = v.w;
    }
    return;
  }
  uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + (size_t)m * p.out_stride + n;
  const uint32_t lo = pack16(p.out_dtype, v.x, v.y), hi = pack16(p.out_dtype, v.z, v.w);
  if (whole) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
  } else {
    dst[0] = (uint16_t)lo;
    if (n + 1 < p.N) dst[1] = (uint16_t)(lo >> 16);
    if (n + 2 < p.N) dst[2] = (uint16_t)hi;
    if (n + 3 < p.N) dst[3] = (uint16_t)(hi >> 16);
  }
}

// Columns [n, n + 128) of row m for a row given up.
__device__ __forceinline__ void store_given_up(const MatmulParams& p, int m, int n) {
#pragma unroll 1
  for (int i = 0; i < kTile; i += 4) store4(p, m, n + i, make_float4(kGivenUp, kGivenUp, kGivenUp, kGivenUp));
}

// A row's word i (of 64 or 128), zero behind the last.
template <bool F32>
__device__ __forceinline__ uint32_t row_word(int out_dtype, const float2* v, int i) {
  if (i >= (F32 ? kTile : kTile / 2)) return 0u;
  return F32 ? __float_as_uint(i & 1 ? v[i / 2].y : v[i / 2].x) : pack16(out_dtype, v[i].x, v[i].y);
}

// `bytes` of a row from one thread, 32 bytes (a sector) at a time: up to the first such boundary, and behind the last, in parts
// of 2, 4, 8 and 16 bytes, each where the address asks for it and the row has as many left.  What goes to a sector is taken out of
// the words by a shift of up to seven of them (and, for 16-bit elements, half of one).  M x 2047 in bf16 (through shared memory by
// single elements / so): M 8192, K 512 66 / 25 us, M 4096, K 2048 38 / 23; in fp32 49 / 30, 37 / 26.
template <bool F32>
__device__ __forceinline__ void store_row_shifted(uint8_t* dst, int out_dtype, const float2* v, int bytes) {
  uint32_t at = (uint32_t)reinterpret_cast<uintptr_t>(dst);
  const bool c2 = !F32 && (at & 2) && bytes >= 2;
  at += c2 ? 2 : 0, bytes -= c2 ? 2 : 0;
  const bool c4 = (at & 4) && bytes >= 4;
  at += c4 ? 4 : 0, bytes -= c4 ? 4 : 0;
  const bool c8 = (at & 8) && bytes >= 8;
  at += c8 ? 8 : 0, bytes -= c8 ? 8 : 0;
  const bool c16 = (at & 16) && bytes >= 16;
  bytes -= c16 ? 16 : 0;
  uint32_t next[8];                                // the window's second half
#pragma unroll
  for (int j = 0; j < 8; ++j) next[j] = row_word<F32>(out_dtype, v, j);
#pragma unroll
  for (int i = -8; i < (F32 ? kTile : kTile / 2); i += 8) {
    uint32_t x[16];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = next[j];
      next[j] = row_word<F32>(out_dtype, v, i + 8 + j);
      x[8 + j] = next[j];
    }
    if (i < 0) {                                   // before the first boundary
      if (c2) *reinterpret_cast<uint16_t*>(dst) = (uint16_t)x[0];
    }
    if (!F32) {
#pragma unroll
      for (int j = 0; j < 15; ++j) x[j] = __funnelshift_r(x[j], x[j + 1], c2 ? 16 : 0);
    }
    if (i < 0) {
      dst += c2 ? 2 : 0;
      if (c4) *reinterpret_cast<uint32_t*>(dst) = x[0];
      dst += c4 ? 4 : 0;
    }
#pragma unroll
    for (int j = 0; j < 14; ++j) x[j] = c4 ? x[j + 1] : x[j];
    if (i < 0) {
      if (c8) *reinterpret_cast<uint2*>(dst) = make_uint2(x[0], x[1]);
      dst += c8 ? 8 : 0;
    }
#pragma unroll
    for (int j = 0; j < 12; ++j) x[j] = c8 ? x[j + 2] : x[j];
    if (i < 0) {
      if (c16) *reinterpret_cast<uint4*>(dst) = make_uint4(x[0], x[1], x[2], x[3]);
      dst += c16 ? 16 : 0;
      continue;                                    // (the window stood still: its second half is the row's first eight words)
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = c16 ? x[j + 4] : x[j];
    if (bytes >= 32) {
      const uint32_t w[8] = {x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]};
      st_global_v8(dst, w);
    } else if (bytes > 0) {
      uint8_t* d = dst;
      if (bytes & 16) {
        *reinterpret_cast<uint4*>(d) = make_uint4(x[0], x[1], x[2], x[3]);
        x[0] = x[4], x[1] = x[5], x[2] = x[6], x[3] = x[7];
        d += 16;
      }
      if (bytes & 8) {
        *reinterpret_cast<uint2*>(d) = make_uint2(x[0], x[1]);
        x[0] = x[2], x[1] = x[3];
        d += 8;
      }
      if (bytes & 4) {
        *reinterpret_cast<uint32_t*>(d) = x[0];
        x[0] = x[1];
        d += 4;
      }
      if (bytes & 2) *reinterpret_cast<uint16_t*>(d) = (uint16_t)x[0];
    }
    dst += 32;
    bytes -= 32;
  }
}

// Columns [n, n + 128) of row m, of which those below N exist, from one thread.
__device__ __forceinline__ void store_row128(const MatmulParams& p, int m, int n, const float2* v) {
  const int cols = min(kTile, p.N - n);
  if (m >= p.M || cols <= 0) return;
  const bool f32 = p.out_dtype == B200MOE_F32;
  uint8_t* dst = reinterpret_cast<uint8_t*>(p.out) + ((size_t)m * p.out_stride + n) * (f32 ? 4 : 2);
  if (p.vec_out < 2 || cols < kTile) {
    if (f32) store_row_shifted<true>(dst, p.out_dtype, v, 4 * cols);
    else store_row_shifted<false>(dst, p.out_dtype, v, 2 * cols);
  } else if (f32) {
#pragma unroll
    for (int i = 0; i < 64; i += 4) {
      uint32_t w[8];
      memcpy(w, v + i, 32);
      st_global_v8(dst + 8 * i, w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 64; i += 8) {
      uint32_t w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = pack16(p.out_dtype, v[i + j].x, v[i + j].y);
      st_global_v8(dst + 4 * i, w);
    }
  }
}

__device__ __forceinline__ void fold(float2* acc, const uint32_t (&r)[32], float s) {
  const float2 s2 = make_float2(s, s);
#pragma unroll
  for (int j = 0; j < 16; ++j)
    acc[j] = __ffma2_rn(make_float2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])), s2, acc[j]);
}

// Folds one K block's 128 columns of a TMEM lane into `acc`; `release` runs once the last of them sits in registers: it hands the
// accumulator back and looks at the next K block's barriers without waiting, so that the last FMAs cover the look's latency.  (A
// look already at the first read-back, where it mostly comes too early, took 2 % more time.)
template <typename Release>
__device__ __forceinline__ void promote(float2* acc, uint32_t taddr, float s, Release release) {
  uint32_t ra[32], rb[32];
  tmem_ld_32x32(taddr, ra);
  tmem_ld_32x32(taddr + 32, rb);
  tmem_ld_wait_on(ra, rb);
  fold(acc, ra, s);
  tmem_ld_32x32(taddr + 64, ra);
  fold(acc + 16, rb, s);
  tmem_ld_32x32(taddr + 96, rb);
  tmem_ld_wait_on(ra, rb);
  tc_fence_before();
  __syncwarp();
  release();
  fold(acc + 32, ra, s);
  fold(acc + 48, rb, s);
}

// Factors sa[row, b] * sb[slab, b] of 32 R of a K block's 128 rows and H slabs, made by one warp in a ring in shared memory with
// a full and an empty barrier for each slot, kScaleBatch K blocks at a time so that their loads are in flight together.  The ring is
// apart from the operands': an MMA does not wait for factors, so the stages' barriers may be phases ahead of this warp.  (The
// promotion threads fetching their own scales cost them 350 cycles a K block by asynchronous copies, the loads' whole latency by
// plain loads; arrivals on a barrier of the other CTA, which release at cluster scope, 1700.)
constexpr int kScaleBatch = 4, kScaleRing = 8;

template <int H, int R, typename WaitFree, typename Publish>
__device__ __forceinline__ bool make_factors(const MatmulParams& p, uint32_t ring, uint32_t it, int row0, int slab0, int kb0, int kb1,
                                             int lane, WaitFree wait_free, Publish publish) {
  const float* a[R];
  const float* b[H];
#pragma unroll
  for (int i = 0; i < R; ++i) a[i] = p.a_scale + (size_t)min(row0 + i * 32 + lane, p.M - 1) * p.as_m;
#pragma unroll
  for (int h = 0; h < H; ++h) b[h] = p.b_scale + (size_t)min(slab0 + h, (p.N - 1) / kBlockK) * p.bs_n;
  for (int kb = kb0; kb < kb1; kb += kScaleBatch) {
    float x[kScaleBatch][R], y[kScaleBatch][H];
#pragma unroll
    for (int j = 0; j < kScaleBatch; ++j) {
      const int k = min(kb + j, kb1 - 1);
#pragma unroll
      for (int i = 0; i < R; ++i) x[j][i] = ld_chained(a[i] + k * p.as_kb);
#pragma unroll
      for (int h = 0; h < H; ++h) y[j][h] = ld_chained(b[h] + k * p.bs_kb);
    }
#pragma unroll
    for (int j = 0; j < kScaleBatch; ++j) {
      if (kb + j >= kb1) break;
      const bool ok = wait_free(it);
      if (!__all_sync(0xffffffffu, ok)) return false;
      const uint32_t dst = ring + (it % kScaleRing) * (H * kTile * 4) + lane * 4;
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int i = 0; i < R; ++i)
          asm volatile("st.shared::cta.f32 [%0], %1;" ::"r"(dst + (h * kTile + i * 32) * 4), "f"(x[j][i] * y[j][h]) : "memory");
      __syncwarp();
      if (lane == 0) publish(it);
      ++it;
    }
  }
  return true;
}
__device__ __forceinline__ float ld_factor(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cta.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// "These TMEM columns sit in my registers", added to a counter (and, for a factor slot, to a barrier) at a shared::cluster
// address.  Relaxed: what it publishes was completed by tcgen05.wait::ld, the tcgen05 fences on both sides order the tensor-memory
// accesses; a releasing arrival waits for the thread's loads from global memory first (1000 cycles a K block, when it had some).
__device__ __forceinline__ void count_relaxed(uint32_t cluster_addr) {
  asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], 1;" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void mbar_arrive_relaxed(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}

// Gives up on a wait that is out of budget (see mbar_wait): `looks` in a row found nothing.
struct Patience {
  long long t0 = 0;
  uint32_t looks = 0;
  __device__ __forceinline__ bool out(volatile int* abort_flag, int* status, int where) {
    if (++looks < 1024u) return false;
    looks = 0;
    if (*abort_flag) return true;
    const long long now = clock64();
    if (t0 == 0) {
      t0 = now;
    } else if (now - t0 > kWaitBudgetCycles) {
      *abort_flag = 1;
      if (atomicCAS(status + kStatusCode, 0, (int)B200MOE_ERR_DEVICE_TIMEOUT) == 0) status[kStatusDetail] = where;
      return true;
    }
    return false;
  }
};
// mbar_wait by looking at the phase again and again instead of sleeping on it.
__device__ __forceinline__ bool mbar_poll(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int where) {
  Patience patience;
  while (!mbar_test_wait(bar, parity))
    if (patience.out(abort_flag, status, where)) return false;
  return true;
}
// The same for a counter that only grows (wrap-safe).
__device__ __forceinline__ bool count_poll(uint32_t addr, uint32_t target, volatile int* abort_flag, int* status, int where) {
  Patience patience;
  while (true) {
    uint32_t v;
    asm volatile("ld.relaxed.cluster.shared::cta.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    if ((int32_t)(v - target) >= 0) return true;
    if (patience.out(abort_flag, status, where)) return false;
  }
}

// (The code goes last: who finds it finds the detail too.  A wait for copies or MMAs in flight that gave up counts like any other.)
__device__ __forceinline__ void report_status(const MatmulParams& p, const int* status) {
  if (status[kStatusCode] && p.status) {
    if (status[kStatusDetail]) p.status[1] = status[kStatusDetail];   // (0: it was another CTA of the cluster that gave up)
    __threadfence_system();
    p.status[0] = status[kStatusCode];
    __threadfence_system();
  }
}

// ------------------------------ 128 x 128 tiles ------------------------------

constexpr int kMidThreads = 256;                 // warps 0: TMA, 1-2: MMA issuers, 3: scales, 4-7: promotion and epilogue
// ACC accumulators in tensor memory: two, with three stages, where CTAs share an SM; four, with six, where each has one alone (a K
// block then takes 300 ns instead of 360: more of its way round runs beside the others').
constexpr int mid_stages(int acc) { return acc == 2 ? 3 : 6; }
constexpr int mid_smem_bytes(int acc) { return mid_stages(acc) * kStageBytes + kScaleRing * kTile * 4 + 1024; }
static_assert(mid_stages(2) >= 2 && mid_stages(4) >= 4, "what an issuer knows of a stage's use before (see there)");
static_assert(mid_stages(2) * kStageBytes >= 3 * 11 * kTile * 16,
              "the join of a split product (three parts of eleven vectors are most) reuses the ring");
// setmaxnreg moves registers inside what the CTA was launched with (256 threads x 128): the four control warps give up
// 128 x (128 - 48), the four promotion warps take 128 x (208 - 128).
constexpr int kMidLaunchRegs = 128, kMidCtrlRegs = 48, kMidPromoRegs = 208;
static_assert(128 * (kMidLaunchRegs - kMidCtrlRegs) >= 128 * (kMidPromoRegs - kMidLaunchRegs),
              "setmaxnreg.inc would wait for registers that nobody releases");

// The sum of a split product.  A row's 32 vectors of four columns are divided over the cluster's CTAs: each receives its part of
// every CTA's partial sums in its ring (idle by then), adds them in the order of the ranks and stores them, neighbouring lanes
// neighbouring rows' vectors.
template <int S>
__device__ __forceinline__ void join_split(const MatmulParams& p, const float2* acc, uint32_t smem_base, int thread, int rows, int m0,
                                           int n0) {
  constexpr int kMost = (kTile / 4 + S - 1) / S;   // vectors of a part
  const int me = (int)cluster_rank();
  if (thread < rows) {
#pragma unroll
    for (int c = 0; c < kTile / 4; ++c) {
      const int j = ((c + 1) * S - 1) / (kTile / 4);   // the CTA whose part [32 j / S, 32 (j + 1) / S) has c
      const uint32_t at = smem_base + ((me * kMost + c - kTile / 4 * j / S) * kTile + thread) * 16;
      const float2 x = acc[2 * c], y = acc[2 * c + 1];
      st_cluster_v4(map_to_rank(at, (uint32_t)j), x.x, x.y, y.x, y.y);
    }
  }
  __syncwarp();
  cluster_arrive();
  cluster_wait();
  // a quarter-warp reads eight rows of one vector column (no bank twice); four vector columns of a row are stored together
  const int first = kTile / 4 * me / S, n = kTile / 4 * (me + 1) / S - first;
  const int row8 = thread & 7, c4 = (thread >> 3) & 3, warp = thread >> 5, groups = (rows + 7) / 8;
  for (int i = warp; i < groups * ((n + 3) / 4); i += 4) {
    const int row = i % groups * 8 + row8, c = i / groups * 4 + c4;
    if (row >= rows || c >= n) continue;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    float4 v[S];
#pragma unroll
    for (int j = 0; j < S; ++j) v[j] = ld_shared_v4(smem_base + ((j * kMost + c) * kTile + row) * 16);
#pragma unroll
    for (int j = 0; j < S; ++j) {
      sum.x += v[j].x;
      sum.y += v[j].y;
      sum.z += v[j].z;
      sum.w += v[j].w;
    }
    store4(p, m0 + row, n0 + (first + c) * 4, sum);
  }
}

template <int ACC>
__global__ void __launch_bounds__(kMidThreads, 2)
block_matmul_kernel(const __grid_constant__ MatmulParams p) {
  constexpr int kStages = mid_stages(ACC);
  const int split = p.split;
  const int tile = blockIdx.x / split, part = blockIdx.x % split;
  const int m0 = tile % p.m_tiles * kTile, n0 = tile / p.m_tiles * kTile;
  const int rows = min(kTile, p.M - m0), promo_warps = (rows + 31) / 32;   // (warps without a row only take part in the barriers)
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t s_bars[2 * kStages + ACC + 2 + 2 * kScaleRing];
  __shared__ uint32_t s_read[ACC];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort[3], s_status[2];   // waits of the loops, for copies in flight, for MMAs in flight: each gives up for itself
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t bar_full = smem_u32(s_bars), bar_empty = bar_full + 8 * kStages;
  const uint32_t bar_done = bar_empty + 8 * kStages, bar_drain = bar_done + 8 * ACC, count_read = smem_u32(s_read);
  const uint32_t bar_factors = bar_drain + 16, bar_slot = bar_factors + 8 * kScaleRing;   // a factor slot is filled, is free
  volatile int* abort_flag = s_abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int b = 0; b < ACC; ++b) {
      mbar_init(bar_done + 8 * b, 1);
      s_read[b] = 0;
    }
    for (int r = 0; r < kScaleRing; ++r) {
      mbar_init(bar_factors + 8 * r, 1);
      mbar_init(bar_slot + 8 * r, promo_warps);
    }
    mbar_init(bar_drain, 1);
    mbar_init(bar_drain + 8, 1);
    s_abort[0] = s_abort[1] = s_abort[2] = 0;
    s_status[0] = s_status[1] = 0;
    fence_mbar_init();
    tma_prefetch_desc(&p.tmap_a);
    tma_prefetch_desc(&p.tmap_b);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&s_tmem), ACC * kTile);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;

  const int kb0 = (int)((long long)p.kblocks * part / split), kb1 = (int)((long long)p.kblocks * (part + 1) / split);
  const int steps = kb1 - kb0;
  const uint32_t factors = smem_base + kStages * kStageBytes;
  chain_wait();
  chain_release();

  if (warp < 4) {
    reg_dealloc<kMidCtrlRegs>();
    if (warp == 0 && lane == 0) {
      int it = 0;
      for (; it < steps; ++it) {
        const int s = it % kStages;
        if (!mbar_poll(bar_empty + 8 * s, ((it / kStages) & 1) ^ 1, abort_flag, s_status, 1)) break;
        mbar_arrive_expect_tx(bar_full + 8 * s, kOperandBytes + p.box_rows * kBlockK);
        const uint32_t dst = smem_base + s * kStageBytes;
        tma_load_2d(dst + kOperandBytes, &p.tmap_b, (kb0 + it) * kBlockK, n0, bar_full + 8 * s);
        tma_load_2d(dst, &p.tmap_a, (kb0 + it) * kBlockK, m0, bar_full + 8 * s);
      }
      // copies still in flight must land before the ring is used otherwise or released
      for (int j = it > kStages ? it - kStages : 0; j < it; ++j)
        (void)mbar_poll(bar_full + 8 * (j % kStages), (j / kStages) & 1, abort_flag + 1, s_status, 2);
    } else if (warp == 1 || warp == 2) {
      // Two issuers take turns, each with accumulators of its own: a turn takes some 700 cycles, an MMA chain's 256.  The whole
      // warp runs the loop and one elected lane issues (a lane of its own took 450 cycles for four MMAs and two commits, this
      // 330 and less).  The stage's barrier is looked at only once K block it - ACC has been read back, and with it all before:
      // so the stage's use before, K block it - kStages, has landed.  A parity is not to be asked about two phases ahead.
      constexpr uint32_t idesc = make_idesc_e4m3(kTile, kTile);
      const int me = warp - 1;
      for (int it = me; it < steps; it += 2) {
        const int s = it % kStages, b = it % ACC;
        bool ok = count_poll(count_read + 4 * b, promo_warps * (it / ACC), abort_flag, s_status, 3);
        ok = ok && mbar_poll(bar_full + 8 * s, (it / kStages) & 1, abort_flag, s_status, 4);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
        const uint32_t a_addr = smem_base + s * kStageBytes;
        if (elect_one()) {
          tc_mma_f8_kblock(tmem + b * kTile, kmajor_sw128_desc_lo(a_addr), kmajor_sw128_desc_lo(a_addr + kOperandBytes),
                           kKmajorSw128DescHi, idesc);
          tc_commit(bar_done + 8 * b);
          tc_commit(bar_empty + 8 * s);
        }
        __syncwarp();
      }
      if (elect_one()) tc_commit(bar_drain + 8 * me);   // all MMAs must have read the ring and written tensor memory before either is released
      (void)mbar_poll(bar_drain + 8 * me, 0, abort_flag + 2, s_status, 5);
    } else if (warp == 3) {
      make_factors<1, 4>(
          p, factors, 0, m0, n0 / kBlockK, kb0, kb1, lane,
          [&](uint32_t it) { return mbar_poll(bar_slot + 8 * (it % kScaleRing), ((it / kScaleRing) & 1) ^ 1, abort_flag, s_status, 7); },
          [&](uint32_t it) { mbar_arrive(bar_factors + 8 * (it % kScaleRing)); });
    }
    __syncwarp();
    if (split > 1) {         // the promotion warps' two barriers, see there
      cluster_arrive();
      cluster_wait();
      if (warp == 3 && lane < split && *abort_flag)   // a part of the sum is lost: the cluster's other CTAs learn of it
        st_cluster_s32(map_to_rank(smem_u32(s_status + kStatusCode), (uint32_t)lane), (int)B200MOE_ERR_DEVICE_TIMEOUT);
      __syncwarp();
      cluster_arrive();
      cluster_wait();
    }
  } else {
    reg_alloc<kMidPromoRegs>();
    const uint32_t own = map_to_rank(smem_base, split > 1 ? (uint32_t)part : 0u) - smem_base;   // this CTA's shared::cluster window
    float2 acc[kTile / 2];
    const int row = m0 + (warp - 4) * 32 + lane;
#pragma unroll
    for (int j = 0; j < kTile / 2; ++j) acc[j] = make_float2(0.f, 0.f);
    uint32_t seen_f = 0, seen_d = 0;   // the coming K block's factors, accumulator are known to be there (looked at below)
    for (int it = 0; it < steps && warp - 4 < promo_warps; ++it) {
      const int b = it % ACC;
      if (!(seen_f & seen_d)) {
        const bool ok = (seen_f || mbar_poll(bar_factors + 8 * (it % kScaleRing), (it / kScaleRing) & 1, abort_flag, s_status, 8)) &&
                        (seen_d || mbar_wait(bar_done + 8 * b, (it / ACC) & 1, abort_flag, s_status, 6));
        if (!__all_sync(0xffffffffu, ok)) break;
      }
      tc_fence_after();
      const float f = ld_factor(factors + ((it % kScaleRing) * kTile + threadIdx.x - 128) * 4);
      promote(acc, tmem + ((uint32_t)((warp - 4) * 32) << 16) + b * kTile, f, [&] {
        if (lane == 0) {
          count_relaxed(own + count_read + 4 * b);
          mbar_arrive_relaxed(own + bar_slot + 8 * (it % kScaleRing));
        }
        const uint32_t n = it + 1;
        seen_f = mbar_test_wait(bar_factors + 8 * (n % kScaleRing), (n / kScaleRing) & 1);
        seen_d = mbar_test_wait(bar_done + 8 * (n % ACC), (n / ACC) & 1);
      });
      seen_f = __all_sync(0xffffffffu, seen_f);
      seen_d = __all_sync(0xffffffffu, seen_d);
    }
    const int thread = threadIdx.x - 128;
    if (split == 1) {
      store_row128(p, row, n0, acc);
    } else {
      // every CTA's ring is idle behind this barrier; the promotion warps then exchange the partial sums
      __syncwarp();
      cluster_arrive();
      cluster_wait();
      switch (split) {
        case 2: join_split<2>(p, acc, smem_base, thread, rows, m0, n0); break;
        case 3: join_split<3>(p, acc, smem_base, thread, rows, m0, n0); break;
        case 4: join_split<4>(p, acc, smem_base, thread, rows, m0, n0); break;
        default: join_split<8>(p, acc, smem_base, thread, rows, m0, n0);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, ACC * kTile);
  if (__builtin_expect(s_status[kStatusCode], 0)) {
    store_given_up(p, m0 + (threadIdx.x & 127), n0);   // (over what was stored: a choice before took 2 to 7 % of a small call, this 0 to 2)
    if (threadIdx.x == 0) report_status(p, s_status);
  }
}

// ------------------------------ 256 x 256 tiles of a CTA pair ------------------------------
//
// The pair's leader issues the MMAs (M = 256, N = 128: two for each 32 bytes of K); each CTA brings its 128 rows of A and half
// of the 256 rows of B, and holds the accumulators of its 128 rows.  Columns [0, 128) of the tile (one weight scale
// block) belong to the first promotion warpgroup, the others to the second, each with two accumulators of its own: while a
// warpgroup folds one K block, the tensor cores make its next one and the other half's.  Two issuing warps take turns with the K
// blocks: a turn takes some 700 cycles, most of them latency of shared memory, which operand reads and copies keep busy.

constexpr int kPairThreads = 384;                // warps 0: TMA, 1-2: MMA issuers (leader), 3: scales, 4-11: promotion
constexpr int kPairStages = 5;
static_assert(kPairStages >= 5, "what an issuer knows of a stage's use before (see there)");
constexpr int kPairStageBytes = kStageBytes;     // a CTA's part: 128 rows of A, 2 x 64 rows of B
constexpr int kPairSmemBytes = kPairStages * kPairStageBytes + kScaleRing * 2 * kTile * 4 + 1024;
constexpr int kPairLaunchRegs = 168, kPairCtrlRegs = 72, kPairPromoRegs = 216;
static_assert(128 * (kPairLaunchRegs - kPairCtrlRegs) >= 256 * (kPairPromoRegs - kPairLaunchRegs),
              "setmaxnreg.inc would wait for registers that nobody releases");
// A CTA that asks for tensor memory waits until there is enough, and CTAs of a cluster wait for one another: so no two of these
// CTAs may be on an SM whose accumulators do not fit together.  Shared memory sees to it.
constexpr int kSmSmemBytes = 228 * 1024;
static_assert(3 * mid_smem_bytes(2) > kSmSmemBytes, "three CTAs with 256 columns each");
static_assert(mid_smem_bytes(4) + mid_smem_bytes(2) > kSmSmemBytes && kPairSmemBytes + mid_smem_bytes(2) > kSmSmemBytes,
              "a CTA with all 512 columns beside another");
constexpr int kPairSuper = 8;                    // M tiles that run beside each other on the same N tiles

__device__ __forceinline__ void pair_tmem_alloc(uint32_t smem_result_addr, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_result_addr), "r"(ncols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void pair_tmem_dealloc(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// A copy into this CTA's shared memory, counted on the barrier at a shared::cluster address (the leader's).
__device__ __forceinline__ void pair_tma_load_2d(uint32_t smem_dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];"
      ::"r"(smem_dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
// Arrives on the barrier at this offset in both CTAs once the MMAs that this thread issued have completed.
__device__ __forceinline__ void pair_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(bar), "h"((uint16_t)3) : "memory");
}
// The four MMAs of a K block, the first from zero (see tc_mma_f8_kblock).
__device__ __forceinline__ void pair_mma_kblock(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t desc_hi, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred pf, pt;\n\t.reg .b64 da, db;\n\t.reg .b32 al, bl;\n\t"
      "setp.ne.b32 pf, 0, 0;\n\t"
      "setp.eq.b32 pt, 0, 0;\n\t"
      "mov.b64 da, {%1, %3};\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], da, db, %4, pf;\n\t"
      "add.u32 al, %1, 2;\n\t"
      "add.u32 bl, %2, 2;\n\t"
      "mov.b64 da, {al, %3};\n\t"
      "mov.b64 db, {bl, %3};\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], da, db, %4, pt;\n\t"
      "add.u32 al, %1, 4;\n\t"
      "add.u32 bl, %2, 4;\n\t"
      "mov.b64 da, {al, %3};\n\t"
      "mov.b64 db, {bl, %3};\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], da, db, %4, pt;\n\t"
      "add.u32 al, %1, 6;\n\t"
      "add.u32 bl, %2, 6;\n\t"
      "mov.b64 da, {al, %3};\n\t"
      "mov.b64 db, {bl, %3};\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], da, db, %4, pt;\n\t}"
      ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(desc_hi), "r"(idesc)
      : "memory");
}

// Tile number -> first row and column: kPairSuper M tiles at a time walk all N tiles, so that what runs together shares operands.
__device__ __forceinline__ void pair_tile(const MatmulParams& p, int tile, int* m, int* n) {
  const int per = kPairSuper * p.n_tiles, group = tile / per, in = tile - group * per;
  const int rows = min(kPairSuper, p.m_tiles - group * kPairSuper);
  *n = in / rows * (2 * kTile);
  *m = (group * kPairSuper + in % rows) * (2 * kTile);
}

__global__ void __launch_bounds__(kPairThreads, 1)
block_matmul_pair_kernel(const __grid_constant__ MatmulParams p) {
  constexpr int S = kPairStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t s_bars[2 * S + 4 + 2 + 2 * kScaleRing];
  __shared__ uint32_t s_read[4];                           // leader's: [half][2] warps of both CTAs that have read an accumulator
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort[3], s_status[2];   // waits of the loops, for copies in flight, for MMAs in flight: each gives up for itself
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t bar_full = smem_u32(s_bars);              // leader's: a stage of both CTAs has landed
  const uint32_t bar_empty = bar_full + 8 * S;             // both: the MMAs have read a stage
  const uint32_t bar_done = bar_empty + 8 * S;             // both: [half][2] an accumulator is written
  const uint32_t count_read = smem_u32(s_read);
  const uint32_t bar_drain = bar_done + 32;                // both: [issuer] its MMAs have retired
  const uint32_t bar_factors = bar_drain + 16;             // own: a factor slot is filled
  const uint32_t bar_slot = bar_factors + 8 * kScaleRing;  // own: it is free
  volatile int* abort_flag = s_abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int b = 0; b < 4; ++b) {
      mbar_init(bar_done + 8 * b, 1);
      s_read[b] = 0;
    }
    mbar_init(bar_drain, 1);
    mbar_init(bar_drain + 8, 1);
    for (int r = 0; r < kScaleRing; ++r) {
      mbar_init(bar_factors + 8 * r, 1);
      mbar_init(bar_slot + 8 * r, 8);
    }
    s_abort[0] = s_abort[1] = s_abort[2] = 0;
    s_status[0] = s_status[1] = 0;
    fence_mbar_init();
    tma_prefetch_desc(&p.tmap_a);
    tma_prefetch_desc(&p.tmap_b);
  }
  if (warp == 1) pair_tmem_alloc(smem_u32(&s_tmem), 512);
  tc_fence_before();
  __syncthreads();
  cluster_arrive();
  cluster_wait();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const uint32_t factors = smem_base + S * kPairStageBytes;   // [kScaleRing][2][128]
  const int tiles = p.m_tiles * p.n_tiles, first = blockIdx.x >> 1, stride = gridDim.x >> 1, kblocks = p.kblocks;
  chain_wait();
  chain_release();

  if (warp < 4) {
    reg_dealloc<kPairCtrlRegs>();
    if (warp == 0 && lane == 0) {
      const uint32_t full = map_to_rank(bar_full, 0);
      uint32_t it = 0;
      bool alive = true;
      for (int tile = first; tile < tiles && alive; tile += stride) {
        int m0, n0;
        pair_tile(p, tile, &m0, &n0);
        m0 += rank * kTile;
        n0 += rank * 64;               // of each 128-column half, this CTA's 64
        for (int kb = 0; kb < kblocks; ++kb, ++it) {
          const uint32_t s = it % S;
          if (!mbar_poll(bar_empty + 8 * s, ((it / S) & 1) ^ 1, abort_flag, s_status, 11)) { alive = false; break; }
          if (rank == 0) mbar_arrive_expect_tx(bar_full + 8 * s, 2 * kPairStageBytes);
          const uint32_t dst = smem_base + s * kPairStageBytes;
          pair_tma_load_2d(dst, &p.tmap_a, kb * kBlockK, m0, full + 8 * s);
          pair_tma_load_2d(dst + kOperandBytes, &p.tmap_b, kb * kBlockK, n0, full + 8 * s);
          pair_tma_load_2d(dst + kOperandBytes + kOperandBytes / 2, &p.tmap_b, kb * kBlockK, n0 + kTile, full + 8 * s);
        }
      }
      // Copies still in flight must land before either CTA leaves (the leader's barriers count both CTAs'), and the leader's
      // arrivals on this CTA's barriers too.
      for (uint32_t j = it > S ? it - S : 0; j < it; ++j) {
        if (rank == 0) (void)mbar_poll(bar_full + 8 * (j % S), (j / S) & 1, abort_flag + 1, s_status, 12);
        (void)mbar_poll(bar_empty + 8 * (j % S), (j / S) & 1, abort_flag + 1, s_status, 12);
      }
      // The issuers are the leader's: only here, behind the last K block, is the wait for their MMAs one of a hand-off's length.
      if (rank != 0)
        for (int i = 0; i < 2; ++i) (void)mbar_poll(bar_drain + 8 * i, 0, abort_flag + 2, s_status, 15);
    } else if (warp == 1 || warp == 2) {
      // (The loop's form: see the other kernel.  What makes the two looks at a stage's barrier safe: this warp's last turn waited
      // until K block it - 4 had been read back, so it - 5, the stage's use before, has landed; and behind the first count_poll
      // the same holds for it - 2 and the use before that of K block it + 2, it - 3.)
      constexpr uint32_t idesc = make_idesc_e4m3(2 * kTile, kTile);
      const uint32_t me = warp - 1;                // the K blocks, and accumulator of each half, of this warp
      const uint32_t steps = rank == 0 && first < tiles ? (uint32_t)((tiles - 1 - first) / stride + 1) * (uint32_t)kblocks : 0u;
      uint32_t seen = 0;
      for (uint32_t it = me; it < steps; it += 2) {
        const uint32_t s = it % S, n = it + 2;
        bool ok = seen || mbar_poll(bar_full + 8 * s, (it / S) & 1, abort_flag, s_status, 13);
        const uint32_t a_addr = smem_base + s * kPairStageBytes;
#pragma unroll
        for (uint32_t half = 0; half < 2; ++half) {
          ok = ok && count_poll(count_read + 4 * (2 * half + me), 8 * (it >> 1), abort_flag, s_status, 14);
          if (!__all_sync(0xffffffffu, ok)) break;
          tc_fence_after();
          if (half == 0) seen = mbar_test_wait(bar_full + 8 * (n % S), (n / S) & 1);
          if (elect_one()) {
            pair_mma_kblock(tmem + (2 * half + me) * kTile, kmajor_sw128_desc_lo(a_addr),
                            kmajor_sw128_desc_lo(a_addr + kOperandBytes + half * (kOperandBytes / 2)), kKmajorSw128DescHi, idesc);
            pair_commit(bar_done + 8 * (2 * half + me));
            if (half == 1) pair_commit(bar_empty + 8 * s);
          }
          __syncwarp();
        }
        if (!__all_sync(0xffffffffu, ok)) break;
        seen = __all_sync(0xffffffffu, seen);
      }
      if (rank == 0) {
        if (elect_one()) pair_commit(bar_drain + 8 * me);
        (void)mbar_poll(bar_drain + 8 * me, 0, abort_flag + 2, s_status, 15);
      }
    } else if (warp == 3) {
      uint32_t it = 0;
      for (int tile = first; tile < tiles; tile += stride, it += kblocks) {
        int m0, n0;
        pair_tile(p, tile, &m0, &n0);
        const bool ok = make_factors<2, 4>(
            p, factors, it, m0 + rank * kTile, n0 / kBlockK, 0, kblocks, lane,
            [&](uint32_t i) { return mbar_poll(bar_slot + 8 * (i % kScaleRing), ((i / kScaleRing) & 1) ^ 1, abort_flag, s_status, 17); },
            [&](uint32_t i) { mbar_arrive(bar_factors + 8 * (i % kScaleRing)); });
        if (!ok) break;
      }
    }
    __syncwarp();
  } else {
    reg_alloc<kPairPromoRegs>();
    const int pw = warp - 4, half = pw >> 2, q = pw & 3;
    const uint32_t read = map_to_rank(count_read + 8 * half, 0), slot = map_to_rank(bar_slot, rank);
    const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16) + half * 2 * kTile;
    uint32_t it = 0, seen_f = 0, seen_d = 0;   // seen: the coming K block's factors, accumulator are known to be there (looked at below)
    bool alive = true;
    int tile = first;
    for (; tile < tiles; tile += stride) {
      int m0, n0;
      pair_tile(p, tile, &m0, &n0);
      m0 += rank * kTile + q * 32;
      n0 += half * kTile;
      float2 acc[kTile / 2];
#pragma unroll
      for (int j = 0; j < kTile / 2; ++j) acc[j] = make_float2(0.f, 0.f);
      for (int kb = 0; kb < kblocks; ++kb, ++it) {
        const uint32_t b = it & 1;
        if (!(seen_f & seen_d)) {
          const bool ok = (seen_f || mbar_poll(bar_factors + 8 * (it % kScaleRing), (it / kScaleRing) & 1, abort_flag, s_status, 18)) &&
                          (seen_d || mbar_wait(bar_done + 8 * (2 * half + b), (it >> 1) & 1, abort_flag, s_status, 16));
          if (!__all_sync(0xffffffffu, ok)) { alive = false; break; }
        }
        tc_fence_after();
        const float f = ld_factor(factors + ((it % kScaleRing) * 2 * kTile + threadIdx.x - 128) * 4);
        promote(acc, taddr + b * kTile, f, [&] {
          if (lane == 0) {
            count_relaxed(read + 4 * b);
            mbar_arrive_relaxed(slot + 8 * (it % kScaleRing));
          }
          const uint32_t n = it + 1;
          seen_f = mbar_test_wait(bar_factors + 8 * (n % kScaleRing), (n / kScaleRing) & 1);
          seen_d = mbar_test_wait(bar_done + 8 * (2 * half + (n & 1)), (n >> 1) & 1);
        });
        seen_f = __all_sync(0xffffffffu, seen_f);
        seen_d = __all_sync(0xffffffffu, seen_d);
      }
      if (!alive) break;
      store_row128(p, m0 + lane, n0, acc);
    }
    for (; tile < tiles; tile += stride) {   // (given up: this tile and those to come)
      int m0, n0;
      pair_tile(p, tile, &m0, &n0);
      m0 += rank * kTile + q * 32 + lane;
      n0 += half * kTile;
      store_given_up(p, m0, n0);
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_arrive();            // neither CTA leaves, or frees tensor memory, while the other may still use it
  cluster_wait();
  tc_fence_after();
  if (warp == 1) pair_tmem_dealloc(tmem, 512);
  if (threadIdx.x == 0) report_status(p, s_status);
}

// Whether every CTA of 128 x 128 tiles with S parts of K has an SM alone.  A cluster's CTAs have to be neighbours, for which not
// all places can be had.
bool mid_alone(long long ctas, int S, int num_sms) { return ctas <= (S == 1 ? num_sms : num_sms * 7 / 8); }

// What a call takes, in ns and less what all take, by a fit to measured times (us, bf16 results, weights of 7 to 117 MB).
// 128 x 128 tiles with S parts of K.  A K block takes 300 ns where CTAs have an SM alone (360 in the last wave of several), 590 where two
// share it; the join's time goes with the rows that travel.  S 1, 2, 3, 4, 8; *: shared SMs.  N 4096, K 7168: 1 row 19.3, 12.3, 10.2,
// 9.4, 9.3*; 128 rows 20.9, 16.0, 14.1, 12.9, 17.0*; 300 rows 21.7, 23.3*, 28.9*, 29.3*, 40.5*.  N 7168, K 2048: 1 row 7.9, 6.9, 7.2*, 7.0*, 11.1*;
// 128 rows 8.6, 10.1, 12.9*, 12.8*, 23.9*.  N 7168, K 16384: 128 rows 45.9, 30.5, 33.2*, 29.8*, 42.4*; 300 rows 69.6*, 74.2*, 59.9*, 68.9*, 91.0*.
// Of several waves each costs CTAs' coming and going too, and from the third on L2's rate: see below.  `rough`: rows of A or B do not
// start on sectors (32 bytes), so that a tile's row is five of them.  512 x 6016 x 1504 11.4, x 1488 14.4; 1536 x 1536 x 7136 22.1,
// x 7152 26.3; 8000 x 1536 x 2080 39, x 2064 51 (pairs 32.3, 33.4).
long long mid_cost(long long tiles, int kblocks, int rows, int S, bool rough, int num_sms) {
  const long long ctas = tiles * S, steps = (kblocks + S - 1) / S, shared = rough ? 860 : 590;
  const long long join = S == 1 ? 300 : 400 + rows * (2300 + 250 * S) / kTile, join2 = S == 1 ? 300 : 600 + rows * (800 + 1000 * S) / kTile;
  if (mid_alone(ctas, S, num_sms)) return steps * (285 + (rough ? 135 : 60) * rows / kTile) + join;
  const long long wave = S == 3 ? num_sms * 7 / 4 : 2 * num_sms, full = ctas / wave, rest = ctas - full * wave;
  const long long last = rest == 0 ? 0 : mid_alone(rest, S, num_sms) ? steps * 360 + join : steps * shared + join2;
  return full * (steps * (full >= 2 ? shared + 30 : shared) + join2 + (full >= 2 ? 2700 : 2200)) + last + (full ? 1000 : 0);
}
// 256 x 256 tiles, one pair of SMs each.  128 x 128 tiles / pairs: M x 1536 x 7168: M 1536 21.9 / 31.0, 2048 32.9 / 30.8, 4096 54.6 / 59.5; M x
// 4096 x 7168: 640 32.7 / 30.9, 1024 33.3 / 30.7, 1536 54.8 / 59.7, 2048 65.8 / 59.7, 3000 104.7 / 88.5, 8192 274 / 225; M x 7168 x 16384: 1024
// 146 / 130, 2048 300 / 261, 4096 575 / 530; 2124 x 2190 x 6352 68 / 50, 3709 x 4480 x 1264 42 / 30, 2138 x 4608 x 704 19 / 17.
long long pair_cost(long long tiles, int kblocks, int num_sms) {
  const long long pairs = num_sms / 2;
  return (tiles + pairs - 1) / pairs * (kblocks * 530ll + 1500);
}

// How a product is made: 256 x 256 tiles of CTA pairs, or 128 x 128 tiles with `split` parts of K, each CTA alone on its SM or not.
struct MatmulForm {
  bool pair;
  int split;
  bool alone;
};
MatmulForm matmul_form(int M, long long m_tiles, long long n_tiles, int kblocks, bool rough, int num_sms) {
  const int rows = M < kTile ? M : kTile;
  MatmulForm f = {false, 1, false};
  long long cost = mid_cost(m_tiles * n_tiles, kblocks, rows, 1, rough, num_sms);
  for (int S : {2, 3, 4, 8}) {
    if (2 * S > kblocks) break;
    const long long c = mid_cost(m_tiles * n_tiles, kblocks, rows, S, rough, num_sms);
    if (c < cost) {
      cost = c;
      f.split = S;
    }
  }
  if (pair_cost(((m_tiles + 1) / 2) * ((n_tiles + 1) / 2), kblocks, num_sms) < cost) return {true, 1, true};
  f.alone = mid_alone(m_tiles * n_tiles * f.split, f.split, num_sms);
  return f;
}
// Rows that do not start on sectors (32 bytes).
bool rough_rows(int64_t a_row_stride, int64_t b_row_stride) { return (a_row_stride | b_row_stride) % 32 != 0; }
bool too_many_tiles(int M, int N, long long m_tiles, long long n_tiles) {
  return m_tiles * n_tiles * kMaxSplit > 0x7fffffffll || M > 0x7fffff00 || N > 0x7fffff00;
}

}  // namespace

cudaError_t configure_block_matmul() {
  cudaError_t e = cudaFuncSetAttribute(block_matmul_kernel<2>, cudaFuncAttributeMaxDynamicSharedMemorySize, mid_smem_bytes(2));
  if (e != cudaSuccess) return e;
  e = cudaFuncSetAttribute(block_matmul_kernel<4>, cudaFuncAttributeMaxDynamicSharedMemorySize, mid_smem_bytes(4));
  if (e != cudaSuccess) return e;
  return cudaFuncSetAttribute(block_matmul_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmemBytes);
}

}  // namespace b200moe

using namespace b200moe;

extern "C" int b200moe_block_matmul_form(int M, int N, int K, int64_t a_row_stride, int64_t b_row_stride, int num_sms) {
  if (M < 1 || N < 1 || K < 1 || num_sms < 1 || a_row_stride < K || b_row_stride < K) return B200MOE_ERR_INVALID_ARGUMENT;
  const long long m_tiles = ((long long)M + kTile - 1) / kTile, n_tiles = ((long long)N + kTile - 1) / kTile;
  if (K % 16 != 0 || too_many_tiles(M, N, m_tiles, n_tiles)) return B200MOE_ERR_UNSUPPORTED_SHAPE;
  const MatmulForm f = matmul_form(M, m_tiles, n_tiles, (K + kBlockK - 1) / kBlockK, rough_rows(a_row_stride, b_row_stride), num_sms);
  return f.pair ? 0 : f.alone ? f.split : 16 + f.split;
}

extern "C" int b200moe_block_matmul(const uint8_t* a, int64_t a_row_stride, const float* a_scale, int64_t a_scale_stride_m,
                                    int64_t a_scale_stride_kb, const uint8_t* b, int64_t b_row_stride, const float* b_scale,
                                    int64_t b_scale_stride_n, int64_t b_scale_stride_kb, int M, int N, int K, void* out,
                                    int out_dtype, int64_t out_row_stride, int32_t* status, void* stream) {
  if (M < 0 || N < 0 || K < 1 || (out_dtype != B200MOE_F32 && out_dtype != B200MOE_BF16 && out_dtype != B200MOE_F16))
    return B200MOE_ERR_INVALID_ARGUMENT;
  if (K % 16 != 0) return B200MOE_ERR_UNSUPPORTED_SHAPE;   // rows of e4m3 start on 16-byte boundaries
  if (M == 0 || N == 0) return B200MOE_OK;
  if (!a || !a_scale || !b || !b_scale || !out || a_row_stride < K || b_row_stride < K || out_row_stride < N)
    return B200MOE_ERR_INVALID_ARGUMENT;
  const uintptr_t size = out_dtype == B200MOE_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(a) | (uintptr_t)a_row_stride | reinterpret_cast<uintptr_t>(b) | (uintptr_t)b_row_stride) % 16 != 0 ||
      reinterpret_cast<uintptr_t>(out) % size != 0 || !words_aligned(a_scale, b_scale, status))
    return B200MOE_ERR_MISALIGNED;
  const long long m_tiles = ((long long)M + kTile - 1) / kTile, n_tiles = ((long long)N + kTile - 1) / kTile;
  if (too_many_tiles(M, N, m_tiles, n_tiles)) return B200MOE_ERR_UNSUPPORTED_SHAPE;
  int num_sms = 0;
  int rc = ensure_device(&num_sms);
  if (rc != B200MOE_OK) return rc;
  MatmulParams p;
  p.a_scale = a_scale;
  p.b_scale = b_scale;
  p.as_m = a_scale_stride_m;
  p.as_kb = a_scale_stride_kb;
  p.bs_n = b_scale_stride_n;
  p.bs_kb = b_scale_stride_kb;
  p.M = M;
  p.N = N;
  p.kblocks = (K + kBlockK - 1) / kBlockK;
  p.out = out;
  p.out_dtype = out_dtype;
  p.out_stride = out_row_stride;
  const uintptr_t out_bits = reinterpret_cast<uintptr_t>(out) | (uintptr_t)(out_row_stride * (long long)size);
  p.vec_out = out_bits % 32 == 0 ? 2 : out_bits % 16 == 0 ? 1 : 0;
  p.status = status;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);

  const MatmulForm form = matmul_form(M, m_tiles, n_tiles, p.kblocks, rough_rows(a_row_stride, b_row_stride), num_sms);
  p.split = form.split;
  if (form.pair) {
    if ((rc = make_tmap(&p.tmap_a, a, (uint64_t)M, (uint64_t)K, (uint64_t)a_row_stride, kTile)) != B200MOE_OK) return rc;
    if ((rc = make_tmap(&p.tmap_b, b, (uint64_t)N, (uint64_t)K, (uint64_t)b_row_stride, kTile / 2)) != B200MOE_OK) return rc;
    p.m_tiles = (int)((m_tiles + 1) / 2);
    p.n_tiles = (int)((n_tiles + 1) / 2);
    const long long pairs = num_sms / 2, pair_tiles = (long long)p.m_tiles * p.n_tiles;
    CUDA_TRY(launch_chained_cluster(block_matmul_pair_kernel, dim3((unsigned)(2 * (pair_tiles < pairs ? pair_tiles : pairs))), dim3(kPairThreads),
                                    kPairSmemBytes, st, 2, p));
    return B200MOE_OK;
  }
  if ((rc = make_tmap(&p.tmap_b, b, (uint64_t)N, (uint64_t)K, (uint64_t)b_row_stride, kTile)) != B200MOE_OK) return rc;
  // fewer rows than a tile has are a smaller copy
  p.box_rows = M < kTile ? M : kTile;
  if ((rc = make_tmap(&p.tmap_a, a, (uint64_t)M, (uint64_t)K, (uint64_t)a_row_stride, (uint32_t)p.box_rows)) != B200MOE_OK) return rc;
  p.m_tiles = (int)m_tiles;
  p.n_tiles = (int)n_tiles;
  CUDA_TRY(launch_chained_cluster(form.alone ? block_matmul_kernel<4> : block_matmul_kernel<2>,
                                  dim3((unsigned)(m_tiles * n_tiles * p.split)), dim3(kMidThreads), mid_smem_bytes(form.alone ? 4 : 2), st,
                                  p.split, p));
  return B200MOE_OK;
}
