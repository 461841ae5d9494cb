// Dense product of e4m3 matrices with block scales on tcgen05 tensor cores.
//
//   out[m,n] = sum_b sa[m,b] sb[n/128,b] * ( sum_{k in block b} a[m,k] b[n,k] ),   blocks of 128 along K
//
// The scales are arbitrary fp32 numbers, so they cannot ride on the MMA: a K block's raw dot products are made in tensor
// memory from zero, read back and folded into fp32 registers with one FMA each, the factor being one number per row (= TMEM
// lane = thread) and 128-column slab.
#include "common.cuh"
#include "host.cuh"
#include "kernels.cuh"

namespace b200moe {

namespace {

constexpr int kThreads = 256;                    // warps 0: TMA, 1: MMA, 4-7: promotion and epilogue
constexpr int kTile = 128;
constexpr int kOperandBytes = kTile * kBlockK;   // 16 KiB
constexpr int kStageBytes = 2 * kOperandBytes;
constexpr int kStages = 3;
constexpr int kAcc = 2;                          // accumulators in tensor memory
constexpr int kSmemBytes = kStages * kStageBytes + 1024;
constexpr int kMaxSplit = 8;
// setmaxnreg moves registers inside what the CTA was launched with (256 threads x 128): the four control warps give up
// 128 x (128 - 48), the four promotion warps take 128 x (208 - 128).
constexpr int kLaunchRegs = 128, kCtrlRegs = 48, kPromoRegs = 208;
static_assert(128 * (kLaunchRegs - kCtrlRegs) >= 128 * (kPromoRegs - kLaunchRegs),
              "setmaxnreg.inc would wait for registers that nobody releases");
static_assert(kStages * kStageBytes >= kTile * kTile * 4, "the join of a split product reuses the ring");

struct MatmulParams {
  CUtensorMap tmap_a, tmap_b;
  const float* a_scale;
  const float* b_scale;
  long long as_m, as_kb, bs_n, bs_kb;
  int M, N, kblocks;
  int n_tiles;
  int split;                                     // CTAs of a cluster, each with a part of the K blocks
  void* out;
  int out_dtype;
  long long out_stride;
  int vec_out;                                   // rows of `out` start on 16-byte boundaries
  int* status;                                   // device-accessible int32[2], or null
};

__device__ __forceinline__ void st_cluster_v4(uint32_t addr, float a, float b, float c, float d) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}
__device__ __forceinline__ float4 ld_shared_v4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cta.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

// Columns [n, n + 2 * PAIRS) of one row; `cols` of them exist.
template <int PAIRS>
__device__ __forceinline__ void store_row(const MatmulParams& p, int m, int n, const float2* v) {
  const int cols = p.N - n;
  if (p.out_dtype == B200MOE_F32) {
    float* dst = reinterpret_cast<float*>(p.out) + (size_t)m * p.out_stride + n;
    if (p.vec_out && cols >= 2 * PAIRS) {
#pragma unroll
      for (int i = 0; i < PAIRS; i += 2)
        *reinterpret_cast<float4*>(dst + 2 * i) = make_float4(v[i].x, v[i].y, v[i + 1].x, v[i + 1].y);
    } else {
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        if (2 * i < cols) dst[2 * i] = v[i].x;
        if (2 * i + 1 < cols) dst[2 * i + 1] = v[i].y;
      }
    }
    return;
  }
  uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + (size_t)m * p.out_stride + n;
  uint32_t w[PAIRS];
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) {
    if (p.out_dtype == B200MOE_BF16) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[i].x, v[i].y);
      memcpy(&w[i], &h, 4);
    } else {
      const __half2 h = __floats2half2_rn(v[i].x, v[i].y);
      memcpy(&w[i], &h, 4);
    }
  }
  if (p.vec_out && cols >= 2 * PAIRS) {
#pragma unroll
    for (int i = 0; i < PAIRS; i += 4) *reinterpret_cast<uint4*>(dst + 2 * i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      if (2 * i < cols) dst[2 * i] = (uint16_t)w[i];
      if (2 * i + 1 < cols) dst[2 * i + 1] = (uint16_t)(w[i] >> 16);
    }
  }
}

__device__ __forceinline__ void fold(float2* acc, const uint32_t (&r)[32], float s) {
  const float2 s2 = make_float2(s, s);
#pragma unroll
  for (int j = 0; j < 16; ++j)
    acc[j] = __ffma2_rn(make_float2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])), s2, acc[j]);
}

// The sum of a split product: CTA j of a cluster of S receives columns [128 j / S, 128 (j+1) / S) of every CTA's partial sums
// in its ring (idle by then), adds them in the order of the ranks and stores them.
template <int S>
__device__ __forceinline__ void join_split(const MatmulParams& p, const float2* acc, uint32_t smem_base, int thread, int m0, int n0) {
  constexpr int kCols = kTile / S, kVecs = kCols / 4;
  const uint32_t me = cluster_rank();
#pragma unroll
  for (int j = 0; j < S; ++j) {
    const uint32_t dst = map_to_rank(smem_base, (uint32_t)j) + (me * kVecs * kTile + thread) * 16;
#pragma unroll
    for (int c = 0; c < kVecs; ++c) {
      const float2 x = acc[(j * kCols) / 2 + 2 * c], y = acc[(j * kCols) / 2 + 2 * c + 1];
      st_cluster_v4(dst + c * kTile * 16, x.x, x.y, y.x, y.y);
    }
  }
  cluster_arrive();
  cluster_wait();
  float2 sum[kCols / 2];
#pragma unroll
  for (int i = 0; i < kCols / 2; ++i) sum[i] = make_float2(0.f, 0.f);
#pragma unroll
  for (int j = 0; j < S; ++j)
#pragma unroll
    for (int c = 0; c < kVecs; ++c) {
      const float4 v = ld_shared_v4(smem_base + ((j * kVecs + c) * kTile + thread) * 16);
      sum[2 * c].x += v.x;
      sum[2 * c].y += v.y;
      sum[2 * c + 1].x += v.z;
      sum[2 * c + 1].y += v.w;
    }
  if (m0 + thread < p.M && n0 + (int)me * kCols < p.N) store_row<kCols / 2>(p, m0 + thread, n0 + me * kCols, sum);
}

__global__ void __launch_bounds__(kThreads, 2)
block_matmul_kernel(const __grid_constant__ MatmulParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t s_bars[2 * kStages + 2 * kAcc + 1];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort[2], s_status[2];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t bar_full = smem_u32(s_bars), bar_empty = bar_full + 8 * kStages;
  const uint32_t bar_done = bar_empty + 8 * kStages, bar_read = bar_done + 8 * kAcc, bar_drain = bar_read + 8 * kAcc;
  volatile int* abort_flag = s_abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int b = 0; b < kAcc; ++b) {
      mbar_init(bar_done + 8 * b, 1);
      mbar_init(bar_read + 8 * b, 4);
    }
    mbar_init(bar_drain, 1);
    s_abort[0] = s_abort[1] = 0;
    s_status[0] = s_status[1] = 0;
    fence_mbar_init();
    tma_prefetch_desc(&p.tmap_a);
    tma_prefetch_desc(&p.tmap_b);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&s_tmem), kAcc * kTile);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;

  const int split = p.split;
  const int tile = blockIdx.x / split, part = blockIdx.x % split;
  const int m0 = tile / p.n_tiles * kTile, n0 = tile % p.n_tiles * kTile;
  const int kb0 = (int)((long long)p.kblocks * part / split), kb1 = (int)((long long)p.kblocks * (part + 1) / split);
  const int steps = kb1 - kb0;
  chain_wait();
  chain_release();

  if (warp < 4) {
    reg_dealloc<kCtrlRegs>();
    if (warp == 0 && lane == 0) {
      int it = 0;
      for (; it < steps; ++it) {
        const int s = it % kStages;
        if (!mbar_wait(bar_empty + 8 * s, ((it / kStages) & 1) ^ 1, abort_flag, s_status, 1)) break;
        mbar_arrive_expect_tx(bar_full + 8 * s, kStageBytes);
        const uint32_t dst = smem_base + s * kStageBytes;
        tma_load_2d(dst, &p.tmap_a, (kb0 + it) * kBlockK, m0, bar_full + 8 * s);
        tma_load_2d(dst + kOperandBytes, &p.tmap_b, (kb0 + it) * kBlockK, n0, bar_full + 8 * s);
      }
      // copies still in flight must land before the ring is used otherwise or released
      for (int j = it > kStages ? it - kStages : 0; j < it; ++j)
        (void)mbar_wait(bar_full + 8 * (j % kStages), (j / kStages) & 1, abort_flag + 1, s_status, 2);
    } else if (warp == 1 && lane == 0) {
      constexpr uint32_t idesc = make_idesc_e4m3(kTile, kTile);
      for (int it = 0; it < steps; ++it) {
        const int s = it % kStages, b = it % kAcc;
        if (!mbar_wait(bar_read + 8 * b, ((it / kAcc) & 1) ^ 1, abort_flag, s_status, 3)) break;
        if (!mbar_wait(bar_full + 8 * s, (it / kStages) & 1, abort_flag, s_status, 4)) break;
        tc_fence_after();
        const uint32_t a_addr = smem_base + s * kStageBytes;
        tc_mma_f8_kblock(tmem + b * kTile, kmajor_sw128_desc_lo(a_addr), kmajor_sw128_desc_lo(a_addr + kOperandBytes),
                         kKmajorSw128DescHi, idesc);
        tc_commit(bar_empty + 8 * s);
        tc_commit(bar_done + 8 * b);
      }
      tc_commit(bar_drain);   // all MMAs must have read the ring and written tensor memory before either is released
      (void)mbar_wait(bar_drain, 0, abort_flag + 1, s_status, 5);
    }
    if (split > 1) {         // the promotion warps' two barriers, see there
      __syncwarp();
      cluster_arrive();
      cluster_wait();
      cluster_arrive();
      cluster_wait();
    }
  } else {
    reg_alloc<kPromoRegs>();
    float2 acc[kTile / 2];
    const int row = m0 + (warp - 4) * 32 + lane;
    const float* sa = p.a_scale + (size_t)min(row, p.M - 1) * p.as_m + (size_t)kb0 * p.as_kb;
    const float* sb = p.b_scale + (size_t)(n0 / kBlockK) * p.bs_n + (size_t)kb0 * p.bs_kb;
#pragma unroll
    for (int j = 0; j < kTile / 2; ++j) acc[j] = make_float2(0.f, 0.f);
    float next = steps > 0 ? __ldg(sa) * __ldg(sb) : 0.f;
    for (int it = 0; it < steps; ++it) {
      const int b = it % kAcc;
      const float s = next;
      if (it + 1 < steps) next = __ldg(sa + (it + 1) * p.as_kb) * __ldg(sb + (it + 1) * p.bs_kb);
      const bool ok = mbar_wait(bar_done + 8 * b, (it / kAcc) & 1, abort_flag, s_status, 6);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      const uint32_t t = tmem + ((uint32_t)((warp - 4) * 32) << 16) + b * kTile;
      uint32_t ra[32], rb[32];
      tmem_ld_32x32(t, ra);
      tmem_ld_32x32(t + 32, rb);
      tmem_ld_wait_on(ra, rb);
      fold(acc, ra, s);
      tmem_ld_32x32(t + 64, ra);
      fold(acc + 16, rb, s);
      tmem_ld_32x32(t + 96, rb);
      tmem_ld_wait_on(ra, rb);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_read + 8 * b);
      fold(acc + 32, ra, s);
      fold(acc + 48, rb, s);
    }
    if (split == 1) {
      if (row < p.M) store_row<kTile / 2>(p, row, n0, acc);
    } else {
      // every CTA's ring is idle behind this barrier; the promotion warps then exchange the partial sums
      __syncwarp();
      cluster_arrive();
      cluster_wait();
      const int thread = threadIdx.x - 128;
      if (split == 2) join_split<2>(p, acc, smem_base, thread, m0, n0);
      else if (split == 4) join_split<4>(p, acc, smem_base, thread, m0, n0);
      else join_split<8>(p, acc, smem_base, thread, m0, n0);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, kAcc * kTile);
  if (threadIdx.x == 0 && s_abort[0] && p.status) {
    p.status[1] = s_status[kStatusDetail];
    p.status[0] = s_status[kStatusCode];
    __threadfence_system();
  }
}

}  // namespace

cudaError_t configure_block_matmul() {
  return cudaFuncSetAttribute(block_matmul_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
}

}  // namespace b200moe

using namespace b200moe;

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
      reinterpret_cast<uintptr_t>(out) % size != 0)
    return B200MOE_ERR_MISALIGNED;
  const long long m_tiles = ((long long)M + kTile - 1) / kTile, n_tiles = ((long long)N + kTile - 1) / kTile;
  if (m_tiles * n_tiles * kMaxSplit > 0x7fffffffll || M > 0x7fffff00 || N > 0x7fffff00) return B200MOE_ERR_UNSUPPORTED_SHAPE;
  int num_sms = 0;
  int rc = ensure_device(&num_sms);
  if (rc != B200MOE_OK) return rc;
  MatmulParams p;
  if ((rc = make_tmap(&p.tmap_a, a, (uint64_t)M, (uint64_t)K, (uint64_t)a_row_stride, kTile)) != B200MOE_OK) return rc;
  if ((rc = make_tmap(&p.tmap_b, b, (uint64_t)N, (uint64_t)K, (uint64_t)b_row_stride, kTile)) != B200MOE_OK) return rc;
  p.a_scale = a_scale;
  p.b_scale = b_scale;
  p.as_m = a_scale_stride_m;
  p.as_kb = a_scale_stride_kb;
  p.bs_n = b_scale_stride_n;
  p.bs_kb = b_scale_stride_kb;
  p.M = M;
  p.N = N;
  p.kblocks = (K + kBlockK - 1) / kBlockK;
  p.n_tiles = (int)n_tiles;
  p.out = out;
  p.out_dtype = out_dtype;
  p.out_stride = out_row_stride;
  p.vec_out = reinterpret_cast<uintptr_t>(out) % 16 == 0 && out_row_stride * (long long)size % 16 == 0;
  p.status = status;
  p.split = 1;
  while (p.split < kMaxSplit && m_tiles * n_tiles * p.split * 2 <= 2 * num_sms && p.kblocks >= 4 * p.split) p.split *= 2;

  CUDA_TRY(launch_chained_cluster(block_matmul_kernel, dim3((unsigned)(m_tiles * n_tiles * p.split)), dim3(kThreads), kSmemBytes,
                                  reinterpret_cast<cudaStream_t>(stream), p.split, p));
  return B200MOE_OK;
}
