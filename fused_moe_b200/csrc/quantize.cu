// Activations to e4m3 codes with one fp32 scale per 1x128 block, optionally behind a SwiGLU.
//
//   s[t,b] = max(max_{k in block b} |x[t,k]|, 1e-12) / 448          (fp32)
//   q[t,k] = e4m3( fp32( x[t,k] / s[t,b] ) )                        (nearest, ties to even)
//   with SwiGLU: x[t,k] = in[t,k] * silu(in[t,K+k]) in fp32, never rounded to the input's type
//
// Bound by HBM: every input byte is read once, one byte per element and four per block are written.  Sixteen lanes
// take a block, eight elements each (16 bytes of a 16-bit type), so that a lane's part stays in registers between the maximum
// and the division.  A CTA takes one block column of 64 rows: every half-warp has four rows in flight, and the scales of
// the [K/128, T] layout leave as 64 neighbours.
#include "common.cuh"
#include "host.cuh"
#include "kernels.cuh"

namespace b200moe {

namespace {

constexpr int kQuantRows = 4;                      // rows of a half-warp, all in flight
constexpr int kQuantThreads = 256;
constexpr int kQuantTile = kQuantRows * kQuantThreads / 16;
constexpr float kAmaxMin = 1e-12f;

// A NaN stays one: it makes its block's scale, and so all codes of the block, NaN (an infinity makes the scale infinite),
// as the formula says.
__device__ __forceinline__ float max_abs_nan(float m, float x) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(x)));
  return r;
}

template <typename T> struct Elem;
template <> struct Elem<float> {
  static constexpr bool kShort = false;
  static __device__ float get(float v) { return v; }
};
template <> struct Elem<__half> {
  static constexpr bool kShort = true;
  static __device__ float get(__half v) { return __half2float(v); }
};
template <> struct Elem<__nv_bfloat16> {
  static constexpr bool kShort = true;
  static __device__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
};

// Eight neighbouring elements; VEC: 16-byte loads.
template <typename T, bool VEC>
struct Raw8 {
  T v[8];
  __device__ __forceinline__ void load(const T* p, int left) {
    if (VEC) {
      constexpr int kVecs = (int)sizeof(T) / 2;
      uint4 u[kVecs];
#pragma unroll
      for (int i = 0; i < kVecs; ++i) u[i] = left > 0 ? __ldg(reinterpret_cast<const uint4*>(p) + i) : make_uint4(0u, 0u, 0u, 0u);
      memcpy(v, u, sizeof(v));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < left ? p[i] : T(0.f);
    }
  }
};

// Correctly rounded x / d for any fp32 x, two at a time: a first correction brings the quotient within one ulp, from where
// Markstein's remainder step (see div2_rn) rounds it correctly.
__device__ __forceinline__ float2 div2_rn_any(float2 x, float d, float inv) {
  const float2 dd = make_float2(d, d), mi = make_float2(-inv, -inv), mx = make_float2(-x.x, -x.y);
  float2 q = __fmul2_rn(x, make_float2(inv, inv));
  q = __ffma2_rn(__ffma2_rn(q, dd, mx), mi, q);
  return __ffma2_rn(__ffma2_rn(q, dd, mx), mi, q);
}

template <typename T, bool SWIGLU, bool VEC>
__global__ void __launch_bounds__(kQuantThreads)
quantize_kernel(const T* __restrict__ x, long long x_stride, int rows, int cols, int kblocks, uint8_t* __restrict__ codes,
                long long codes_stride, float* __restrict__ scale, long long s_stride_t, long long s_stride_kb) {
  __shared__ float s_scale[kQuantTile];
  chain_wait();
  chain_release();
  const int kb = blockIdx.x % kblocks;
  const int row0 = (int)(blockIdx.x / kblocks) * kQuantTile;
  const int part = threadIdx.x & 15, hw = threadIdx.x >> 4;
  const int col = kb * kBlockK + part * 8;
  const int left = cols - col;                     // columns from this lane's first on
  Raw8<T, VEC> a[kQuantRows], b[SWIGLU ? kQuantRows : 1];
#pragma unroll
  for (int r = 0; r < kQuantRows; ++r) {
    const int row = row0 + r * (kQuantThreads / 16) + hw;
    const T* p = x + (size_t)row * x_stride + col;
    a[r].load(p, row < rows ? left : 0);
    if (SWIGLU) b[r].load(p + cols, row < rows ? left : 0);
  }
#pragma unroll
  for (int r = 0; r < kQuantRows; ++r) {
    const int rt = r * (kQuantThreads / 16) + hw, row = row0 + rt;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = Elem<T>::get(a[r].v[i]);
      if (SWIGLU) {
        const float u = Elem<T>::get(b[r].v[i]);
        v[i] *= u * (1.0f / (1.0f + expf(-u)));
      }
    }
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max_abs_nan(m, v[i]);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max_abs_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float s = (m < kAmaxMin ? kAmaxMin : m) / 448.0f;
    if (part == 0) s_scale[rt] = s;
    float2 q[4];
    if (s < INFINITY) {
      const float inv = __frcp_rn(s);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 e = make_float2(v[2 * i], v[2 * i + 1]);
        q[i] = Elem<T>::kShort && !SWIGLU ? div2_rn(e, s, inv) : div2_rn_any(e, s, inv);
      }
    } else {   // an infinity or a NaN in the block: the remainder step has no meaning there
#pragma unroll
      for (int i = 0; i < 4; ++i) q[i] = make_float2(v[2 * i] / s, v[2 * i + 1] / s);
    }
    if (row < rows) {
      const uint2 c = make_uint2(pack4_e4m3(q[0].x, q[0].y, q[1].x, q[1].y), pack4_e4m3(q[2].x, q[2].y, q[3].x, q[3].y));
      uint8_t* dst = codes + (size_t)row * codes_stride + col;
      if (VEC) {
        if (left > 0) *reinterpret_cast<uint2*>(dst) = c;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < left) dst[i] = (uint8_t)((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
      }
    }
  }
  __syncthreads();
  const int row = row0 + (int)threadIdx.x;
  if (threadIdx.x < kQuantTile && row < rows)
    scale[(size_t)row * s_stride_t + (size_t)kb * s_stride_kb] = s_scale[threadIdx.x];
}

template <typename T, bool SWIGLU>
cudaError_t launch_one(const void* x, long long x_stride, int rows, int cols, uint8_t* codes, long long codes_stride,
                       float* scale, long long s_stride_t, long long s_stride_kb, cudaStream_t stream) {
  const int kblocks = (cols + kBlockK - 1) / kBlockK;
  const long long grid = (long long)kblocks * ((rows + kQuantTile - 1) / kQuantTile);
  // 16-byte loads and 8-byte stores where every row and every lane's part starts on such a boundary
  const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && x_stride * (long long)sizeof(T) % 16 == 0 && cols % 8 == 0 &&
                   reinterpret_cast<uintptr_t>(codes) % 8 == 0 && codes_stride % 8 == 0;
  auto* kern = vec ? quantize_kernel<T, SWIGLU, true> : quantize_kernel<T, SWIGLU, false>;
  return launch_chained(kern, dim3((unsigned)grid), dim3(kQuantThreads), 0, stream, reinterpret_cast<const T*>(x), x_stride,
                        rows, cols, kblocks, codes, codes_stride, scale, s_stride_t, s_stride_kb);
}

template <typename T>
cudaError_t launch_type(bool swiglu, const void* x, long long x_stride, int rows, int cols, uint8_t* codes,
                        long long codes_stride, float* scale, long long s_stride_t, long long s_stride_kb,
                        cudaStream_t stream) {
  return swiglu ? launch_one<T, true>(x, x_stride, rows, cols, codes, codes_stride, scale, s_stride_t, s_stride_kb, stream)
                : launch_one<T, false>(x, x_stride, rows, cols, codes, codes_stride, scale, s_stride_t, s_stride_kb, stream);
}

}  // namespace

}  // namespace b200moe

using namespace b200moe;

extern "C" int b200moe_quantize(const void* x, int dtype, int64_t row_stride, int rows, int cols, int swiglu, uint8_t* codes,
                                int64_t codes_row_stride, float* scale, int64_t scale_stride_t, int64_t scale_stride_kb,
                                void* stream) {
  if (rows < 0 || cols < 0 || (dtype != B200MOE_F32 && dtype != B200MOE_BF16 && dtype != B200MOE_F16))
    return B200MOE_ERR_INVALID_ARGUMENT;
  if (rows == 0 || cols == 0) return B200MOE_OK;
  if (!x || !codes || !scale || codes_row_stride < cols || row_stride < (swiglu ? 2ll : 1ll) * cols)
    return B200MOE_ERR_INVALID_ARGUMENT;
  if ((long long)((cols + kBlockK - 1) / kBlockK) * ((rows + kQuantTile - 1) / kQuantTile) > 0x7fffffffll ||
      cols > 0x3fffffff || rows > 0x7fffffff - kQuantTile)
    return B200MOE_ERR_UNSUPPORTED_SHAPE;
  const uintptr_t elem = dtype == B200MOE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(x) % elem != 0 || reinterpret_cast<uintptr_t>(scale) % 4 != 0)
    return B200MOE_ERR_MISALIGNED;
  int num_sms = 0;
  const int rc = ensure_device(&num_sms);
  if (rc != B200MOE_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool sw = swiglu != 0;
  cudaError_t e;
  if (dtype == B200MOE_F32)
    e = launch_type<float>(sw, x, row_stride, rows, cols, codes, codes_row_stride, scale, scale_stride_t, scale_stride_kb, st);
  else if (dtype == B200MOE_BF16)
    e = launch_type<__nv_bfloat16>(sw, x, row_stride, rows, cols, codes, codes_row_stride, scale, scale_stride_t,
                                   scale_stride_kb, st);
  else
    e = launch_type<__half>(sw, x, row_stride, rows, cols, codes, codes_row_stride, scale, scale_stride_t, scale_stride_kb, st);
  CUDA_TRY(e);
  return B200MOE_OK;
}
