// Activations to e4m3 codes with one fp32 scale per 1x128 block, optionally behind a SwiGLU.
//
//   s[t,b] = max(max_{k in block b} |x[t,k]|, 1e-12) / 448          (fp32)
//   q[t,k] = e4m3( fp32( x[t,k] / s[t,b] ) )                        (nearest, ties to even)
//   with SwiGLU: x[t,k] = in[t,k] * silu(in[t,K+k]) in fp32, never rounded to the input's type
//
// Bound by HBM: every input byte is read once, one byte per element and four per block are written.  Sixteen lanes
// take a block, eight elements each (16 bytes of a 16-bit type), so that a lane's part stays in registers between the maximum
// and the division.  A CTA takes eight blocks of eight rows (fewer blocks of more rows, see quantize_log_width): every half-warp has
// four of them in flight, reads come in pieces of 2 KB, and scales leave by the sector in either layout.
#include "common.cuh"
#include "host.cuh"
#include "kernels.cuh"

namespace b200moe {

namespace {

constexpr int kQuantThreads = 256;
constexpr int kQuantHalves = kQuantThreads / 16;   // half-warps of a CTA
// Blocks of a half-warp, all in flight: four, two behind a SwiGLU, whose exponentials take as long as memory does (with twice
// as many CTAs one computes while another loads: 14.4 us instead of 14.7 for 4099 x 2048).
__host__ __device__ constexpr int quant_units(bool swiglu) { return swiglu ? 2 : 4; }
constexpr float kAmaxMin = 1e-12f;

// A NaN stays one: it makes its block's scale, and so all codes of the block, NaN (an infinity makes the scale infinite),
// as the formula says.
__device__ __forceinline__ float max_abs_nan(float m, float x) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(x)));
  return r;
}

// 1 / x, correctly rounded, for x from 1/4 on: Newton's step from an approximation within one ulp (Markstein, as at div2_rn, who
// excludes only a fraction of all ones).  0 from 2^126 on, infinity included.  13.0 -> 10.6 us for 4099 x 2048 against the
// division, with the same bits in every test.
__device__ __forceinline__ float rcp_from_quarter(float x) {
  x = fminf(x, 3.4028234e38f);   // (a NaN is the factor u's business)
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return fmaf(fmaf(-x, y, 1.0f), y, y);
}

// max_abs2: the same for two 16-bit numbers at once (the sign of the result is free)
template <typename T> struct Elem;
template <> struct Elem<float> {
  static constexpr bool kShort = false;
  static __device__ float get(float v) { return v; }
  static __device__ uint32_t max_abs2(uint32_t, uint32_t) { return 0u; }
  static __device__ float lower(uint32_t) { return 0.f; }
};
template <> struct Elem<__half> {
  static constexpr bool kShort = true;
  static __device__ float get(__half v) { return __half2float(v); }
  static __device__ uint32_t max_abs2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ float lower(uint32_t v) { return __half2float(__ushort_as_half((unsigned short)v)); }
  static __device__ float upper(uint32_t v) { return __half2float(__ushort_as_half((unsigned short)(v >> 16))); }
};
template <> struct Elem<__nv_bfloat16> {
  static constexpr bool kShort = true;
  static __device__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ uint32_t max_abs2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ float lower(uint32_t v) { return __uint_as_float(v << 16); }
  static __device__ float upper(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }
};

// A lane's eight elements of a block: neighbours, by 16-byte loads (VEC), or every sixteenth, so that a half-warp's lanes take
// neighbours at a time (8192 x 4097 bf16 33 us; by single neighbouring elements 43).
template <typename T, bool VEC>
struct Raw8 {
  T v[8];
  __device__ __forceinline__ void load(const T* p, int left) {
    if (VEC) {
      constexpr int kVecs = (int)sizeof(T) / 2;
      uint4 u[kVecs];
#pragma unroll
      for (int i = 0; i < kVecs; ++i) u[i] = left > 0 ? ld_chained(reinterpret_cast<const uint4*>(p) + i) : make_uint4(0u, 0u, 0u, 0u);
      memcpy(v, u, sizeof(v));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 16 * i < left ? p[16 * i] : T(0.f);
    }
  }
  // (16-bit elements out of whole words)
  __device__ __forceinline__ float get(int i) const {
    if constexpr (Elem<T>::kShort) {
      uint32_t w;
      memcpy(&w, v + (i & ~1), 4);
      return i & 1 ? Elem<T>::upper(w) : Elem<T>::lower(w);
    } else {
      return Elem<T>::get(v[i]);
    }
  }
};

// div2_rn with the remainders one at a time: two scalar instructions take the minus sign with them, a packed one does not.
__device__ __forceinline__ float2 div2_rn_short(float2 x, float d, float inv) {
  const float2 q = __fmul2_rn(x, make_float2(inv, inv));
  return __ffma2_rn(make_float2(fmaf(q.x, d, -x.x), fmaf(q.y, d, -x.y)), make_float2(-inv, -inv), q);
}
// Correctly rounded x / d for any fp32 x, two at a time: a first correction brings the quotient within one ulp, from where
// Markstein's remainder step (see div2_rn) rounds it correctly.
__device__ __forceinline__ float2 div2_rn_any(float2 x, float d, float inv) {
  const float2 mi = make_float2(-inv, -inv);
  float2 q = __fmul2_rn(x, make_float2(inv, inv));
  q = __ffma2_rn(make_float2(fmaf(q.x, d, -x.x), fmaf(q.y, d, -x.y)), mi, q);
  return __ffma2_rn(make_float2(fmaf(q.x, d, -x.x), fmaf(q.y, d, -x.y)), mi, q);
}

template <typename T, bool SWIGLU, bool VEC>
__global__ void __launch_bounds__(kQuantThreads)
quantize_kernel(const T* x, long long x_stride, int rows, int cols, int kblocks, uint8_t* __restrict__ codes,
                long long codes_stride, float* __restrict__ scale, long long s_stride_t, long long s_stride_kb, int log_width) {
  constexpr int kQuantUnits = quant_units(SWIGLU), kTileBlocks = kQuantUnits * kQuantHalves;
  const int width = 1 << log_width, step = kQuantHalves >> log_width, tile_rows = kTileBlocks >> log_width;   // (step: rows of a pass)
  __shared__ float s_scale[kTileBlocks];
  chain_wait();
  chain_release();
  const int groups = (kblocks + width - 1) >> log_width;
  const int kb0 = (int)(blockIdx.x % groups) << log_width, row0 = (int)(blockIdx.x / groups) * tile_rows;
  const int part = threadIdx.x & 15, hw = threadIdx.x >> 4;
  const int my_kb = hw & (width - 1), my_row = hw >> log_width;
  const int col = (kb0 + my_kb) * kBlockK + (VEC ? part * 8 : part);
  const int left = cols - col;                     // columns from this lane's first on
  Raw8<T, VEC> a[kQuantUnits], b[SWIGLU ? kQuantUnits : 1];
#pragma unroll
  for (int r = 0; r < kQuantUnits; ++r) {
    const int row = row0 + r * step + my_row;
    const T* p = x + (size_t)row * x_stride + col;
    a[r].load(p, row < rows ? left : 0);
    if (SWIGLU) b[r].load(p + cols, row < rows ? left : 0);
  }
  // Largest absolute values of the half-warp's blocks.  16-bit numbers are compared two at a time, and two blocks'
  // maxima go through the lanes together.
  constexpr bool kPacked = Elem<T>::kShort && !SWIGLU;
  float v[kPacked ? 1 : kQuantUnits][8], m[kQuantUnits];
  if (kPacked) {
    uint32_t h[kQuantUnits];
#pragma unroll
    for (int r = 0; r < kQuantUnits; ++r) {
      uint32_t w[4];
      memcpy(w, a[r].v, 16);
      h[r] = Elem<T>::max_abs2(Elem<T>::max_abs2(w[0], w[1]), Elem<T>::max_abs2(w[2], w[3]));
      h[r] = Elem<T>::max_abs2(h[r], h[r] >> 16);   // (its lower half)
    }
#pragma unroll
    for (int r = 0; r < kQuantUnits; r += 2) {
      uint32_t two = __byte_perm(h[r], h[r + 1], 0x5410);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) two = Elem<T>::max_abs2(two, __shfl_xor_sync(0xffffffffu, two, o));
      two &= 0x7fff7fffu;
      m[r] = Elem<T>::lower(two);
      m[r + 1] = Elem<T>::lower(two >> 16);
    }
  } else {
#pragma unroll
    for (int r = 0; r < kQuantUnits; ++r) {
      m[r] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float x = a[r].get(i);
        if (SWIGLU) {
          const float u = b[r].get(i);
          // (a quarter of the divisor: its reciprocal is a normal number for all that expf gives below infinity)
          x *= 0.25f * u * rcp_from_quarter(fmaf(expf(-u), 0.25f, 0.25f));
        }
        v[r][i] = x;
        m[r] = max_abs_nan(m[r], x);
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) m[r] = max_abs_nan(m[r], __shfl_xor_sync(0xffffffffu, m[r], o));
    }
  }
  // a lane makes the scale of one of the blocks, and hands it to the others
  const float mine = kQuantUnits == 4 && (part & 2) ? (part & 1 ? m[kQuantUnits - 1] : m[kQuantUnits - 2]) : (part & 1 ? m[1] : m[0]);
  const float my_s = (mine < kAmaxMin ? kAmaxMin : mine) / 448.0f, my_inv = __frcp_rn(my_s);
  if (part < kQuantUnits)
    s_scale[my_kb * tile_rows + part * step + my_row] = my_s;
#pragma unroll
  for (int r = 0; r < kQuantUnits; ++r) {
    const int row = row0 + r * step + my_row;
    const float s = __shfl_sync(0xffffffffu, my_s, r, 16), inv = __shfl_sync(0xffffffffu, my_inv, r, 16);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = kPacked ? a[r].get(i) : v[kPacked ? 0 : r][i];
    float2 q[4];
    if (s < INFINITY) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 e = make_float2(x[2 * i], x[2 * i + 1]);
        q[i] = kPacked ? div2_rn_short(e, s, inv) : div2_rn_any(e, s, inv);
      }
    } else {   // an infinity or a NaN in the block: the remainder step has no meaning there
#pragma unroll
      for (int i = 0; i < 4; ++i) q[i] = make_float2(x[2 * i] / s, x[2 * i + 1] / s);
    }
    if (row < rows) {
      const uint2 c = make_uint2(pack4_e4m3(q[0].x, q[0].y, q[1].x, q[1].y), pack4_e4m3(q[2].x, q[2].y, q[3].x, q[3].y));
      uint8_t* dst = codes + (size_t)row * codes_stride + col;
      if (VEC) {
        if (left > 0) *reinterpret_cast<uint2*>(dst) = c;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (16 * i < left) dst[16 * i] = (uint8_t)((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
      }
    }
  }
  __syncthreads();
  // neighbouring threads neighbouring rows of the [K/128, T] layout, neighbouring blocks of the other
  if (threadIdx.x < kTileBlocks) {
    const int i = threadIdx.x;
    const int rt = s_stride_t == 1 ? i & (tile_rows - 1) : i >> log_width, kb = s_stride_t == 1 ? i / tile_rows : i & (width - 1);
    if (row0 + rt < rows && kb0 + kb < kblocks)
      scale[(size_t)(row0 + rt) * s_stride_t + (size_t)(kb0 + kb) * s_stride_kb] = s_scale[kb * tile_rows + rt];
  }
}

// Blocks that a CTA's tile has of a row: the largest power of two up to eight that leaves no tile with blocks behind the row's end.
// us, bf16, with 1, 2, 4, 8: 8192 x 7168 32.5, 32.2, 31.9, 31.7; 8192 x 4480 21.1, 21.5, 21.3, 23.0; 32768 x 1152 21.8, 23.3, 26.4, 33.0;
// 65536 x 512 19.1, 18.9, 18.7, 32.2; 262144 x 128 18.7, 32.2, 59.1, 115.
int quantize_log_width(int kblocks) { return kblocks % 8 == 0 ? 3 : kblocks % 4 == 0 ? 2 : kblocks % 2 == 0 ? 1 : 0; }

long long quantize_grid(int rows, int kblocks, bool swiglu) {
  const int log_width = quantize_log_width(kblocks), tile_rows = quant_units(swiglu) * kQuantHalves >> log_width;
  return (long long)((kblocks + (1 << log_width) - 1) >> log_width) * (((long long)rows + tile_rows - 1) / tile_rows);
}

template <typename T, bool SWIGLU>
cudaError_t launch_one(const void* x, long long x_stride, int rows, int cols, uint8_t* codes, long long codes_stride,
                       float* scale, long long s_stride_t, long long s_stride_kb, cudaStream_t stream) {
  const int kblocks = (cols + kBlockK - 1) / kBlockK;
  const long long grid = quantize_grid(rows, kblocks, SWIGLU);
  // 16-byte loads and 8-byte stores where every row and every lane's part starts on such a boundary
  const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && x_stride * (long long)sizeof(T) % 16 == 0 && cols % 8 == 0 &&
                   reinterpret_cast<uintptr_t>(codes) % 8 == 0 && codes_stride % 8 == 0;
  auto* kern = vec ? quantize_kernel<T, SWIGLU, true> : quantize_kernel<T, SWIGLU, false>;
  return launch_chained(kern, dim3((unsigned)grid), dim3(kQuantThreads), 0, stream, reinterpret_cast<const T*>(x), x_stride,
                        rows, cols, kblocks, codes, codes_stride, scale, s_stride_t, s_stride_kb, quantize_log_width(kblocks));
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
  if (cols > 0x3fffffff || rows > 0x7fffff00 ||
      quantize_grid(rows, (cols + kBlockK - 1) / kBlockK, swiglu != 0) > 0x7fffffffll)
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
