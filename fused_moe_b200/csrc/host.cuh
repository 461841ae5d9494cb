// Host-side helpers that the entry points share (defined in capi.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace b200moe {

// Whether tables of 4-byte numbers start where such numbers may (null ones do).
template <typename... P>
inline bool words_aligned(const P*... p) {
  return ((reinterpret_cast<uintptr_t>(p) | ...) & 3) == 0;
}

// Records the error's text for b200moe_last_cuda_error and returns B200MOE_ERR_CUDA.
int cuda_fail(cudaError_t e, const char* what);

// Once per process: the driver entry point for tensor-map encoding; once per device: the
// SM count and the opt-in shared memory sizes of the kernels that need them.
int ensure_device(int* num_sms);

// Tensor map over bytes, boxes with 128-byte swizzle.
int encode_tmap(CUtensorMap* map, const void* base, uint32_t rank, const cuuint64_t* dims, const cuuint64_t* strides,
                const cuuint32_t* box);
// rows x K e4m3 matrix, row pitch `pitch` bytes; box = box_rows x 128 bytes, 128-byte swizzle.
int make_tmap(CUtensorMap* map, const void* base, uint64_t rows, uint64_t k, uint64_t pitch, uint32_t box_rows);

}  // namespace b200moe

#define CUDA_TRY(expr)                                           \
  do {                                                           \
    cudaError_t _e = (expr);                                     \
    if (_e != cudaSuccess) return b200moe::cuda_fail(_e, #expr); \
  } while (0)
