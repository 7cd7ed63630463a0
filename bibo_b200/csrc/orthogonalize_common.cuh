// What the two files of the Newton-Schulz orthogonalisation share (see orthogonalize.cu).
#pragma once
#include <cuda_fp16.h>

#include "tc_common.cuh"

namespace bibo {
namespace tc {

constexpr float NS_ONE = 4096.f;                 // 1.0 as stored
constexpr float NS_LO = 2048.f;                  // scale of the lower half of a value beside the upper one

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ float2 unpack_f16(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }

// orthogonalize_small.cu: CTAs per matrix of the one-launch kernel (0: it does not take these sizes), and the launch
int ns_small_cluster(int64_t batch, int rows, int cols);
int ns_small_launch(const void* u, int dtype, int64_t batch, int64_t batch_stride, int rows, int cols, int64_t row_stride, int steps,
                    bool joint, const float* coefficients, float eps, int cluster, void* out, cudaStream_t st);

}  // namespace tc
}  // namespace bibo
