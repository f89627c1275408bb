// Residual addition + RMS norm of a decoder layer, with a bf16 or an e4m3 + scales output:
//   z = x + residual;  y = z * rsqrt(mean(z^2) + eps) * weight
//   e4m3: per group (a whole row, or group_size columns) s = max(max|y|, 1e-12) / 448,
//         y8 = e4m3(y / s)
// z, the sum of squares and the scales are fp32; z is rounded to bf16 once for residual_out and
// is normalised unrounded, y is rounded once to its output type.
#include <string>

#include <cuda_fp8.h>

#include "lm_common.cuh"

namespace lm {
namespace {

constexpr int kNormThreads = 256;
constexpr int kMaxHidden = 16384;
constexpr float kE4m3Max = 448.f;
constexpr float kScaleFloor = 1e-12f;

struct NormParams {
  const uint16_t* x;
  const uint16_t* residual;
  const uint16_t* weight;
  uint16_t* residual_out;
  uint16_t* y;
  uint8_t* y8;
  float* scales;
  int64_t x_stride, residual_stride, residual_out_stride, y_stride, y8_stride;
  float eps;
  int hidden, group;
};

__device__ __forceinline__ float block_reduce(float v, bool is_max, float* s_red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float u = __shfl_xor_sync(0xffffffffu, v, o);
    v = is_max ? fmaxf(v, u) : v + u;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s_red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s_red[0];
  for (int i = 1; i < kNormThreads / 32; ++i) v = is_max ? fmaxf(v, s_red[i]) : v + s_red[i];
  return v;
}

// One block per row, z held in shared memory.
__global__ void __launch_bounds__(kNormThreads) add_rms_norm_kernel(const NormParams p) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ float s_z[];
  __shared__ float s_red[kNormThreads / 32];
  const int64_t t = blockIdx.x;
  const int H = p.hidden;
  float ss = 0.f;
  for (int c = threadIdx.x; c < H; c += kNormThreads) {
    float z = bf16_bits_to_f32(p.x[t * p.x_stride + c]);
    if (p.residual != nullptr) z += bf16_bits_to_f32(p.residual[t * p.residual_stride + c]);
    if (p.residual_out != nullptr) p.residual_out[t * p.residual_out_stride + c] = f32_to_bf16_bits(z);
    s_z[c] = z;
    ss += z * z;
  }
  const float r = rsqrtf(block_reduce(ss, false, s_red) / H + p.eps);
  for (int c = threadIdx.x; c < H; c += kNormThreads) {
    const float y = s_z[c] * r * bf16_bits_to_f32(p.weight[c]);
    if (p.y != nullptr) p.y[t * p.y_stride + c] = f32_to_bf16_bits(y);
    s_z[c] = y;
  }
  if (p.y8 == nullptr) return;
  __syncthreads();
  const int group = p.group > 0 ? p.group : H;
  for (int g = 0; g < H / group; ++g) {
    float m = 0.f;
    for (int c = threadIdx.x; c < group; c += kNormThreads) m = fmaxf(m, fabsf(s_z[g * group + c]));
    m = block_reduce(m, true, s_red);
    const float s = fmaxf(m, kScaleFloor) / kE4m3Max;
    for (int c = threadIdx.x; c < group; c += kNormThreads)
      p.y8[t * p.y8_stride + g * group + c] =
          __nv_cvt_float_to_fp8(s_z[g * group + c] / s, __NV_SATFINITE, __NV_E4M3);
    if (threadIdx.x == 0) p.scales[t * (H / group) + g] = s;
  }
}

}  // namespace
}  // namespace lm

using namespace lm;

extern "C" int lm_add_rms_norm(const uint16_t* x, int64_t x_stride, const uint16_t* residual,
                               int64_t residual_stride, const uint16_t* weight, float eps,
                               int64_t num_tokens, int32_t hidden_size, uint16_t* residual_out,
                               int64_t residual_out_stride, uint16_t* y, int64_t y_stride,
                               uint8_t* y8, int64_t y8_stride, float* scales, int32_t group_size,
                               void* stream) {
  if (hidden_size <= 0 || hidden_size > kMaxHidden || num_tokens < 0 || num_tokens > 0x7fffffff)
    return fail(LM_ERR_INVALID_ARGUMENT,
                "lm_add_rms_norm: need 1 <= hidden_size <= 16384 and 0 <= num_tokens < 2^31");
  if ((y == nullptr) == (y8 == nullptr) && num_tokens > 0)
    return fail(LM_ERR_INVALID_ARGUMENT, "lm_add_rms_norm: give one of y and y8");
  if (y8 != nullptr && (scales == nullptr || group_size < 0 ||
                        (group_size != 0 && (group_size % 32 != 0 || hidden_size % group_size != 0))))
    return fail(LM_ERR_INVALID_ARGUMENT,
                "lm_add_rms_norm: y8 needs scales and a group_size of 0 (a row) or a multiple of "
                "32 that divides hidden_size");
  if (num_tokens == 0) return LM_OK;
  if (x == nullptr || weight == nullptr)
    return fail(LM_ERR_INVALID_ARGUMENT, "lm_add_rms_norm: null pointer");
  if (x_stride < hidden_size || (residual != nullptr && residual_stride < hidden_size) ||
      (residual_out != nullptr && residual_out_stride < hidden_size) ||
      (y != nullptr && y_stride < hidden_size) || (y8 != nullptr && y8_stride < hidden_size))
    return fail(LM_ERR_INVALID_ARGUMENT, "lm_add_rms_norm: a row stride is below hidden_size");
  const NormParams p{x, residual, weight, residual_out, y, y8, scales, x_stride, residual_stride,
                     residual_out_stride, y_stride, y8_stride, eps, hidden_size, group_size};
  const size_t smem = static_cast<size_t>(hidden_size) * 4;
  if (smem > 48 * 1024) {
    const int rc = check_cuda(cudaFuncSetAttribute(add_rms_norm_kernel,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   kMaxHidden * 4),
                              "lm_add_rms_norm: smem attribute");
    if (rc) return rc;
  }
  return check_cuda(launch_dependent(add_rms_norm_kernel, dim3(static_cast<unsigned>(num_tokens)),
                                     dim3(kNormThreads), smem, static_cast<cudaStream_t>(stream), p),
                    "lm_add_rms_norm");
}
