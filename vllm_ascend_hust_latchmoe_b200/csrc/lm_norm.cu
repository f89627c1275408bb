// Residual addition + RMS norm of a decoder layer, with a bf16 or an e4m3 + scales output:
//   z = x + residual;  y = z * rsqrt(mean(z^2) + eps) * weight
//   e4m3: per group (a whole row, or group_size columns) s = max(max|y|, 1e-12) / 448,
//         y8 = e4m3(y / s), the quotient in fp32 as a product with 1 / s: within 3 units of its last
//         place, so that a value next to the middle of two e4m3 values may take the other one
// z, the sum of squares and the scales are fp32; z is rounded to bf16 once for residual_out and
// is normalised unrounded, y is rounded once to its output type.
#include <atomic>
#include <string>

#include <cuda_fp8.h>

#include "lm_common.cuh"

namespace lm {
namespace {

constexpr int kMaxHidden = 16384;
constexpr int kMaxGroups = kMaxHidden / 32;
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
  int num_tokens, hidden, group;
};

template <int VEC>
struct Vec;  // VEC bf16 values as one load
template <>
struct Vec<8> {
  uint4 v;
};
template <>
struct Vec<1> {
  uint16_t v;
};

__device__ __forceinline__ void unpack(const Vec<8>& a, float (&f)[8]) {
  unpack_bf16x2(a.v.x, f[0], f[1]);
  unpack_bf16x2(a.v.y, f[2], f[3]);
  unpack_bf16x2(a.v.z, f[4], f[5]);
  unpack_bf16x2(a.v.w, f[6], f[7]);
}
__device__ __forceinline__ void unpack(const Vec<1>& a, float (&f)[1]) { f[0] = bf16_bits_to_f32(a.v); }

__device__ __forceinline__ Vec<8> pack(const float (&f)[8]) {
  return {make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                     pack_bf16x2(f[6], f[7]))};
}
__device__ __forceinline__ Vec<1> pack(const float (&f)[1]) { return {f32_to_bf16_bits(f[0])}; }

__device__ __forceinline__ void store_e4m3(uint8_t* dst, const float (&f)[8]) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * i], f[4 * i + 1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * i + 2], f[4 * i + 3]), __NV_SATFINITE, __NV_E4M3);
    w[i] = lo | hi << 16;
  }
  *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
}
__device__ __forceinline__ void store_e4m3(uint8_t* dst, const float (&f)[1]) {
  *dst = __nv_cvt_float_to_fp8(f[0], __NV_SATFINITE, __NV_E4M3);
}

// Sum or maximum over the block; s_red is not written again before every thread has passed the
// next call's barrier on the other buffer.
template <bool MAX>
__device__ __forceinline__ float block_reduce(float v, float* s_red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float u = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? fmaxf(v, u) : v + u;
  }
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (lane == 0) s_red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = lane < warps ? s_red[lane] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float u = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? fmaxf(v, u) : v + u;
  }
  return v;
}

// A block takes rows blockIdx.x, + gridDim.x, ...: the row lives in registers (VPT pieces of VEC
// values a thread, piece i of thread t at column (i * blockDim + t) * VEC), the weight is loaded
// once, and the next row's loads are issued before this row's sums are joined. HBM-bound: measured
// 6.4 TB/s (99 % of the copy rate) at 16384 x 4096 with e4m3 output, 6.0 TB/s with bf16 output;
// 12.1 to 12.8 us at 4093 x 2048 (5.2 to 5.5 TB/s) and 1.5 us a call at 16 x 2048, both replayed from a
// graph. Rows that no 16-byte load fits (VEC 1, with 2-byte loads and 2- or 1-byte stores) run at 4.1 TB/s
// with bf16 output and 2.0 with e4m3 (16384 x 4095; 4096 x 1001: 10.4 and 17.4 us).
template <int VEC, int VPT, bool FP8>
__global__ void __launch_bounds__(VEC == 8 ? 256 : 1024)
    add_rms_norm_kernel(const NormParams p) {
  __shared__ float s_red[3][32];
  __shared__ uint32_t s_group[FP8 ? kMaxGroups : 1];
  const int H = p.hidden, pieces = H / VEC;
  auto col = [&](int i) { return (i * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)); };
  auto load = [&](const uint16_t* base, int64_t stride, int64_t t, Vec<VEC> (&v)[VPT]) {
    const Vec<VEC>* row = reinterpret_cast<const Vec<VEC>*>(base + t * stride);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      v[i] = Vec<VEC>{};
      if (col(i) < pieces) v[i] = row[col(i)];
    }
  };
  Vec<VEC> w[VPT], x[VPT], r[VPT];
  pdl_wait();
  pdl_trigger();
  load(p.weight, 0, 0, w);
  // the pieces' groups do not change from row to row
  const int groups = FP8 && p.group > 0 ? H / p.group : 1;
  const int per_group = FP8 && p.group > 0 ? p.group / VEC : pieces;  // pieces
  const bool by_lanes = per_group <= 32 && (per_group & (per_group - 1)) == 0;
  int group_of[VPT];
  bool leads[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    group_of[i] = FP8 && groups > 1 ? col(i) / per_group : 0;
    leads[i] = FP8 && col(i) == group_of[i] * per_group;
  }
  int t = blockIdx.x;
  if (t < p.num_tokens) {
    load(p.x, p.x_stride, t, x);
    if (p.residual != nullptr) load(p.residual, p.residual_stride, t, r);
  }
  for (int it = 0; t < p.num_tokens; t += gridDim.x, ++it) {
    float z[VPT][VEC];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      unpack(x[i], z[i]);
      if (p.residual != nullptr) {
        float f[VEC];
        unpack(r[i], f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) z[i][e] += f[e];
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) ss += z[i][e] * z[i][e];
    }
    if (t + gridDim.x < p.num_tokens) {
      load(p.x, p.x_stride, t + gridDim.x, x);
      if (p.residual != nullptr) load(p.residual, p.residual_stride, t + gridDim.x, r);
    }
    const float inv_rms = rsqrtf(block_reduce<false>(ss, s_red[it & 1]) / H + p.eps);
    if (p.residual_out != nullptr) {
      Vec<VEC>* row = reinterpret_cast<Vec<VEC>*>(p.residual_out + t * p.residual_out_stride);
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if (col(i) < pieces) row[col(i)] = pack(z[i]);
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float f[VEC];
      unpack(w[i], f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) z[i][e] = z[i][e] * inv_rms * f[e];
    }
    if constexpr (!FP8) {
      Vec<VEC>* row = reinterpret_cast<Vec<VEC>*>(p.y + t * p.y_stride);
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if (col(i) < pieces) row[col(i)] = pack(z[i]);
    } else {
      float top[VPT];  // max |y| of each piece, then of its group
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        top[i] = 0.f;
#pragma unroll
        for (int e = 0; e < VEC; ++e) top[i] = fmaxf(top[i], fabsf(z[i][e]));
      }
      if (groups == 1) {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) m = fmaxf(m, top[i]);
        m = block_reduce<true>(m, s_red[2]);
#pragma unroll
        for (int i = 0; i < VPT; ++i) top[i] = m;
        __syncthreads();  // one buffer for the maxima: read before the next row's are written
      } else if (by_lanes) {
        // a group is 4 .. 32 neighbouring lanes
#pragma unroll
        for (int i = 0; i < VPT; ++i)
          for (int o = per_group >> 1; o > 0; o >>= 1)
            top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
      } else {
        for (int g = threadIdx.x; g < groups; g += blockDim.x) s_group[g] = 0u;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < VPT; ++i)  // magnitudes order like their bits
          if (col(i) < pieces) atomicMax(&s_group[group_of[i]], __float_as_uint(top[i]));
        __syncthreads();
#pragma unroll
        for (int i = 0; i < VPT; ++i)
          if (col(i) < pieces) top[i] = __uint_as_float(s_group[group_of[i]]);
        __syncthreads();
      }
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        if (col(i) >= pieces) continue;
        const float s = fmaxf(top[i], kScaleFloor) * (1.f / kE4m3Max);
        const float inv = __fdividef(1.f, s);  // s < 2^126: within 2 units of its last place
#pragma unroll
        for (int e = 0; e < VEC; ++e) z[i][e] *= inv;
        store_e4m3(p.y8 + t * p.y8_stride + col(i) * VEC, z[i]);
        if (leads[i]) p.scales[static_cast<int64_t>(t) * groups + group_of[i]] = s;
      }
    }
  }
}

// Blocks of up to 256 threads (1024 for single values); as many as are resident at once.
template <int VEC, int VPT, bool FP8>
int launch_norm(const NormParams& p, cudaStream_t s) {
  const int pieces = p.hidden / VEC;
  const int threads = ((pieces + VPT - 1) / VPT + 31) / 32 * 32;
  static std::atomic<int> resident[64][33];  // blocks of this many warps that the GPU holds at once
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return fail(LM_ERR_UNSUPPORTED, "lm_add_rms_norm: device index >= 64");
  int most = resident[dev][threads / 32].load(std::memory_order_relaxed);
  if (most == 0) {
    int sms = 0, per_sm = 0;
    int rc = check_cuda(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev), "lm_add_rms_norm");
    if (!rc)
      rc = check_cuda(cudaOccupancyMaxActiveBlocksPerMultiprocessor(
                          &per_sm, add_rms_norm_kernel<VEC, VPT, FP8>, threads, 0),
                      "lm_add_rms_norm: occupancy");
    if (rc) return rc;
    most = sms * (per_sm > 0 ? per_sm : 1);
    resident[dev][threads / 32].store(most, std::memory_order_relaxed);
  }
  const int grid = p.num_tokens < most ? p.num_tokens : most;
  return check_cuda(launch_dependent(add_rms_norm_kernel<VEC, VPT, FP8>, dim3(grid), dim3(threads), 0, s, p),
                    "lm_add_rms_norm");
}

template <bool FP8>
int launch_norm(const NormParams& p, bool wide, cudaStream_t s) {
  if (wide) {
    if (p.hidden <= 2048) return launch_norm<8, 1, FP8>(p, s);
    if (p.hidden <= 4096) return launch_norm<8, 2, FP8>(p, s);
    if (p.hidden <= 8192) return launch_norm<8, 4, FP8>(p, s);
    return launch_norm<8, 8, FP8>(p, s);
  }
  if (p.hidden <= 4096) return launch_norm<1, 4, FP8>(p, s);
  return p.hidden <= 8192 ? launch_norm<1, 8, FP8>(p, s) : launch_norm<1, 16, FP8>(p, s);
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
  if (hidden_size <= 0 || hidden_size > kMaxHidden || num_tokens < 0 || num_tokens > 0x3fffffff)
    return fail(LM_ERR_INVALID_ARGUMENT,
                "lm_add_rms_norm: need 1 <= hidden_size <= 16384 and 0 <= num_tokens < 2^30");
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
                     residual_out_stride, y_stride, y8_stride, eps,
                     static_cast<int>(num_tokens), hidden_size, group_size};
  // 16-byte loads where every row starts on a 16-byte boundary, else single values
  auto at16 = [](const void* ptr, int64_t stride) {
    return ptr == nullptr || ((reinterpret_cast<uintptr_t>(ptr) & 15) == 0 && stride % 8 == 0);
  };
  const bool wide = hidden_size % 8 == 0 && at16(x, x_stride) && at16(residual, residual_stride) &&
                    at16(weight, 0) && at16(residual_out, residual_out_stride) && at16(y, y_stride) &&
                    (reinterpret_cast<uintptr_t>(y8) & 7) == 0 && y8_stride % 8 == 0;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return y8 != nullptr ? launch_norm<true>(p, wide, s) : launch_norm<false>(p, wide, s);
}
