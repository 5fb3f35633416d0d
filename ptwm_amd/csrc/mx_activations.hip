// mx_activations.hip -- activations in 8 bits for the MXFP4 product: the
// root-mean-square norm with the residual's addition, and the gated
// activation silu(gate) * up.
//
// Both read their inputs once and are bound by memory.  A thread holds eight
// consecutive values, a quad one block of 32, so a block's largest magnitude
// takes two lane exchanges and no shared memory.
#include <hip/hip_runtime.h>

#include "mx_device.h"

namespace ptwm {
namespace {

constexpr uint32_t kNormThreads = 256;

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
  return v;
}

// s = x + residual, y = s * rsqrt(mean(s^2) + eps) * weight in 32 bits; sum
// receives s in x's type, codes and scales receive y.  One workgroup a row.
template <uint32_t T, uint32_t WT>
__global__ __launch_bounds__(kNormThreads) void rms_norm_mx_kernel(MxNormArgs a) {
  __shared__ float part[kNormThreads / 64];
  const uint64_t row = blockIdx.x;
  const uint64_t x = a.x.ptr + row * a.x.stride * type_bytes(T);
  const uint64_t r = a.residual.ptr + row * a.residual.stride * type_bytes(T);
  auto load = [&](uint32_t c, float(&v)[8]) {
    load8<T>(x + (uint64_t)c * type_bytes(T), v);
    if (a.residual.ptr) {
      float w[8];
      load8<T>(r + (uint64_t)c * type_bytes(T), w);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += w[i];
    }
  };
  float total = 0;
  for (uint32_t c = threadIdx.x * 8; c < a.cols; c += kNormThreads * 8) {
    float v[8];
    load(c, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) total += v[i] * v[i];
  }
  total = wave_sum(total);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = total;
  __syncthreads();
  total = 0;
#pragma unroll
  for (uint32_t i = 0; i < kNormThreads / 64; ++i) total += part[i];
  const float scale = 1.0f / sqrtf(total / (float)a.cols + a.eps);
  // the sum is written here, after its last read: it may be x or the residual
  for (uint32_t c = threadIdx.x * 8; c < a.cols; c += kNormThreads * 8) {
    float v[8], w[8];
    load(c, v);
    if (a.sum.ptr) store8<T>(a.sum.ptr + (row * a.sum.stride + c) * type_bytes(T), v);
    load8<WT>(a.weight + (uint64_t)c * type_bytes(WT), w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] * scale * w[i];
    uint32_t lo, hi;
    const uint32_t b = quantise8(v, lo, hi);
    st8(a.codes.ptr + row * a.codes.stride + c, lo | (uint64_t)hi << 32);
    if ((threadIdx.x & 3) == 0) g_st<uint8_t>(a.scales.ptr + row * a.scales.stride + c / kMxBlock, (uint8_t)b);
  }
}

// y = gate / (1 + exp(-gate)) * up in 32 bits.
template <uint32_t T>
__global__ __launch_bounds__(256) void swiglu_mx_kernel(MxSwigluArgs a) {
  const uint32_t per_row = a.cols / 8;
  const uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const uint64_t row = at / per_row;
  if (row >= a.rows) return;
  const uint64_t c = (at - row * per_row) * 8;
  float g[8], u[8];
  load8<T>(a.gate.ptr + (row * a.gate.stride + c) * type_bytes(T), g);
  load8<T>(a.up.ptr + (row * a.up.stride + c) * type_bytes(T), u);
#pragma unroll
  for (int i = 0; i < 8; ++i) g[i] = g[i] / (1.0f + expf(-g[i])) * u[i];
  uint32_t lo, hi;
  const uint32_t b = quantise8(g, lo, hi);
  st8(a.codes.ptr + row * a.codes.stride + c, lo | (uint64_t)hi << 32);
  if ((threadIdx.x & 3) == 0) g_st<uint8_t>(a.scales.ptr + row * a.scales.stride + c / kMxBlock, (uint8_t)b);
}

template <uint32_t T>
hipError_t norm_of(uint32_t weight_type, const MxNormArgs& a, hipStream_t stream) {
  switch (weight_type) {
    case kTypeF32: return launch(rms_norm_mx_kernel<T, kTypeF32>, a.rows, kNormThreads, a, stream);
    case kTypeF16: return launch(rms_norm_mx_kernel<T, kTypeF16>, a.rows, kNormThreads, a, stream);
    case kTypeBf16: return launch(rms_norm_mx_kernel<T, kTypeBf16>, a.rows, kNormThreads, a, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

hipError_t launch_rms_norm_mx(uint32_t type, uint32_t weight_type, const MxNormArgs& a, hipStream_t stream) {
  switch (type) {
    case kTypeF32: return norm_of<kTypeF32>(weight_type, a, stream);
    case kTypeF16: return norm_of<kTypeF16>(weight_type, a, stream);
    case kTypeBf16: return norm_of<kTypeBf16>(weight_type, a, stream);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_swiglu_mx(uint32_t type, const MxSwigluArgs& a, hipStream_t stream) {
  const uint64_t groups = (a.rows * (a.cols / 8) + 255) / 256;
  switch (type) {
    case kTypeF32: return launch(swiglu_mx_kernel<kTypeF32>, groups, 256, a, stream);
    case kTypeF16: return launch(swiglu_mx_kernel<kTypeF16>, groups, 256, a, stream);
    case kTypeBf16: return launch(swiglu_mx_kernel<kTypeBf16>, groups, 256, a, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace ptwm
