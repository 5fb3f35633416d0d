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

constexpr uint32_t kThreads = 256;

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
  return v;
}

__device__ __forceinline__ void load_weight8(const MxNormArgs& a, uint32_t c, float (&v)[8]) {
  if (a.weight_type == kTypeBf16)
    load8<kTypeBf16>(a.weight + (uint64_t)c * 2, v);
  else if (a.weight_type == kTypeF16)
    load8<kTypeF16>(a.weight + (uint64_t)c * 2, v);
  else
    load8<kTypeF32>(a.weight + (uint64_t)c * 4, v);
}

// Codes and scale of a row's values c .. c+7.
__device__ __forceinline__ void store_codes(const MxRows& codes, const MxRows& scales, uint64_t row, uint64_t c,
                                            const float (&v)[8]) {
  uint32_t lo, hi;
  const uint32_t b = quantise8(v, lo, hi);
  st8(codes.ptr + row * codes.stride + c, lo | (uint64_t)hi << 32);
  if ((threadIdx.x & 3) == 0) g_st<uint8_t>(scales.ptr + row * scales.stride + c / kMxBlock, (uint8_t)b);
}

// s = x + residual, y = s * rsqrt(mean(s^2) + eps) * weight in 32 bits; sum
// receives s in x's type, codes and scales receive y.  W wavefronts to a row,
// which they hold in registers in CH pieces of 8 values a thread, so each
// input is read once, all of it requested before any is used; with CH = 0 rows
// of any length are read twice.
template <uint32_t T, int W, int CH>
__global__ __launch_bounds__(W > 4 ? 64 * W : kThreads) void rms_norm_mx_kernel(MxNormArgs a) {
  constexpr uint32_t kRowThreads = 64 * W, kRows = W > 4 ? 1 : 4 / W;
  __shared__ float part[W];
  const uint64_t row = (uint64_t)blockIdx.x * kRows + threadIdx.x / kRowThreads;
  if (kRows > 1 && row >= a.rows) return;  // whole wavefronts, which meet no other
  const uint32_t first = threadIdx.x % kRowThreads * 8;
  const uint64_t x = a.x.ptr + row * a.x.stride * type_bytes(T);
  const uint64_t r = a.residual.ptr + row * a.residual.stride * type_bytes(T);
  constexpr int N = CH ? CH : 1;
  Raw8<T> xv[N], rv[N];
  float v[N][8], w[N][8], total = 0;
  auto request = [&](int k, uint32_t c) {
    xv[k] = load_raw8<T>(x + (uint64_t)c * type_bytes(T));
    if (a.residual.ptr) rv[k] = load_raw8<T>(r + (uint64_t)c * type_bytes(T));
  };
  auto take = [&](int k) {
    values_of<T>(xv[k], v[k]);
    if (a.residual.ptr) {
      float u[8];
      values_of<T>(rv[k], u);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[k][i] += u[i];
    }
  };
  auto add = [&](int k) {
#pragma unroll
    for (int i = 0; i < 8; ++i) total += v[k][i] * v[k][i];
  };
  if constexpr (CH > 0) {
    // past the row's end its last piece is loaded again and not used
#pragma unroll
    for (int k = 0; k < CH; ++k) request(k, min(first + k * kRowThreads * 8, a.cols - 8));
#pragma unroll
    for (int k = 0; k < CH; ++k) load_weight8(a, min(first + k * kRowThreads * 8, a.cols - 8), w[k]);
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      take(k);
      if (first + k * kRowThreads * 8 < a.cols) add(k);
    }
  } else {
    for (uint32_t c = first; c < a.cols; c += kRowThreads * 8) {
      request(0, c);
      take(0);
      add(0);
    }
  }
  total = wave_sum(total);
  if constexpr (kRows == 1) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = total;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) total += part[i];
  }
  const float scale = 1.0f / sqrtf(total / (float)a.cols + a.eps);
  auto finish = [&](uint32_t c, float(&y)[8], const float(&g)[8]) {
    if (a.sum.ptr) store8<T>(a.sum.ptr + (row * a.sum.stride + c) * type_bytes(T), y);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = y[i] * scale * g[i];
    store_codes(a.codes, a.scales, row, c, y);
  };
  // the sum is written after the last read of its place: it may be x or the residual
  if constexpr (CH > 0) {
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const uint32_t c = first + k * kRowThreads * 8;
      if (c < a.cols) finish(c, v[k], w[k]);
    }
  } else {
    for (uint32_t c = first; c < a.cols; c += kRowThreads * 8) {
      request(0, c);
      load_weight8(a, c, w[0]);
      take(0);
      finish(c, v[0], w[0]);
    }
  }
}

// y = gate / (1 + exp(-gate)) * up in 32 bits.  The exponential and the
// reciprocal are the hardware's, each within a unit in the last place: with
// the library's exact forms the arithmetic took longer than the memory
// (2048x14336 bf16: 35 us, 28 to 29.5 this way).  The exponential's argument,
// -gate * log2(e), is carried in two parts, whose low one is multiplied in
// afterwards: rounded to 32 bits alone it puts the exponential off by half a
// unit for every unit of |gate| (the result by 65 * 2^-24 at gate = -87).
// The reciprocal's argument is a quarter of the sum, so that it stays a normal
// number as far as the exponential is finite, and the other quarter is taken
// of the reciprocal: a gate below the normal numbers may have none.  (Below
// gate = -87.3 that takes it below them itself, up to 4 * 2^-24.)
__device__ __forceinline__ float exp_of_minus(float g) {
  constexpr float kHigh = -0x1.715476p+0f, kLow = -0x1.4ae0c0p-26f;  // -log2(e) = kHigh + kLow
  const float t = g * kHigh;
  // an infinity has no low part: the limit makes NaN a number there, and no low part reaches it
  const float low = fminf(__builtin_fmaf(g, kLow, __builtin_fmaf(g, kHigh, -t)), 1.0f);
  return __builtin_amdgcn_exp2f(t) * __builtin_fmaf(low, 0x1.62e430p-1f, 1.0f);
}

template <uint32_t T>
__global__ __launch_bounds__(kThreads) void swiglu_mx_kernel(MxSwigluArgs a) {
  const uint32_t per_row = a.cols / 8;
  const uint64_t at = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
  const uint64_t row = at / per_row;
  if (row >= a.rows) return;
  const uint64_t c = (at - row * per_row) * 8;
  float g[8], u[8];
  load8<T>(a.gate.ptr + (row * a.gate.stride + c) * type_bytes(T), g);
  load8<T>(a.up.ptr + (row * a.up.stride + c) * type_bytes(T), u);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float e = exp_of_minus(g[i]);
    g[i] = __builtin_amdgcn_rcpf(__builtin_fmaf(e, 0.25f, 0.25f)) * 0.25f * g[i] * u[i];
  }
  store_codes(a.codes, a.scales, row, c, g);
}

template <uint32_t T, int W, int CH>
hipError_t norm_by(const MxNormArgs& a, hipStream_t stream) {
  constexpr uint32_t kRows = W > 4 ? 1 : 4 / W, kGroup = W > 4 ? 64 * W : kThreads, kSize = type_bytes(T);
  return in_parts(a.rows, kMaxThreads / kGroup * kRows, [&](uint64_t first, uint64_t rows) {
    MxNormArgs p = a;
    p.x = rows_from(a.x, first, kSize), p.residual = rows_from(a.residual, first, kSize);
    p.sum = rows_from(a.sum, first, kSize);
    p.codes = rows_from(a.codes, first, 1), p.scales = rows_from(a.scales, first, 1);
    p.rows = rows;
    return launch(rms_norm_mx_kernel<T, W, CH>, (rows + kRows - 1) / kRows, kGroup, p, stream);
  });
}

template <uint32_t T>
hipError_t norm_of(const MxNormArgs& a, hipStream_t stream) {
  // Few pieces a thread: measured (us, against four wavefronts with as many pieces as it takes) 1x4096 bf16 2.7 and 2.9,
  // 2048x4096 11.3 and 11.5, 64x14336 4.4 and 8.4, 2048x8192 25.5 and 27.4.
  if (a.cols <= 512) return norm_by<T, 1, 1>(a, stream);
  if (a.cols <= 1024) return norm_by<T, 1, 2>(a, stream);
  if (a.cols <= 2048) return norm_by<T, 4, 1>(a, stream);
  if (a.cols <= 4096) return norm_by<T, 8, 1>(a, stream);
  if (a.cols <= 8192) return norm_by<T, 16, 1>(a, stream);
  if (a.cols <= 16384) return norm_by<T, 16, 2>(a, stream);
  return norm_by<T, 16, 0>(a, stream);
}

template <uint32_t T>
hipError_t swiglu_of(const MxSwigluArgs& a, hipStream_t stream) {
  const uint32_t per_row = a.cols / 8;
  return in_parts(a.rows, (kMaxThreads - kThreads) / per_row, [&](uint64_t first, uint64_t rows) {
    const MxSwigluArgs p{rows_from(a.gate, first, type_bytes(T)), rows_from(a.up, first, type_bytes(T)),
                         rows_from(a.codes, first, 1), rows_from(a.scales, first, 1), rows, a.cols};
    return launch(swiglu_mx_kernel<T>, (rows * per_row + kThreads - 1) / kThreads, kThreads, p, stream);
  });
}

}  // namespace

hipError_t launch_rms_norm_mx(uint32_t type, const MxNormArgs& a, hipStream_t stream) {
  switch (type) {
    case kTypeF32: return norm_of<kTypeF32>(a, stream);
    case kTypeF16: return norm_of<kTypeF16>(a, stream);
    case kTypeBf16: return norm_of<kTypeBf16>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_swiglu_mx(uint32_t type, const MxSwigluArgs& a, hipStream_t stream) {
  switch (type) {
    case kTypeF32: return swiglu_of<kTypeF32>(a, stream);
    case kTypeF16: return swiglu_of<kTypeF16>(a, stream);
    case kTypeBf16: return swiglu_of<kTypeBf16>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace ptwm
