// mx_quantise.hip -- values to MXFP4: e2m1 codes, two a byte with the first
// in the low nibble, and a scale byte for every 32.
//
// Each value is read once and the bytes are written once: bound by memory.  A
// thread holds eight consecutive values, a quad one block, so a block's
// largest magnitude takes two lane exchanges and no shared memory.
#include <hip/hip_runtime.h>

#include "mx_device.h"

namespace ptwm {
namespace {

constexpr uint32_t kThreads = 256;

template <uint32_t T>
__device__ __forceinline__ uint32_t codes8(const Raw8<T>& r, float scale) {
  uint32_t c = 0;
  if constexpr (T == kTypeF32) {
    float v[8];
    values_of<T>(r, v);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], scale, 3);
  } else if constexpr (T == kTypeBf16) {
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, (uint32_t)r.w[0][0]), scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, (uint32_t)r.w[0][1]), scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, (uint32_t)r.w[0][2]), scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, (uint32_t)r.w[0][3]), scale, 3);
  } else {
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2, (uint32_t)r.w[0][0]), scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2, (uint32_t)r.w[0][1]), scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2, (uint32_t)r.w[0][2]), scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2, (uint32_t)r.w[0][3]), scale, 3);
  }
  return c;
}

// A block's largest magnitude 1.m * 2^(E-127) and its scale byte:
//   saturate  E - 2, which leaves the magnitude in [4, 8); above 6, e2m1's
//             largest value, it is cut to 6;
//   else      the smallest with which nothing is above 6 = 1.5 * 2^2: one
//             more where 1.m > 1.5.
// At least 0: below 2^-125 blocks share the smallest scale.  The conversion
// divides by the scale, which is exact, and rounds to nearest even.  A block
// with an infinity or NaN gets the scale NaN and zero codes.
template <uint32_t T>
__global__ __launch_bounds__(kThreads) void mxfp4_quantise_kernel(MxQuantiseArgs a) {
  const uint32_t per_row = a.cols / 8;
  const uint32_t at = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t row = at / per_row;
  if (row >= a.rows) return;  // whole quads
  const uint32_t c = (at - row * per_row) * 8;
  const Raw8<T> r = load_raw8<T>(a.x.ptr + (row * a.x.stride + c) * type_bytes(T));
  float v[8];
  values_of<T>(r, v);
  uint32_t m = 0;  // magnitudes compare as integers, infinities and NaN last
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, f32_bits(v[i]) & 0x7FFFFFFFu);
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xF, 0xF, true));  // lanes 1 0 3 2
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xF, 0xF, true));  // lanes 2 3 0 1
  const bool broken = m >= 0x7F800000u;
  const uint32_t b = (uint32_t)max((int)(m >> 23) - 2 + (!a.saturate && (m & 0x7FFFFFu) > 0x400000u ? 1 : 0), 0);
  const uint32_t codes = codes8<T>(r, scale_f32(b));
  st4(a.codes.ptr + row * a.codes.stride + c / 2, broken ? 0u : codes);
  if ((threadIdx.x & 3) == 0)
    g_st<uint8_t>(a.scales.ptr + row * a.scales.stride + c / kMxBlock, (uint8_t)(broken ? 255u : b));
}

template <uint32_t T>
hipError_t quantise_of(const MxQuantiseArgs& a, hipStream_t stream) {
  const uint32_t per_row = a.cols / 8;
  return in_parts(a.rows, (kMaxThreads - kThreads) / per_row, [&](uint64_t first, uint64_t rows) {
    const MxQuantiseArgs p{rows_from(a.x, first, type_bytes(T)), rows_from(a.codes, first, 1),
                           rows_from(a.scales, first, 1), rows, a.cols, a.saturate};
    return launch(mxfp4_quantise_kernel<T>, (rows * per_row + kThreads - 1) / kThreads, kThreads, p, stream);
  });
}

}  // namespace

hipError_t launch_mxfp4_quantise(uint32_t type, const MxQuantiseArgs& a, hipStream_t stream) {
  switch (type) {
    case kTypeF32: return quantise_of<kTypeF32>(a, stream);
    case kTypeF16: return quantise_of<kTypeF16>(a, stream);
    case kTypeBf16: return quantise_of<kTypeBf16>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace ptwm
