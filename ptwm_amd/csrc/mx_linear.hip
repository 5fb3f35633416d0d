// mx_linear.hip -- out = x * W^T (+ bias) with MXFP4 weights W, read as a
// decode restores them.
//
//   out[t, n] = sum_k x[t, k] * e2m1(W[n, k]) * 2^(S[n, k/32] - 127) + bias[n]
//
// The weights are the matrix instruction's first operand (16 rows), the
// tokens its second, and sums are held in 32 bits.  Both operands are widened
// to bf16, in which every value is exact, and so are products in 32 bits:
//   - a weight, a code times its scale, has 2 significant bits and 8 exponent
//     bits (v_cvt_scalef32_pk_bf16_fp4, subnormals included);
//   - x in e4m3 with scales has 4 significant bits
//     (v_cvt_scalef32_pk_bf16_fp8);
//   - x in f16 or f32 is split into two or three bf16 values whose sum is x,
//     one product each.
// The instruction that takes codes and scales as they lie in memory
// (v_mfma_scale_f32_16x16x128_f8f6f4) would halve the matrix time with 8-bit
// x, but it adds the products of eight neighbours with 13 bits below the
// largest of them: measured, sums are off by 1.2e-5 of their norm with
// normal activations, against 2.5e-8 here, and by 2^-12 of the sum of
// magnitudes where codes spread over e4m3's whole range.
#include <hip/hip_runtime.h>

#include "mx_device.h"

namespace ptwm {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// bf16 parts that hold a value of type T exactly.
constexpr int parts_of(uint32_t type) { return type == kTypeF32 ? 3 : type == kTypeF16 ? 2 : 1; }

// Eight values at address a as P bf16 parts, each cut from what the ones
// before it leave (truncation, so nothing rounds up to infinity); the rest of
// an infinity or NaN is zero, which keeps it what it is in the sum.  scale:
// of e4m3 codes, read for its exponent only.
template <uint32_t T>
__device__ __forceinline__ void load_parts(uint64_t a, float scale, u32x4 (&p)[parts_of(T)]) {
  if constexpr (T == kTypeBf16) {
    p[0] = ld16(a);
  } else if constexpr (T == kTypeE4m3) {
    const uint64_t w = ld8(a);
    const uint32_t w0 = (uint32_t)w, w1 = (uint32_t)(w >> 32);
    p[0] = u32x4_make(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, true)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, true)));
  } else {
    float v[8];
    load8<T>(a, v);
#pragma unroll
    for (int i = 0; i < 8; ++i)  // a NaN whose cut would read as an infinity
      if (v[i] != v[i]) v[i] = bits_f32(0x7FC00000u);
#pragma unroll
    for (int j = 0; j < parts_of(T); ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t b0 = f32_bits(v[2 * i]), b1 = f32_bits(v[2 * i + 1]);
        p[j][i] = __builtin_amdgcn_perm(b1, b0, 0x07060302u);
        if (j + 1 < parts_of(T)) {
          const float h0 = bits_f32(b0 & 0xFFFF0000u), h1 = bits_f32(b1 & 0xFFFF0000u);
          v[2 * i] = __builtin_isfinite(h0) ? v[2 * i] - h0 : 0.0f;
          v[2 * i + 1] = __builtin_isfinite(h1) ? v[2 * i + 1] - h1 : 0.0f;
        }
      }
    }
  }
}

// A 16x16 tile of outputs by one workgroup, whose wavefronts take turns in
// steps of 128 values (four blocks) along the rows and add up in LDS.  Lane l
// holds weight row l % 16 and block l / 16 of the step, and token l % 16.
template <uint32_t T, uint32_t OT>
__global__ __launch_bounds__(256) void mxfp4_linear_kernel(MxLinearArgs a) {
  __shared__ float part[4][16][17];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, i = lane & 15;
  const uint32_t row_tiles = (a.rows + 15) / 16;
  const uint32_t n0 = blockIdx.x % row_tiles * 16;
  const uint64_t t0 = (uint64_t)(blockIdx.x / row_tiles) * 16;
  const uint32_t blocks = a.cols / kMxBlock;
  // past the last row or token the last one is computed again and not stored
  const uint64_t n = min(n0 + i, a.rows - 1);
  const uint64_t t = min(t0 + i, a.tokens - 1);
  const uint64_t w = a.weight.ptr + n * a.weight.stride;
  const uint64_t s = a.scales.ptr + n * a.scales.stride;
  const uint64_t x = a.x.ptr + t * a.x.stride * type_bytes(T);
  const uint64_t xs = a.x_scales.ptr + t * a.x_scales.stride;
  f32x4 acc = {};
  for (uint32_t k = wave * 4; k < blocks; k += 16) {
    const bool in = k + q < blocks;  // the last step may be short: zero codes there
    u32x4 wv = {};
    uint32_t sv = 127;
    if (in) {
      wv = ld16(w + (uint64_t)(k + q) * 16);
      sv = g_ld<uint8_t>(s + k + q);
    }
    // the conversions read the scale's exponent only: byte 0 is 2^-127, 255 is NaN
    const float scale = bits_f32(sv << 23);
    float x_scale = 1.0f;
    if constexpr (T == kTypeE4m3)
      if (in) x_scale = bits_f32((uint32_t)g_ld<uint8_t>(xs + k + q) << 23);
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      u32x4 p[parts_of(T)] = {};
      if (in) load_parts<T>(x + ((uint64_t)(k + q) * 32 + f * 8) * type_bytes(T), x_scale, p);
      const uint32_t wf = wv[f];
      const u32x4 A = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(wf, scale, 0)),
                       __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(wf, scale, 1)),
                       __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(wf, scale, 2)),
                       __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(wf, scale, 3))};
#pragma unroll
      for (int j = parts_of(T) - 1; j >= 0; --j)
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, A), __builtin_bit_cast(bf16x8, p[j]),
                                                      acc, 0, 0, 0);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) part[wave][i][q * 4 + j] = acc[j];
  __syncthreads();
  const uint32_t on = threadIdx.x & 15, ot = threadIdx.x >> 4;
  if (n0 + on < a.rows && t0 + ot < a.tokens) {
    float v = part[0][ot][on] + part[1][ot][on] + part[2][ot][on] + part[3][ot][on];
    if (a.bias) v += load1<OT>(a.bias + (uint64_t)(n0 + on) * type_bytes(OT));
    store1<OT>(a.out.ptr + ((t0 + ot) * a.out.stride + n0 + on) * type_bytes(OT), v);
  }
}

template <uint32_t T>
hipError_t linear_of(uint32_t out_type, const MxLinearArgs& a, hipStream_t stream) {
  const uint64_t tiles = (uint64_t)((a.rows + 15) / 16) * ((a.tokens + 15) / 16);
  if (tiles > 0x7FFFFFFFu) return hipErrorInvalidValue;
  const dim3 grid((uint32_t)tiles), block(256);
  switch (out_type) {
    case kTypeF32: hipLaunchKernelGGL((mxfp4_linear_kernel<T, kTypeF32>), grid, block, 0, stream, a); break;
    case kTypeF16: hipLaunchKernelGGL((mxfp4_linear_kernel<T, kTypeF16>), grid, block, 0, stream, a); break;
    case kTypeBf16: hipLaunchKernelGGL((mxfp4_linear_kernel<T, kTypeBf16>), grid, block, 0, stream, a); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_mxfp4_linear(uint32_t x_type, uint32_t out_type, const MxLinearArgs& a, hipStream_t stream) {
  switch (x_type) {
    case kTypeF32: return linear_of<kTypeF32>(out_type, a, stream);
    case kTypeF16: return linear_of<kTypeF16>(out_type, a, stream);
    case kTypeBf16: return linear_of<kTypeBf16>(out_type, a, stream);
    case kTypeE4m3: return linear_of<kTypeE4m3>(out_type, a, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace ptwm
