// mx_matmul.hip -- out = x * W^T (+ bias) with both matrices in MXFP4.
//
//   out[t, n] = sum_b 2^(X[t, b] + S[n, b] - 254) * sum_k<32 e2m1(x[t, 32b + k]) * e2m1(W[n, 32b + k]) + bias[n]
//
// The matrix instruction takes codes and scales as they lie in memory
// (v_mfma_scale_f32_16x16x128_f8f6f4).  With e2m1 on both sides it sums in 32
// bits: products of a block are whole multiples of 1/4 up to 36 and their
// sums, up to 1152, are exact; checked against 64 bits, an instruction's four
// blocks and accumulator are off by 2^-23 of the sum of magnitudes at most,
// whatever the scales, subnormal numbers included.
#include <hip/hip_runtime.h>

#include "mx_device.h"

namespace ptwm {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// 16 weight rows and 16 tokens, 128 values of each: lane l holds row (token) l % 16 and block l / 16, and its scale.
__device__ __forceinline__ f32x4 mfma_mx4(u32x4 w, uint32_t ws, u32x4 x, uint32_t xs, f32x4 c) {
  const i32x8 wv = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
  const i32x8 xv = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, xv, c, 4, 4, 0, (int)ws, 0, (int)xs);
}

// A 16x16 tile of outputs by one workgroup, whose wavefronts take turns in
// steps of 128 values along the rows and add up in LDS, operands straight from
// memory.
__global__ __launch_bounds__(256) void mxfp4_matmul_kernel(MxLinearArgs a) {
  __shared__ float part[4][16][17];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, i = lane & 15;
  const uint32_t row_tiles = (a.rows + 15) / 16;
  const uint32_t n0 = blockIdx.x % row_tiles * 16;
  const uint64_t t0 = (uint64_t)(blockIdx.x / row_tiles) * 16;
  const uint32_t blocks = a.cols / kMxBlock;
  // past the last row or token the last one is computed again and not stored
  const uint64_t n = min(n0 + i, a.rows - 1);
  const uint64_t t = min(t0 + i, a.tokens - 1);
  const uint64_t w = a.weight.ptr + n * a.weight.stride, s = a.scales.ptr + n * a.scales.stride;
  const uint64_t x = a.x.ptr + t * a.x.stride, xs = a.x_scales.ptr + t * a.x_scales.stride;
  f32x4 acc = {};
  for (uint32_t k = wave * 4 + q; k < (blocks + 3) / 4 * 4; k += 16) {
    u32x4 wv = {}, xv = {};
    uint32_t ws = 127, sx = 127;
    if (k < blocks) {  // the last step may be short: zero codes there
      wv = ld16(w + (uint64_t)k * 16), xv = ld16(x + (uint64_t)k * 16);
      ws = g_ld<uint8_t>(s + k), sx = g_ld<uint8_t>(xs + k);
    }
    acc = mfma_mx4(wv, ws, xv, sx, acc);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) part[wave][i][q * 4 + j] = acc[j];
  __syncthreads();
  if (threadIdx.x < 64) {
    const uint32_t ot = threadIdx.x >> 2, on = (threadIdx.x & 3) * 4;
    f32x4 v = {};
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += part[g][ot][on + j];
    if (t0 + ot < a.tokens) store4(a, t0 + ot, n0 + on, v);
  }
}

}  // namespace

hipError_t launch_mxfp4_matmul(const MxLinearArgs& a, hipStream_t stream) {
  return launch_tiles<1, 16, 16>(mxfp4_matmul_kernel, 256, a, stream);
}

}  // namespace ptwm
