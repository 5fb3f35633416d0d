// mx_ops.h -- operators on microscaled (MX) blocks: the product with MXFP4
// weights as a decode restores them, and the norm and gated activation whose
// 8-bit outputs feed it.
//
// A block is 32 consecutive values of a row with one scale byte b (E8M0):
// 2^(b - 127), or NaN for 255.  Weights are e2m1 codes, two a byte, the first
// value in the low nibble; activations in 8 bits are e4m3 codes.
#pragma once

#include "ptwm_common.h"

namespace ptwm {

// Element types by their public dtype codes (dtype.rs:79-103).
constexpr uint32_t kTypeF32 = 1, kTypeF16 = 4, kTypeBf16 = 6, kTypeE4m3 = 29;
constexpr uint32_t kMxBlock = 32;
__host__ __device__ constexpr uint32_t type_bytes(uint32_t type) {
  return type == kTypeF32 ? 4 : type == kTypeE4m3 ? 1 : 2;
}

// A row-major operand: device address and row stride in elements (of scales:
// in bytes).  Addresses need no alignment beyond the element's.
struct MxRows {
  uint64_t ptr;
  uint64_t stride;
};

struct MxNormArgs {
  MxRows x, residual, sum, codes, scales;  // residual.ptr, sum.ptr: 0 if absent
  uint64_t weight;
  uint64_t rows;
  uint32_t cols;
  float eps;
  uint32_t weight_type;
};

struct MxSwigluArgs {
  MxRows gate, up, codes, scales;
  uint64_t rows;
  uint32_t cols;
};

struct MxLinearArgs {
  MxRows x, x_scales, weight, scales, out;  // x_scales.ptr: 0 unless x is e4m3; weight.stride in bytes
  uint64_t bias;                            // 0 if absent; of the output's type
  uint64_t tokens;
  uint32_t rows;   // output features
  uint32_t cols;   // input features, a multiple of kMxBlock
  uint32_t out_type;
};

// Each queues its work on `stream` of the current device and returns.
hipError_t launch_rms_norm_mx(uint32_t type, const MxNormArgs& a, hipStream_t stream);
hipError_t launch_swiglu_mx(uint32_t type, const MxSwigluArgs& a, hipStream_t stream);
hipError_t launch_mxfp4_linear(uint32_t x_type, const MxLinearArgs& a, hipStream_t stream);

}  // namespace ptwm
