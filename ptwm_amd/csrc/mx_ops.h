// mx_ops.h -- operators on microscaled (MX) blocks: the product with MXFP4
// weights as a decode restores them, the norm and gated activation whose
// 8-bit outputs feed it, the quantisation to MXFP4, the product of two MXFP4
// matrices, and a mixture-of-experts layer on MXFP4 experts.
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
// bf16 parts that hold a value of type T exactly.
constexpr int parts_of(uint32_t type) { return type == kTypeF32 ? 3 : type == kTypeF16 ? 2 : 1; }

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

struct MxQuantiseArgs {
  MxRows x, codes, scales;  // codes.stride in bytes
  uint64_t rows;
  uint32_t cols;
  bool saturate;
};

// The weights of all experts for one of their products: the operand of an
// expert, how far apart experts lie (bytes), and a bias of the output's type
// (bias 0: none) with its strides in elements.
struct MxExperts {
  MxRows codes, scales;
  uint64_t codes_expert, scales_expert;
  uint64_t bias, bias_expert, bias_stride;
};

struct MxMoeArgs {
  MxRows x, router, out;
  uint64_t router_bias;  // of the router's type; 0 if absent
  MxExperts gate, up, down;
  uint64_t experts_out, weights_out;  // int32 and f32 [tokens][top_k]; 0 if absent
  uint64_t workspace;
  uint64_t tokens;
  uint32_t experts, top_k, cols, inner;
  uint32_t x_type, router_type, out_type;
};
constexpr uint64_t kMoeMaxExperts = 1024, kMoeMaxTopK = 32, kMoeMaxWidth = 1 << 17;
constexpr uint32_t kMoeTokens = 64;  // of a launch; longer calls run in several
constexpr uint32_t kMoeStep = 256;   // values of a row that go through LDS together: a cache line of codes
// h's parts: all 24 bits of a sum in 32, whatever the outputs' type.
constexpr uint32_t kMoeInnerParts = 3;
// Bytes of workspace, at a multiple of 256, that a call takes.
uint64_t mxfp4_moe_workspace(const MxMoeArgs& a);

// Each queues its work on `stream` of the current device and returns.
hipError_t launch_rms_norm_mx(uint32_t type, const MxNormArgs& a, hipStream_t stream);
hipError_t launch_swiglu_mx(uint32_t type, const MxSwigluArgs& a, hipStream_t stream);
hipError_t launch_mxfp4_linear(uint32_t x_type, const MxLinearArgs& a, hipStream_t stream);
hipError_t launch_mxfp4_quantise(uint32_t type, const MxQuantiseArgs& a, hipStream_t stream);
hipError_t launch_mxfp4_matmul(const MxLinearArgs& a, hipStream_t stream);  // x: codes, stride in bytes, with x_scales
hipError_t launch_mxfp4_moe(const MxMoeArgs& a, hipStream_t stream);

}  // namespace ptwm
