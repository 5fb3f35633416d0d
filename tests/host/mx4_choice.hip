// mx4_choice.hip -- which kernel a product of two MXFP4 matrices takes
// (ptwm_amd/csrc/mx_choice.h), on the host.
#include "mx_choice.h"

using namespace ptwm;

// x, x_scales, weight, scales: address and stride of each.  out: kind, dma.
extern "C" void mx4_choice(uint64_t tokens, uint32_t rows, uint32_t cols, const uint64_t* at, uint32_t* out) {
  const MxLinearArgs a{{at[0], at[1]}, {at[2], at[3]}, {at[4], at[5]}, {at[6], at[7]}, {16, rows}, 0,
                       tokens, rows, cols, kTypeF32};
  const MxMatmulChoice k = choose_mxfp4_matmul(a);
  out[0] = k.kind, out[1] = (uint32_t)k.dma;
}
