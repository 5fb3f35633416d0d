// mx_choice.hip -- which kernel a product with MXFP4 weights takes
// (ptwm_amd/csrc/mx_choice.h), on the host.
#include "mx_choice.h"

using namespace ptwm;

// out: kind (0 small, 1 few tokens, 2 tiles), tokens, rows, ct, rg, kg, aligned.
extern "C" void mx_choice(uint32_t type, uint64_t tokens, uint32_t rows, uint32_t cols, uint64_t x, uint64_t x_stride,
                          uint64_t x_scales_stride, uint64_t weight, uint64_t weight_stride, uint64_t scales_stride,
                          uint32_t* out) {
  const MxLinearArgs a{{x, x_stride}, {1, x_scales_stride}, {weight, weight_stride}, {1, scales_stride}, {16, rows}, 0,
                       tokens, rows, cols, kTypeF32};
  const MxLinearChoice k = choose_mxfp4_linear(type, a);
  const uint32_t v[] = {k.kind, k.tokens, k.rows, k.ct, k.rg, k.kg, k.aligned};
  for (int i = 0; i < 7; ++i) out[i] = v[i];
}
