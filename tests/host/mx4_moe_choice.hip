// mx4_moe_choice.hip -- how the products of a mixture-of-experts layer are made
// (ptwm_amd/csrc/mx_choice.h), on the host.
#include "mx_choice.h"

using namespace ptwm;

// sizes: tokens, experts, top_k, cols, inner, type of x.  at: of gate, up and down each the codes' address, stride and
// experts' stride, and the scales' stride.  out: inner, outer, inner_dma, outer_dma, routed, span, chunks.
extern "C" void mx4_moe_choice(const uint64_t* sizes, const uint64_t* at, uint32_t* out) {
  MxMoeArgs a{};
  a.tokens = sizes[0], a.experts = (uint32_t)sizes[1], a.top_k = (uint32_t)sizes[2];
  a.cols = (uint32_t)sizes[3], a.inner = (uint32_t)sizes[4], a.x_type = (uint32_t)sizes[5];
  MxExperts* const w[] = {&a.gate, &a.up, &a.down};
  for (int k = 0; k < 3; ++k) {
    w[k]->codes = {at[4 * k], at[4 * k + 1]}, w[k]->codes_expert = at[4 * k + 2];
    w[k]->scales = {16, at[4 * k + 3]};
  }
  const MxMoeChoice c = choose_mxfp4_moe(a);
  out[0] = c.inner, out[1] = c.outer, out[2] = c.inner_dma, out[3] = c.outer_dma, out[4] = c.routed;
  out[5] = c.span, out[6] = c.chunks;
}
