// mx_moe.hip -- a mixture-of-experts layer on MXFP4 experts for a few tokens.
//
//   logits[t, e] = sum_k x[t, k] * router[e, k] (+ router_bias[e])
//   p[t, .] = softmax over the top_k largest logits of token t
//   h[t, e] = silu(G_e x_t + g_e) * (U_e x_t + u_e)
//   out[t] = sum over the chosen e of p[t, e] * (D_e h[t, e] + d_e)
#include <hip/hip_runtime.h>

#include "mx_device.h"

namespace ptwm {
namespace {

constexpr uint32_t kTokens = 64;  // of a launch; longer calls run in several

// Where a launch's intermediate results lie in the workspace.
struct MoeParts {
  uint64_t logits;   // f64 [tokens][experts]
  uint64_t chosen;   // int32 [tokens][top_k], -1 where a chosen expert is masked
  uint64_t weights;  // f32 [tokens][top_k]
  uint64_t h;        // f32 [tokens * top_k][inner], the routing weight multiplied in
  uint64_t end;
};
MoeParts parts_of_workspace(const MxMoeArgs& a) {
  const uint64_t t = a.tokens < kTokens ? a.tokens : kTokens;
  const auto align = [](uint64_t n) { return (n + 255) / 256 * 256; };
  MoeParts p;
  p.logits = a.workspace;
  p.chosen = p.logits + align(t * a.experts * 8);
  p.weights = p.chosen + align(t * a.top_k * 4);
  p.h = p.weights + align(t * a.top_k * 4);
  p.end = p.h + align(t * a.top_k * a.inner * 4);
  return p;
}

struct MoeArgs {
  MxMoeArgs a;
  MoeParts p;
};

__device__ __forceinline__ void load8_as(uint32_t type, uint64_t base, uint64_t at, float (&v)[8]) {
  if (type == kTypeBf16)
    load8<kTypeBf16>(base + at * 2, v);
  else if (type == kTypeF16)
    load8<kTypeF16>(base + at * 2, v);
  else
    load8<kTypeF32>(base + at * 4, v);
}
__device__ __forceinline__ float load1_as(uint32_t type, uint64_t base, uint64_t at) {
  if (type == kTypeBf16) return load1<kTypeBf16>(base + at * 2);
  if (type == kTypeF16) return load1<kTypeF16>(base + at * 2);
  return load1<kTypeF32>(base + at * 4);
}
__device__ __forceinline__ float bias_of(const MxExperts& w, uint32_t type, uint32_t e, uint32_t n) {
  return w.bias ? load1_as(type, w.bias, e * w.bias_expert + n * w.bias_stride) : 0.0f;
}

// Logits in 64 bits: products are exact there, and which of two near experts is chosen does not depend on the order of
// the additions.  A wavefront a logit.
template <uint32_t T>
__global__ __launch_bounds__(256) void moe_logits_kernel(MoeArgs m) {
  const MxMoeArgs& a = m.a;
  const uint32_t lane = threadIdx.x & 63, at = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= a.tokens * a.experts) return;
  const uint32_t t = at / a.experts, e = at % a.experts;
  double sum = 0;
  for (uint32_t k = lane * 8; k < a.cols; k += 512) {
    float x[8], r[8];
    load8<T>(a.x.ptr + (t * a.x.stride + k) * type_bytes(T), x);
    load8_as(a.router_type, a.router.ptr, e * a.router.stride + k, r);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += (double)x[i] * (double)r[i];
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) sum += __shfl_xor(sum, d, 64);
  if (lane == 0) {
    if (a.router_bias) sum += (double)load1_as(a.router_type, a.router_bias, e);
    g_st<double>(m.p.logits + (uint64_t)at * 8, sum);
  }
}

// Logits as integers of the same order, from 1 on: NaN last, zeros alike.  0 is below all.
__device__ __forceinline__ uint64_t order_of(double v) {
  if (v != v) return ~0ull;
  const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.0);
  return b >> 63 ? ~b : b | 1ull << 63;
}

// A wavefront a token: top_k times the largest logit that is left, the lowest expert of equal ones.
__global__ __launch_bounds__(64) void moe_route_kernel(MoeArgs m) {
  const MxMoeArgs& a = m.a;
  const uint32_t lane = threadIdx.x, t = blockIdx.x;
  constexpr int N = kMoeMaxExperts / 64;
  uint64_t key[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const uint32_t e = j * 64 + lane;
    key[j] = e < a.experts ? order_of(g_ld<double>(m.p.logits + ((uint64_t)t * a.experts + e) * 8)) : 0;
  }
  uint32_t mine = 0;
  double logit = 0, top = 0;
  for (uint32_t k = 0; k < a.top_k; ++k) {
    uint64_t best = 0;
    uint32_t at = 0;
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (key[j] > best) best = key[j], at = j * 64 + lane;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
      const uint64_t other = __shfl_xor(best, d, 64);
      const uint32_t where = __shfl_xor(at, d, 64);
      if (other > best || (other == best && where < at)) best = other, at = where;
    }
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j * 64 + lane == at) key[j] = 0;
    const double l = g_ld<double>(m.p.logits + ((uint64_t)t * a.experts + at) * 8);
    if (k == 0) top = l;
    if (k == lane) mine = at, logit = l;
  }
  const bool in = lane < a.top_k;
  // an expert at minus infinity has no weight, not even among its like
  const bool masked = logit == -__builtin_inf();
  float w = in && !masked ? expf((float)(logit - top)) : 0.0f, sum = w;
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) sum += __shfl_xor(sum, d, 64);
  w = masked ? 0.0f : w / sum;
  if (!in) return;
  const uint64_t at = (uint64_t)t * a.top_k + lane;
  g_st<int32_t>(m.p.chosen + at * 4, masked ? -1 : (int32_t)mine);
  g_st<float>(m.p.weights + at * 4, w);
  if (a.experts_out) g_st<int32_t>(a.experts_out + at * 4, (int32_t)mine);
  if (a.weights_out) g_st<float>(a.weights_out + at * 4, w);
}

// 16 rows of one expert's gate and up products for its tokens, 16 at a time; four wavefronts take turns in steps of 128
// values and add up in LDS.
template <uint32_t T>
__global__ __launch_bounds__(256) void moe_inner_kernel(MoeArgs m) {
  const MxMoeArgs& a = m.a;
  __shared__ float part[2][4][16][17];
  __shared__ uint16_t pairs[kTokens];
  __shared__ uint32_t count;
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, i = lane & 15;
  const uint32_t tiles = (a.inner + 15) / 16, e = blockIdx.x / tiles, n0 = blockIdx.x % tiles * 16;
  if (wave == 0) {
    uint32_t n = 0;
    const uint32_t all = a.tokens * a.top_k;
    for (uint32_t at = 0; at < all; at += 64) {
      const bool is = at + lane < all && g_ld<int32_t>(m.p.chosen + (uint64_t)(at + lane) * 4) == (int32_t)e;
      const uint64_t mask = __ballot(is);
      if (is) pairs[n + __popcll(mask & ((1ull << lane) - 1))] = at + lane;
      n += __popcll(mask);
    }
    if (lane == 0) count = n;
  }
  __syncthreads();
  const uint32_t blocks = a.cols / kMxBlock, n = min(n0 + i, a.inner - 1);
  const uint64_t gw = a.gate.codes.ptr + e * a.gate.codes_expert + n * a.gate.codes.stride;
  const uint64_t gs = a.gate.scales.ptr + e * a.gate.scales_expert + n * a.gate.scales.stride;
  const uint64_t uw = a.up.codes.ptr + e * a.up.codes_expert + n * a.up.codes.stride;
  const uint64_t us = a.up.scales.ptr + e * a.up.scales_expert + n * a.up.scales.stride;
  for (uint32_t first = 0; first < count; first += 16) {
    const uint32_t t = pairs[min(first + i, count - 1)] / a.top_k;
    const uint64_t x = a.x.ptr + t * a.x.stride * type_bytes(T);
    f32x4 acc[2] = {};
    for (uint32_t k = wave * 4 + q; k < (blocks + 3) / 4 * 4; k += 16) {
      const bool in = k < blocks;
      u32x4 wv[2] = {};
      float sf[2] = {1.0f, 1.0f};
      if (in) {
        wv[0] = ld16(gw + (uint64_t)k * 16), wv[1] = ld16(uw + (uint64_t)k * 16);
        sf[0] = scale_f32(g_ld<uint8_t>(gs + k)), sf[1] = scale_f32(g_ld<uint8_t>(us + k));
      }
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        u32x4 p[parts_of(T)] = {};
        if (in) parts_of_raw<T>(load_raw8<T>(x + ((uint64_t)k * 32 + f * 8) * type_bytes(T)), 1.0f, p);
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int j = parts_of(T) - 1; j >= 0; --j) acc[r] = mfma(weights8(wv[r][f], sf[r]), p[j], acc[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int j = 0; j < 4; ++j) part[r][wave][i][q * 4 + j] = acc[r][j];
    __syncthreads();
    const uint32_t ot = threadIdx.x >> 4, on = threadIdx.x & 15;
    if (first + ot < count && n0 + on < a.inner) {
      float g = bias_of(a.gate, a.out_type, e, n0 + on), u = bias_of(a.up, a.out_type, e, n0 + on);
#pragma unroll
      for (int w = 0; w < 4; ++w) g += part[0][w][ot][on], u += part[1][w][ot][on];
      const uint32_t pair = pairs[first + ot];
      const float h = g / (1.0f + expf(-g)) * u * g_ld<float>(m.p.weights + (uint64_t)pair * 4);
      g_st<float>(m.p.h + ((uint64_t)pair * a.inner + n0 + on) * 4, h);
    }
    __syncthreads();
  }
}

// 16 output rows of 16 tokens: one expert after the other, its product added for the tokens that chose it (a column of
// zeros would take a broken scale to the others).
__global__ __launch_bounds__(256) void moe_outer_kernel(MoeArgs m) {
  const MxMoeArgs& a = m.a;
  __shared__ float part[4][16][17];
  __shared__ uint32_t used[kMoeMaxExperts / 32];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, i = lane & 15;
  const uint32_t tiles = (a.cols + 15) / 16, n0 = blockIdx.x % tiles * 16, t0 = blockIdx.x / tiles * 16;
  const uint32_t tokens = min((uint32_t)a.tokens - t0, 16u);
  if (threadIdx.x < kMoeMaxExperts / 32) used[threadIdx.x] = 0;
  __syncthreads();
  for (uint32_t p = threadIdx.x; p < tokens * a.top_k; p += 256) {
    const int32_t e = g_ld<int32_t>(m.p.chosen + ((uint64_t)t0 * a.top_k + p) * 4);
    if (e >= 0) atomicOr(&used[e / 32], 1u << (e & 31));
  }
  __syncthreads();
  const uint32_t blocks = a.inner / kMxBlock, n = min(n0 + i, a.cols - 1);
  f32x4 total = {};
  for (uint32_t e = 0; e < a.experts; ++e) {
    if (!(used[e / 32] >> (e & 31) & 1)) continue;
    uint32_t slot = ~0u;
    for (uint32_t k = 0; k < a.top_k && i < tokens; ++k)
      if (g_ld<int32_t>(m.p.chosen + ((uint64_t)(t0 + i) * a.top_k + k) * 4) == (int32_t)e) slot = k;
    const bool mine = slot != ~0u;
    const uint64_t pair = (uint64_t)(t0 + i) * a.top_k + slot;
    const uint64_t h = m.p.h + pair * a.inner * 4;
    const uint64_t w = a.down.codes.ptr + e * a.down.codes_expert + n * a.down.codes.stride;
    const uint64_t s = a.down.scales.ptr + e * a.down.scales_expert + n * a.down.scales.stride;
    f32x4 acc = {};
    for (uint32_t k = wave * 4 + q; k < (blocks + 3) / 4 * 4; k += 16) {
      const bool in = k < blocks;
      u32x4 wv = {};
      float sf = 1.0f;
      if (in) wv = ld16(w + (uint64_t)k * 16), sf = scale_f32(g_ld<uint8_t>(s + k));
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        u32x4 p[3] = {};
        if (in && mine) parts_of_raw<kTypeF32>(load_raw8<kTypeF32>(h + ((uint64_t)k * 32 + f * 8) * 4), 1.0f, p);
#pragma unroll
        for (int j = 2; j >= 0; --j) acc = mfma(weights8(wv[f], sf), p[j], acc);
      }
    }
    if (mine) {
      total += acc;
      if (wave == 0) {
        const float weight = g_ld<float>(m.p.weights + pair * 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) total[j] += weight * bias_of(a.down, a.out_type, e, min(n0 + q * 4 + j, a.cols - 1));
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) part[wave][i][q * 4 + j] = total[j];
  __syncthreads();
  const uint32_t ot = threadIdx.x >> 4, on = threadIdx.x & 15;
  if (ot < tokens && n0 + on < a.cols) {
    const float v = (part[0][ot][on] + part[1][ot][on]) + (part[2][ot][on] + part[3][ot][on]);
    const uint64_t at = (t0 + ot) * a.out.stride + n0 + on;
    if (a.out_type == kTypeBf16)
      store1<kTypeBf16>(a.out.ptr + at * 2, v);
    else if (a.out_type == kTypeF16)
      store1<kTypeF16>(a.out.ptr + at * 2, v);
    else
      store1<kTypeF32>(a.out.ptr + at * 4, v);
  }
}

template <uint32_t T>
hipError_t moe_of(const MxMoeArgs& a, hipStream_t stream) {
  return in_parts(a.tokens, kTokens, [&](uint64_t first, uint64_t tokens) {
    MoeArgs m{a, parts_of_workspace(a)};
    m.a.tokens = tokens;
    m.a.x = rows_from(a.x, first, type_bytes(T)), m.a.out = rows_from(a.out, first, type_bytes(a.out_type));
    if (a.experts_out) m.a.experts_out += first * a.top_k * 4;
    if (a.weights_out) m.a.weights_out += first * a.top_k * 4;
    hipError_t e = launch(moe_logits_kernel<T>, (tokens * a.experts + 3) / 4, 256, m, stream);
    if (e == hipSuccess) e = launch(moe_route_kernel, tokens, 64, m, stream);
    if (e == hipSuccess) e = launch(moe_inner_kernel<T>, (uint64_t)a.experts * ((a.inner + 15) / 16), 256, m, stream);
    if (e == hipSuccess) e = launch(moe_outer_kernel, (a.cols + 15) / 16 * ((tokens + 15) / 16), 256, m, stream);
    return e;
  });
}

}  // namespace

uint64_t mxfp4_moe_workspace(const MxMoeArgs& a) { return parts_of_workspace(a).end - a.workspace; }

hipError_t launch_mxfp4_moe(const MxMoeArgs& a, hipStream_t stream) {
  switch (a.x_type) {
    case kTypeF32: return moe_of<kTypeF32>(a, stream);
    case kTypeF16: return moe_of<kTypeF16>(a, stream);
    case kTypeBf16: return moe_of<kTypeBf16>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace ptwm
