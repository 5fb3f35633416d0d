// mx_moe.hip -- a mixture-of-experts layer on MXFP4 experts for a few tokens.
//
//   logits[t, e] = sum_k x[t, k] * router[e, k] (+ router_bias[e])
//   p[t, .] = softmax over the top_k largest logits of token t
//   h[t, e] = silu(G_e x_t + g_e) * (U_e x_t + u_e)
//   out[t] = sum over the chosen e of p[t, e] * (D_e h[t, e] + d_e)
//
// What it cannot do without is the chosen experts' weights from memory, each
// once; all else is small.  The kernels:
//   logits   a workgroup an expert and four tokens; x as bf16 parts
//   route    the choice, a wavefront a token (few tokens: within the next one)
//   inner    gate and up products of an expert's tokens, h as bf16 parts
//   outer    the down products; of a few tokens, their weighted sums at once
//   combine  (many tokens) the weighted sums
// Inner and outer products are each one of two kernels: moe_product_kernel, a
// workgroup a few rows of an expert, whose columns go through LDS beside the
// weights, and moe_stream_kernel, a workgroup a compute unit for all of a
// launch, whose columns stay in registers.
//
// The products are of bf16 on the matrix unit.  Weights are widened to bf16,
// which is exact; x is the sum of one to three bf16 values (parts), h of three,
// each of which is a column of the product of its own, summed with its like at
// the end.  So an instruction's 16 columns are one to three columns a token,
// whatever the types, and few tokens in two parts cost no more than in one.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "mx_choice.h"
#include "mx_device.h"

namespace ptwm {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));

// Where a launch's intermediate results lie in the workspace.  A pair is a token's k-th expert, token * top_k + k.
struct MoePlaces {
  uint64_t logits;   // f64 [tokens][experts]
  uint64_t x;        // bf16 [parts][tokens][x_len]
  uint64_t h;        // bf16 [parts][pairs][h_len]
  uint64_t y;        // f32 [chunks][pairs][cols]
  uint64_t chosen;   // int32 [pairs], -1 where a chosen expert is masked
  uint64_t weights;  // f32 [pairs]
  uint64_t end;
  uint32_t x_len, h_len;  // cols and inner in whole steps, zeros past their ends
};
MoePlaces places_of(const MxMoeArgs& a) {
  const uint64_t t = a.tokens < kMoeTokens ? a.tokens : kMoeTokens, pairs = t * a.top_k;
  uint64_t at = a.workspace;
  const auto take = [&](uint64_t bytes) {
    const uint64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  MoePlaces p;
  p.x_len = (a.cols + kMoeStep - 1) / kMoeStep * kMoeStep, p.h_len = (a.inner + kMoeStep - 1) / kMoeStep * kMoeStep;
  p.logits = take(t * a.experts * 8);
  p.x = take(parts_of(a.x_type) * t * p.x_len * 2);
  p.h = take(kMoeInnerParts * pairs * p.h_len * 2);
  const uint64_t chunks = (p.h_len / kMoeStep + 7) / 8;
  p.y = take((chunks <= kMoeChunks ? chunks : 1) * pairs * a.cols * 4);
  p.chosen = take(pairs * 4), p.weights = take(pairs * 4);
  p.end = at;
  return p;
}

struct MoeArgs {
  MxMoeArgs a;
  MoePlaces p;
  uint32_t span, chunks;  // of moe_stream_kernel's rows: steps of a chunk, chunks
  bool routed;            // moe_route_kernel has run
};

// Where a row of x or h in the workspace has 16-byte chunk `c`: of a step's, the f-th of block b (of eight) lies at
// (b / 4 * 4 + f) * 4 + b % 4, so that what four lanes need for one product lies together.
__device__ __forceinline__ uint32_t chunk_at(uint32_t c) {
  return c / 16 * 16 + c % 4 * 4 + c / 4 % 4;
}

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
__device__ __forceinline__ void store1_as(uint32_t type, uint64_t base, uint64_t at, float v) {
  if (type == kTypeBf16)
    store1<kTypeBf16>(base + at * 2, v);
  else if (type == kTypeF16)
    store1<kTypeF16>(base + at * 2, v);
  else
    store1<kTypeF32>(base + at * 4, v);
}
// An expert's N biases from row n on, zeros without one.
template <int N>
__device__ __forceinline__ void biases_of(const MxExperts& w, uint32_t type, uint32_t e, uint32_t n, float (&b)[N]) {
  const uint64_t at = e * w.bias_expert + n * w.bias_stride;
  auto load = [&](auto t) {  // all on their way at once
#pragma unroll
    for (int j = 0; j < N; ++j) b[j] = load1<t>(w.bias + (at + j * w.bias_stride) * type_bytes(t));
  };
  if (!w.bias) {
#pragma unroll
    for (int j = 0; j < N; ++j) b[j] = 0.0f;
  } else if (type == kTypeBf16) {
    load(std::integral_constant<uint32_t, kTypeBf16>{});
  } else if (type == kTypeF16) {
    load(std::integral_constant<uint32_t, kTypeF16>{});
  } else {
    load(std::integral_constant<uint32_t, kTypeF32>{});
  }
}

// Outputs n .. n + 3 of token t.
__device__ __forceinline__ void store_out(const MxMoeArgs& a, uint64_t t, uint32_t n, f32x4 v) {
  const uint64_t to = t * a.out.stride + n;
  if (a.out_type == kTypeBf16)
    st8(a.out.ptr + to * 2, pack2<kTypeBf16>(v[0], v[1]) | (uint64_t)pack2<kTypeBf16>(v[2], v[3]) << 32);
  else if (a.out_type == kTypeF16)
    st8(a.out.ptr + to * 2, pack2<kTypeF16>(v[0], v[1]) | (uint64_t)pack2<kTypeF16>(v[2], v[3]) << 32);
  else
    st16(a.out.ptr + to * 4, __builtin_bit_cast(u32x4, v));
}

// silu(g) * u.  Below g = -64 the 1 is nothing beside exp(-g), which 32 bits do not hold from -88.8 on though its quotient
// with a large u may be a value: there four times exp(g / 4), the first one with g and u, each a number down to g = -349.
__device__ __forceinline__ float activated(float g, float u) {
  const bool deep = g < -64.0f;
  const float e = expf(deep ? 0.25f * g : -g);
  return deep ? g * e * u * e * e * e : g / (1.0f + e) * u;
}

// Two neighbours of a pair's h, the parts `apart` bytes apart: as x's; the last is exact too, down to 2^-133.
__device__ __forceinline__ void store_h(uint64_t to, uint64_t apart, f32x2 h) {
#pragma unroll
  for (uint32_t p = 0; p < kMoeInnerParts; ++p, to += apart) {
    uint32_t b;
    if (p + 1 < kMoeInnerParts) {
      const uint32_t low = f32_bits(__builtin_amdgcn_fmed3f(h[0], -kBf16Max, kBf16Max)) & 0xFFFF0000u;
      const uint32_t high = f32_bits(__builtin_amdgcn_fmed3f(h[1], -kBf16Max, kBf16Max)) & 0xFFFF0000u;
      h -= f32x2{bits_f32(low), bits_f32(high)};
      b = low >> 16 | high;
    } else {
      b = pack2<kTypeBf16>(h[0], h[1]);
    }
    st4(to, b);
  }
}

// The value that the lane K further on has, of 16.
template <int K>
__device__ __forceinline__ float right(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x100 + K, 0xF, 0xF, true));
}

// A wavefront's sum, in its last lane.
template <int CTRL, int ROWS>
__device__ __forceinline__ double plus_by(double v) {
  const u32x2 b = __builtin_bit_cast(u32x2, v);
  const u32x2 o = {(uint32_t)__builtin_amdgcn_update_dpp(0, (int)b[0], CTRL, ROWS, 0xF, false),
                   (uint32_t)__builtin_amdgcn_update_dpp(0, (int)b[1], CTRL, ROWS, 0xF, false)};
  return v + __builtin_bit_cast(double, o);
}
__device__ __forceinline__ double wave_sum(double v) {
  v = plus_by<0x111, 0xF>(v), v = plus_by<0x112, 0xF>(v), v = plus_by<0x114, 0xF>(v), v = plus_by<0x118, 0xF>(v);
  return plus_by<0x143, 0xC>(plus_by<0x142, 0xA>(v));
}

// Logits of one expert and four tokens: the threads take turns along the rows.  Summed in 64 bits, in which products
// are exact, so that which of two near experts is chosen does not depend on the order of the additions.  The
// workgroups after these write x's parts, and zeros past h's ends, a token each.  Bound by the launch
// and one trip to memory: 2.9 us for 128 experts of 2048, 1 token.
constexpr uint32_t kLogitTokens = 4;
constexpr uint32_t kLogitThreads = 512;
template <uint32_t T>
__global__ __launch_bounds__(kLogitThreads) void moe_logits_kernel(MoeArgs m) {
  const MxMoeArgs& a = m.a;
  __shared__ double part[kLogitTokens][kLogitThreads / 64];
  const uint32_t groups = ((uint32_t)a.tokens + kLogitTokens - 1) / kLogitTokens;
  if (blockIdx.x >= a.experts * groups) {
    const uint32_t t = blockIdx.x - a.experts * groups;
    for (uint32_t k = threadIdx.x * 8; k < m.p.x_len; k += kLogitThreads * 8) {
      u32x4 p[parts_of(T)] = {};
      if (k < a.cols) parts_of_raw<T>(load_raw8<T>(a.x.ptr + (t * a.x.stride + k) * type_bytes(T)), 1.0f, p);
#pragma unroll
      for (int j = 0; j < parts_of(T); ++j) st16(m.p.x + (j * a.tokens + t) * m.p.x_len * 2 + chunk_at(k / 8) * 16, p[j]);
    }
    const uint32_t none = (m.p.h_len - a.inner) / 8, rows = a.top_k * kMoeInnerParts;  // chunks of a row
    for (uint32_t j = threadIdx.x; j < none * rows; j += kLogitThreads) {
      const uint32_t row = j / none, part = row / a.top_k, pair = t * a.top_k + row % a.top_k;
      st16(m.p.h + (part * a.tokens * a.top_k + pair) * m.p.h_len * 2 + chunk_at(a.inner / 8 + j % none) * 16, u32x4{});
    }
    return;
  }
  const uint32_t e = blockIdx.x / groups, t0 = blockIdx.x % groups * kLogitTokens;
  double sum[kLogitTokens] = {};
  for (uint32_t k = threadIdx.x * 8; k < a.cols; k += kLogitThreads * 8) {
    float r[8], x[kLogitTokens][8];
    load8_as(a.router_type, a.router.ptr, e * a.router.stride + k, r);
#pragma unroll
    for (uint32_t t = 0; t < kLogitTokens; ++t)
      if (t0 + t < a.tokens) load8<T>(a.x.ptr + ((t0 + t) * a.x.stride + k) * type_bytes(T), x[t]);
#pragma unroll
    for (uint32_t t = 0; t < kLogitTokens; ++t)
      if (t0 + t < a.tokens)
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[t] = __builtin_fma((double)x[t][i], (double)r[i], sum[t]);
  }
  const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
  for (uint32_t t = 0; t < kLogitTokens; ++t) {
    sum[t] = wave_sum(sum[t]);
    if (lane == 63) part[t][wave] = sum[t];
  }
  __syncthreads();
  const uint32_t t = threadIdx.x;
  if (t >= kLogitTokens || t0 + t >= a.tokens) return;
  double v = part[t][0];
#pragma unroll
  for (uint32_t k = 1; k < kLogitThreads / 64; ++k) v += part[t][k];
  if (a.router_bias) v += (double)load1_as(a.router_type, a.router_bias, e);
  g_st<double>(m.p.logits + ((uint64_t)(t0 + t) * a.experts + e) * 8, v);
}

// Logits as integers of the same order, from 1 on: NaN last, zeros alike.  0 is below all.
__device__ __forceinline__ uint64_t order_of(double v) {
  if (v != v) return ~0ull;
  const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.0);
  return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double logit_of(uint64_t order) {
  return __builtin_bit_cast(double, order >> 63 ? order ^ 1ull << 63 : ~order);
}

// The largest of a wavefront's values, in all lanes.  By DPP: eight choices of 128 experts through LDS took 2 us more.
template <int CTRL>
__device__ __forceinline__ uint32_t larger_by(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = larger_by<0x111>(v), v = larger_by<0x112>(v), v = larger_by<0x114>(v), v = larger_by<0x118>(v);  // in rows of 16
  v = larger_by<0x142>(v), v = larger_by<0x143>(v);  // a row's last lane to the next rows
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// The sum of a lane's and the lower lanes' values.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t plus_by(uint32_t v) {
  return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ uint32_t wave_up_to(uint32_t v) {
  v = plus_by<0x111, 0xF>(v), v = plus_by<0x112, 0xF>(v), v = plus_by<0x114, 0xF>(v), v = plus_by<0x118, 0xF>(v);
  return plus_by<0x143, 0xC>(plus_by<0x142, 0xA>(v));
}

// Chooses a token's experts: the largest that is left, the lowest expert of equal ones.  One wavefront, N logits a
// lane; lane k returns the k-th, with its weight.  An expert at minus infinity has none, not even among its like.
struct Chosen {
  int32_t expert;  // -1 where masked
  float weight;
  int32_t reported;
};
template <uint32_t N>
__device__ __forceinline__ Chosen choose_of(const MoeArgs& m, uint32_t t) {
  const uint32_t lane = threadIdx.x & 63;
  uint64_t key[N];
#pragma unroll
  for (uint32_t j = 0; j < N; ++j) {
    const uint32_t e = j * 64 + lane;
    key[j] = e < m.a.experts ? order_of(g_ld<double>(m.p.logits + ((uint64_t)t * m.a.experts + e) * 8)) : 0;
  }
  Chosen mine{0, 0, 0};
  uint64_t own = 0, top = 0;
  for (uint32_t k = 0; k < m.a.top_k; ++k) {
    uint64_t most = key[0];
#pragma unroll
    for (uint32_t j = 1; j < N; ++j) most = key[j] > most ? key[j] : most;
    // by the upper halves, and by the lower ones where several lanes have the same
    const uint32_t upper = (uint32_t)(most >> 32), high = wave_max(upper);
    uint64_t at = __ballot(upper == high);
    uint32_t owner = (uint32_t)__ffsll((long long)at) - 1;
    uint32_t low = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)most, (int)owner);
    if (at & (at - 1)) {
      low = wave_max(upper == high ? (uint32_t)most : 0);
      at = __ballot(upper == high && (uint32_t)most == low);
    }
    const uint64_t best = low | (uint64_t)high << 32;
    uint32_t j0 = 0;  // the lane's first with that logit
#pragma unroll
    for (uint32_t j = N; j-- > 0;)
      if (key[j] == best) j0 = j;
    if (at & (at - 1)) {  // of several lanes the one whose expert is the lowest
#pragma unroll
      for (uint32_t j = N; j-- > 0;)
        if (const uint64_t with = __ballot(key[j] == best)) at = with;
    }
    owner = (uint32_t)__ffsll((long long)at) - 1;
    const uint32_t first = (uint32_t)__builtin_amdgcn_readlane((int)j0, (int)owner), e = first * 64 + owner;
#pragma unroll
    for (uint32_t j = 0; j < N; ++j)
      if (lane == owner && j == first) key[j] = 0;
    if (k == 0) top = best;
    if (k == lane) mine.reported = (int32_t)e, own = best;
  }
  const bool in = lane < m.a.top_k;
  const double logit = logit_of(own);
  const bool masked = logit == -__builtin_inf();
  const float w = in && !masked ? expf((float)(logit - logit_of(top))) : 0.0f;
  float sum = w;
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) sum += __shfl_xor(sum, d, 64);
  mine.weight = masked ? 0.0f : w / sum;
  mine.expert = masked ? -1 : mine.reported;
  return mine;
}
__device__ __forceinline__ Chosen choose(const MoeArgs& m, uint32_t t) {
  if (m.a.experts <= 64) return choose_of<1>(m, t);
  if (m.a.experts <= 128) return choose_of<2>(m, t);
  return choose_of<kMoeMaxExperts / 64>(m, t);
}
__device__ __forceinline__ void store_choice(const MoeArgs& m, uint32_t t, const Chosen& c) {
  const uint32_t lane = threadIdx.x & 63;
  if (lane >= m.a.top_k) return;
  const uint64_t at = (uint64_t)t * m.a.top_k + lane;
  g_st<int32_t>(m.p.chosen + at * 4, c.expert);
  g_st<float>(m.p.weights + at * 4, c.weight);
  if (m.a.experts_out) g_st<int32_t>(m.a.experts_out + at * 4, c.reported);
  if (m.a.weights_out) g_st<float>(m.a.weights_out + at * 4, c.weight);
}

__global__ __launch_bounds__(64) void moe_route_kernel(MoeArgs m) { store_choice(m, blockIdx.x, choose(m, blockIdx.x)); }

// Rows of one expert's products for its tokens (or, ALL, of the outer products
// of all experts of up to 64 pairs, weighted and added up).  WR wavefronts hold
// 16 rows each, of gate and up (INNER) or of down, and share the XC columns; KG
// groups of them take turns in steps of 256 values along the rows and add up in
// LDS at the end.
//
// Codes, scales and columns go through LDS by DMA, NS - 1 steps ahead: the
// matrix instruction's order, a row a lane, would cost the address unit a cycle
// a lane, and the requests need no registers.  A wavefront's codes and scales
// are its own; the columns of a group are loaded by all of it.  16-byte chunks
// of a row of codes (8) or of a column (32) lie at chunk ^ (row / 2 % 8) and
// chunk ^ (column % 16), so that the 16 lanes that read together meet every bank
// once.  In a product lane l takes block l / 16 of row (column) l % 16, values
// 8f .. 8f+7 with product f of four.
//
// A step's eight scales of a row lie at any byte, within three words, of which
// those come that hold one of the row's own; four lanes a row.  kDma: codes lie
// at multiples of 16 bytes; else they go through registers.
//
// Memory's latency bounds it: a workgroup ends after 1 to 56 steps at the
// measured sizes (512 at most, and that of each where it walks along several
// experts), of which NS - 1 are on their way, and the chip's bytes on their way
// are what its workgroups have.  8 experts of 4096x14336, 1 token: inner 27 us
// (125 MB, 4.6 TB/s), outer 15 us (62 MB, 4.2 TB/s).  Three stages of the inner
// products, two workgroups a compute unit instead of three, 30.6 us.
template <bool INNER, bool ALL, int WR, int KG, int XC, int NS, bool kDma>
__global__ __launch_bounds__(64 * WR * KG) void moe_product_kernel(MoeArgs m) {
  static_assert(WR == 1 || KG == 1, "groups of several wavefronts meet at barriers of the whole workgroup");
  static_assert(!(INNER && ALL) && XC <= 16, "a product has 16 columns");
  constexpr int M = INNER ? 2 : 1;  // matrices
  constexpr uint32_t G = 64 * WR, kWaves = WR * KG, kRows = 16 * WR;
  constexpr uint32_t kCodes = M * 128, kColumns = XC * 32;  // chunks of a stage
  constexpr int JW = kCodes / 64, JX = kColumns / G, JS = M;
  constexpr int N = JX + (kDma ? JW : 0) + JS;  // requests of a step
  constexpr uint32_t kScales = JS * 64;                                          // words of a stage
  static_assert(kColumns % G == 0 && (NS - 2) * N < 64, "whole requests, and a wait that counts them");
  __shared__ u32x4 columns[KG * NS * kColumns], codes[KG * WR * NS * kCodes];
  __shared__ u32x4 scales[KG * WR * NS * kScales / 4];
  __shared__ int32_t list[64], table[ALL ? 64 * XC : 1], fused[INNER ? kMoeFusedPairs : 1];
  __shared__ float weights[ALL ? 64 : 1];
  const MxMoeArgs& a = m.a;
  const uint32_t lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
  const uint64_t below = (1ull << lane) - 1;  // lanes
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t group = wave / WR, wr = wave % WR, gi = wr * 64 + lane;
  const uint32_t rows = INNER ? a.inner : a.cols, length = INNER ? a.cols : a.inner, blocks = length / kMxBlock;
  const uint32_t x_len = INNER ? m.p.x_len : m.p.h_len, steps = x_len / kMoeStep;
  const uint32_t tiles = (rows + kRows - 1) / kRows;
  const uint32_t slot = blockIdx.x / tiles, n0 = blockIdx.x % tiles * kRows;
  const uint32_t parts = INNER ? parts_of(a.x_type) : kMoeInnerParts, each = XC / parts;  // tokens of XC columns
  const uint32_t pairs = (uint32_t)a.tokens * a.top_k;

  // The expert and the pairs that chose it (every wavefront writes the same to LDS); ALL: the experts that any pair
  // chose, lane k holding the k-th, and for each the pairs of the tokens, -1 without one.
  uint32_t e0 = 0, count = (uint32_t)a.tokens, experts = 0;
  int32_t expert_k = 0;
  if constexpr (ALL) {
    const bool in = lane < pairs;
    const int32_t e = in ? g_ld<int32_t>(m.p.chosen + lane * 4) : -1;
    if (in) weights[lane] = g_ld<float>(m.p.weights + lane * 4);
    uint32_t leader = lane;  // the first pair of the same expert
    if (a.tokens > 1) {
      for (uint32_t p = pairs; p-- > 0;)
        if (__builtin_amdgcn_readlane(e, (int)p) == e && p < leader) leader = p;
    }
    const uint64_t leaders = __ballot(e >= 0 && leader == lane);
    experts = __popcll(leaders);
    for (uint32_t k = lane; k < experts * XC; k += 64) table[k] = -1;
    if (e >= 0) {
      const uint32_t k = __popcll(leaders & ((1ull << leader) - 1));
      table[k * XC + lane / a.top_k] = (int32_t)lane;
      if (leader == lane) list[k] = e;
    }
    __syncthreads();
    if (lane < experts) expert_k = list[lane];
  } else {
    const bool choosing = INNER && !m.routed;
    if (choosing) {
      for (uint32_t t = wave; t < a.tokens; t += kWaves) {
        const Chosen c = choose(m, t);
        if (lane < a.top_k) fused[INNER ? t * a.top_k + lane : 0] = c.expert;
        if (blockIdx.x == 0) store_choice(m, t, c);
      }
      __syncthreads();
    }
    auto expert_of = [&](uint32_t p) { return choosing ? fused[INNER ? p : 0] : g_ld<int32_t>(m.p.chosen + p * 4); };
    // a workgroup an expert, or a pair where there are fewer: the first one of an expert's serves all
    const bool by_pair = pairs < a.experts;
    const int32_t e = by_pair ? __builtin_amdgcn_readfirstlane(expert_of(slot)) : (int32_t)slot;
    if (e < 0) return;
    count = 0;
    for (uint32_t p = 0; p < pairs; p += 64) {
      const bool is = p + lane < pairs && expert_of(p + lane) == e;
      const uint64_t mask = __ballot(is);
      if (is) list[count + __popcll(mask & below)] = (int32_t)(p + lane);
      count += __popcll(mask);
    }
    if (count == 0 || (by_pair && list[0] != (int32_t)slot)) return;
    e0 = (uint32_t)e;
  }
  const uint32_t units = ALL ? experts * steps : steps;

  // Rows past the last one take its place; their sums are not stored, or as zeros.
  uint64_t w_at[JW], s_at[JS];  // codes and scales
  auto matrix = [&](int r) -> const MxExperts& { return INNER ? (r ? a.up : a.gate) : a.down; };
  auto row_of = [&](uint32_t in) { return min(n0 + wr * 16 + in, rows - 1); };
  auto scales_of = [&](int r, uint32_t n) {
    const MxExperts& w = matrix(r);
    return w.scales.ptr + e0 * w.scales_expert + n * w.scales.stride;
  };
#pragma unroll
  for (int j = 0; j < JW; ++j) {
    const MxExperts& w = matrix(j / 2);
    w_at[j] = w.codes.ptr + e0 * w.codes_expert + row_of(j % 2 * 8 + lane / 8) * w.codes.stride;
  }
  uint32_t shift[M];  // bytes from a word to the scales of row i, the expert's aside
#pragma unroll
  for (int j = 0; j < JS; ++j) s_at[j] = scales_of(j, row_of(lane / 4)), shift[j] = (uint32_t)scales_of(j, row_of(i));
  const uint32_t columns_at = lds_address(columns) + group * (NS * kColumns * 16);
  const uint32_t codes_at = lds_address(codes) + wave * (NS * kCodes * 16);
  const uint32_t scales_at = lds_address(scales) + wave * (NS * kScales * 4);

  for (uint32_t t0 = 0; t0 < count; t0 += each) {
    const uint32_t tokens = min(count - t0, each);
    // A lane's chunks of the columns, as offsets: column c holds part c % parts of a token; columns without one repeat
    // the first.  (2^31 bytes hold 3 parts of 2048 pairs of the longest rows.)
    uint32_t x_at[JX], x_token[ALL ? JX : 1];
#pragma unroll
    for (int j = 0; j < JX; ++j) {
      const uint32_t column = (j * G + gi) / 32;
      uint32_t t = column / parts, part = column % parts;
      if (t >= tokens) t = 0, part = 0;
      const uint32_t chunk = (gi & 31) ^ (column & 15);
      uint32_t row = part * pairs;
      if constexpr (ALL) {
        x_token[j] = t;
      } else {
        const uint32_t pair = (uint32_t)list[t0 + t];
        row = INNER ? part * (uint32_t)a.tokens + pair / a.top_k : part * pairs + pair;
      }
      x_at[j] = row * x_len * 2 + chunk * 16;
    }
    const GlobalBytes x0 = global_bytes(INNER ? m.p.x : m.p.h);
    // Where along its way a group is: a step, of the k-th expert.
    struct Unit {
      uint32_t step, k;
    };
    auto forward = [&](Unit& u) {
      u.step += KG;
      while (ALL && u.step >= steps) u.step -= steps, ++u.k;
    };
    auto expert_of = [&](const Unit& u) { return (uint64_t)(uint32_t)__builtin_amdgcn_readlane(expert_k, (int)u.k); };
    auto request = [&](const Unit& u, uint32_t stage) {
      const uint64_t e = ALL ? expert_of(u) : 0;
#pragma unroll
      for (int j = 0; j < JW; ++j) {
        const uint32_t chunk = (lane & 7) ^ (j * 4 + (lane >> 4) & 7);
        const uint64_t from = w_at[j] + e * a.down.codes_expert + min(u.step * 8 + chunk, blocks - 1) * 16;
        if constexpr (kDma)
          dma16_once(from, codes_at + (stage * kCodes + j * 64) * 16);
        else
          ((LdsChunks)(codes_at + (stage * kCodes + lane) * 16))[j * 64] = ld16(from);
      }
      const uint32_t last = min(blocks - 1 - u.step * 8, 7u);  // block of the step
#pragma unroll
      for (int j = 0; j < JS; ++j) {
        const uint64_t from = s_at[j] + e * a.down.scales_expert + u.step * 8;
        dma4(from / 4 * 4 + min(lane % 4, ((uint32_t)from % 4 + last) / 4) * 4,
             scales_at + (stage * kScales + j * 64) * 4);
      }
#pragma unroll
      for (int j = 0; j < JX; ++j) {
        uint32_t from = x_at[j] + u.step * (kMoeStep * 2);
        if constexpr (ALL) {
          // a token that did not choose the expert has another's h here, whose sums are left out
          const int32_t pair = table[u.k * XC + x_token[j]];
          from += (uint32_t)max(pair, 0) * x_len * 2;
        }
        dma16(x0, from, columns_at + (stage * kColumns + j * G + wr * 64) * 16);
      }
    };
    f32x4 acc[M] = {}, total = {};
    auto compute = [&](const Unit& now, uint32_t stage) {
      const uint32_t last = min(blocks - 1 - now.step * 8, 7u);
      const uint32_t expert = ALL ? (uint32_t)(expert_of(now) * a.down.scales_expert) : 0;
      u32x4 wv[2][M];
      float sf[2][M];
#pragma unroll
      for (int r = 0; r < M; ++r) {
        const u32x4 words = *(LdsChunks)(scales_at + (stage * kScales + (r * 16 + i) * 4) * 4);
        const uint32_t low = __builtin_amdgcn_alignbyte(words[1], words[0], (shift[r] + expert) % 4);
        const uint32_t high = __builtin_amdgcn_alignbyte(words[2], words[1], (shift[r] + expert) % 4);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const uint32_t row = r * 16 + i, c = s * 4 + q;
          wv[s][r] = *(LdsChunks)(codes_at + (stage * kCodes + row * 8 + (c ^ (row / 2 & 7))) * 16);
          // blocks past the row's end have the last one's
          sf[s][r] = scale_f32(__builtin_amdgcn_perm(high, low, min(c, last) | 0x0C0C0C00));
        }
      }
      const uint32_t column = i % XC;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const u32x4 xv = *(LdsChunks)(columns_at + (stage * kColumns + column * 32 + ((u * 4 + q) ^ column)) * 16);
#pragma unroll
        for (int r = 0; r < M; ++r) acc[r] = mfma(weights8(wv[u / 4][r][u % 4], sf[u / 4][r]), xv, acc[r]);
      }
    };
    auto add_expert = [&](uint32_t k) {  // an expert's sums, weighted, for the tokens that chose it
      const uint32_t c = i % XC, t = c / parts;
      const int32_t pair = t < tokens ? table[ALL ? k * XC + t : 0] : -1;
      const f32x4 more = total + weights[ALL ? max(pair, 0) : 0] * acc[0];
      total = pair >= 0 ? more : total;
      acc[0] = f32x4{};
    };
    const uint32_t n = group < units ? (units - group + KG - 1) / KG : 0;  // of this group
    if (t0) __syncthreads();  // before LDS is used again
    if (n) {
      Unit now{group, 0};
      while (ALL && now.step >= steps) now.step -= steps, ++now.k;
      Unit ahead = now;  // the next one to be requested
#pragma unroll
      for (uint32_t k = 0; k < NS - 1; ++k) {
        request(ahead, k);
        if (k + 1 < n) forward(ahead);
      }
      uint32_t stage = 0, into = NS - 1;
      for (uint32_t k = 0; k < n; ++k) {
        if (k + NS - 2 < n)
          asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NS - 2) * N) : "memory");
        else
          asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        if constexpr (WR > 1)
          __builtin_amdgcn_s_barrier();
        else
          __builtin_amdgcn_wave_barrier();
        asm volatile("" ::: "memory");
        Unit next = now;
        forward(next);
        if (k + NS - 1 < n) {
          request(ahead, into);
          if (k + NS < n) forward(ahead);
        }
        compute(now, stage);
        if constexpr (ALL) {
          if (k + 1 == n || next.k != now.k) add_expert(now.k);
        }
        now = next;
        stage = stage + 1 == NS ? 0 : stage + 1, into = into + 1 == NS ? 0 : into + 1;
      }
    }
    // Sums to LDS, in place of the codes: 16 rows and 16 columns at a time, lane l rows 4 (l / 16) .. + 3 of column l % 16.
    __syncthreads();
    f32x4* const sums = reinterpret_cast<f32x4*>(codes);
    static_assert(M * 64 <= NS * kCodes, "a wavefront's sums fit its codes");
#pragma unroll
    for (int r = 0; r < M; ++r) sums[(wave * M + r) * 64 + lane] = ALL ? total : acc[r];
    __syncthreads();
    // of matrix r, rows 4 `quad` .. + 3 of wavefront w of a group, token t: over its parts and the groups
    auto sum_of = [&](uint32_t w, uint32_t r, uint32_t quad, uint32_t t) {
      f32x4 v = {};
#pragma unroll
      for (uint32_t g = 0; g < KG; ++g)
        for (uint32_t p = 0; p < parts; ++p) v += sums[((g * WR + w) * M + r) * 64 + quad * 16 + t * parts + p];
      return v;
    };
    for (uint32_t at = threadIdx.x; at < tokens * kRows / 4; at += 64 * kWaves) {
      const uint32_t t = at / (kRows / 4), in = at % (kRows / 4), w = in / 4, n = n0 + in * 4;
      const uint64_t pair = ALL ? 0 : (uint32_t)list[t0 + t];
      if constexpr (INNER) {
        if (n >= rows) continue;
        float gb[4], ub[4];
        biases_of(a.gate, a.out_type, e0, n, gb), biases_of(a.up, a.out_type, e0, n, ub);
        const f32x4 g = sum_of(w, 0, in % 4, t), u = sum_of(w, 1, in % 4, t);
        f32x4 h;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) h[j] = activated(g[j] + gb[j], u[j] + ub[j]);
        const uint64_t to = m.p.h + pair * m.p.h_len * 2 + chunk_at(n / 8) * 16 + n % 8 * 2;
        const uint64_t apart = pairs * (uint64_t)m.p.h_len * 2;
        store_h(to, apart, f32x2{h[0], h[1]}), store_h(to + 4, apart, f32x2{h[2], h[3]});
      } else if (n < rows) {
        f32x4 v = sum_of(w, 0, in % 4, t);
        if constexpr (ALL) {
          for (uint32_t k = 0; a.down.bias && k < experts; ++k) {
            const int32_t pair = table[k * XC + t];
            float bias[4];
            biases_of(a.down, a.out_type, (uint32_t)list[k], n, bias);
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j)
              if (pair >= 0) v[j] += weights[pair] * bias[j];
          }
          store_out(a, t, n, v);
        } else {
          st16(m.p.y + (pair * rows + n) * 4, __builtin_bit_cast(u32x4, v));
        }
      }
    }
  }
}

// The same products where an expert has several tokens and its codes lie at multiples of 16 bytes: the columns stay in
// registers.  A workgroup walks along consecutive tiles (16 rows of gate and of up, or 32 of down), of one expert after
// the other; of a tile's rows wavefront w of eight has steps w, w + 8, ... of a chunk of the rows, S at most, and keeps
// the values of 16 * NC columns there.  So LDS is for the weights, NS steps of each wavefront on their way, across the
// ends of tiles and of experts.  A tile's sums are added up over the wavefronts through LDS, read before the next tile's
// products and stored after them.  INNER: sums of whole rows; else of a chunk of them, which the combining kernel adds.
//
// 8 experts of 4096x14336, 64 tokens: inner 97 us (499 MB, 5.1 TB/s: memory), outer 86 us (250 MB, 2.9 TB/s; 44 without
// products and sums: a tile's 16 products a wavefront and 16 columns, its two barriers and the sums' way through LDS
// take longer than its bytes, and experts of more than 20 tokens go by twice).  With h in two parts, 69; so with columns
// through LDS they took 120 and 101, and weights that stayed in L2 as others do (no "once") 114 and 75: lines of h and
// y, of which a tile writes 32 or 64 bytes, left L2 in pieces.
constexpr uint32_t kStreamGroups = kMoeUnits;
constexpr uint32_t kStreamSlots = 16;    // experts of a workgroup, see below
// What a tile costs beside its groups of columns, in the like of one: 64 tokens' outer products took 74 us by equal tiles
// and 70, 69, 68.7 with 8, 6, 2 (h in two parts); the call with three takes 197, 197, 196, 195 with 9, 6, 4, 2.
constexpr uint32_t kInnerWeight = 8, kOuterWeight = 2;

template <bool INNER, int S, int NC>
__global__ __launch_bounds__(512) void moe_stream_kernel(MoeArgs m) {
  constexpr int M = 2, U = M * S, NS = S == 4 ? 7 : S == 2 ? 6 : 5, D = NS % U;  // steps of a tile, on their way
  constexpr uint32_t kCodes = 128, kWords = 64, N = 3;  // chunks and words of a step, its requests
  constexpr uint32_t kBiasTiles = 16;                   // whose biases are held at a time
  __shared__ u32x4 codes[8 * NS * kCodes];
  __shared__ uint32_t scales[8 * NS * kWords];
  __shared__ f32x2 sums[8 * M * NC * 128];
  __shared__ int16_t chosen[kMoeTokens * kMoeMaxTopK];
  __shared__ u32x4 none[8];
  __shared__ uint32_t slots[kStreamSlots], share[4];
  __shared__ int32_t list[kMoeTokens];
  __shared__ float biases[M][INNER ? kBiasTiles * 16 : 1];
  const MxMoeArgs& a = m.a;
  const uint32_t lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t rows = INNER ? a.inner : a.cols, length = INNER ? a.cols : a.inner, tiles = rows / (INNER ? 16 : 32);
  const uint32_t x_len = INNER ? m.p.x_len : m.p.h_len, steps = x_len / kMoeStep;
  const uint32_t span = m.span, chunks = m.chunks;
  const uint32_t parts = INNER ? parts_of(a.x_type) : kMoeInnerParts, each = 16 / parts, most = each * NC;
  const uint32_t pairs = (uint32_t)a.tokens * a.top_k;
  // A slot is an expert's up to `most` tokens; a tile of it weighs kTileWeight + its groups of columns, and every
  // workgroup has an equal share of that.  There are at most 2048 / 5 + 1024 slots (three parts, one group of columns),
  // and one weighs twice another at most, so no share meets more than thirteen.
  constexpr uint32_t kTileWeight = INNER ? kInnerWeight : kOuterWeight;
  {
    uint32_t* const counts = reinterpret_cast<uint32_t*>(sums);
    static_assert(sizeof(sums) >= kMoeMaxExperts * 4);
    for (uint32_t e = threadIdx.x; e < a.experts; e += 512) counts[e] = 0;
    __syncthreads();
    const auto count = [&](uint32_t p, int32_t e) {
      chosen[p] = (int16_t)e;
      if (e >= 0) atomicAdd(&counts[e], 1u);
    };
    if (!INNER || m.routed) {
      for (uint32_t p = threadIdx.x; p < pairs; p += 512) count(p, g_ld<int32_t>(m.p.chosen + p * 4));
    } else {
      for (uint32_t t = wave; t < a.tokens; t += 8) {
        const Chosen c = choose(m, t);
        if (lane < a.top_k) count(t * a.top_k + lane, c.expert);
        if (blockIdx.x == 0) store_choice(m, t, c);
      }
    }
    __syncthreads();
    if (wave == 0) {
      const uint32_t of_slot = chunks * tiles;
      // for 64 experts at a time, one a lane: its slots, their weight (of a tile each), and both with the ones before
      uint32_t all = 0, weight = 0, n = 0, own = 0, n_to = 0, to = 0;
      const auto each_slot = [&](auto f) {
        all = weight = 0;
        for (uint32_t e = lane; e - lane < a.experts; e += 64) {
          const uint32_t count = e < a.experts ? counts[e] : 0;
          n = (count + most - 1) / most;
          own = n ? n * (kTileWeight + NC) - (n * most - count) / each : 0;
          n_to = wave_up_to(n), to = wave_up_to(own);
          for (uint32_t j = 0; j < n; ++j)
            f(e, j, all + n_to - n + j, weight + to - own + j * (kTileWeight + NC),
              j + 1 < n ? kTileWeight + NC : own - j * (kTileWeight + NC));
          all += (uint32_t)__builtin_amdgcn_readlane((int)n_to, 63);
          weight += (uint32_t)__builtin_amdgcn_readlane((int)to, 63);
        }
      };
      each_slot([](uint32_t, uint32_t, uint32_t, uint32_t, uint32_t) {});
      const uint64_t total = (uint64_t)weight * of_slot;
      const uint64_t first = total * blockIdx.x / kStreamGroups, end = total * (blockIdx.x + 1) / kStreamGroups;
      if (lane < 4) share[lane] = lane % 2 ? 0 : all;
      each_slot([&](uint32_t, uint32_t, uint32_t slot, uint32_t before, uint32_t w) {
        const uint64_t from = (uint64_t)before * of_slot, past = from + (uint64_t)w * of_slot;
        if (first >= from && first < past) share[0] = slot, share[1] = (uint32_t)(first - from) / w;
        if (end >= from && end < past) share[2] = slot, share[3] = (uint32_t)(end - from) / w;
      });
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      const uint32_t slot0 = share[0];
      each_slot([&](uint32_t e, uint32_t j, uint32_t slot, uint32_t, uint32_t) {
        if (slot - slot0 < kStreamSlots) slots[slot - slot0] = e | j << 16;
      });
    }
    __syncthreads();
  }
  auto scalar = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); };
  uint32_t left = scalar((share[2] - share[0]) * (chunks * tiles) + share[3] - share[1]), slot = 0;
  uint32_t chunk = scalar(share[1]) / tiles, tile = scalar(share[1]) % tiles;
  if (left == 0) return;
  auto steps_of = [&](uint32_t chunk) {  // of this wavefront
    const uint32_t have = min(span, steps - chunk * span);
    return wave < have ? (have - wave + 7) / 8 : 0;
  };

  auto part_of = [&](uint32_t chunk, uint32_t n) {  // which of n steps is only part of one
    return length % kMoeStep && chunk * span + wave + (n - 1) * 8 == steps - 1 ? n - 1 : ~0u;
  };
  // The tile to be requested next: of it `n` steps, `run` tiles to the end of the expert's or the chunk's, `left` to the
  // end of all.  Rows come by 32, so all of a tile's are there.
  struct {
    uint32_t left, run, slot, chunk, tile, n, part;
    uint64_t codes[M], scales[M];  // the first row, at the wavefront's first step; scales at words
  } next{left, 0, 0, chunk, tile, 0, 0, {}, {}};
  // A lane's chunks and word from there, in a whole step and in the part of one that a row may end with, where the last
  // chunk is read over again.  A step's eight scales are at any byte, within three words, of which only those are read
  // that hold one of the row's own.
  uint32_t from[2][2], word[M][2];
  const uint32_t last = (length - 1) / kMxBlock % 8;  // block of the last step
  auto enter = [&] {
    const uint32_t e = scalar(slots[next.slot]) & 0xFFFF, step = next.chunk * span + wave;
    next.run = min(tiles - next.tile, next.left), next.n = steps_of(next.chunk);
    next.part = part_of(next.chunk, next.n);
#pragma unroll
    for (int r = 0; r < M; ++r) {
      const MxExperts& w = INNER ? (r ? a.up : a.gate) : a.down;
      const uint64_t n = INNER ? next.tile * 16 : next.tile * 32 + r * 16;
      next.codes[r] = w.codes.ptr + e * w.codes_expert + n * w.codes.stride + step * 128;
      const uint64_t at = w.scales.ptr + e * w.scales_expert + n * w.scales.stride + step * 8;
      const uint32_t row = (uint32_t)at % 4 + lane / 4 * (uint32_t)w.scales.stride;  // bytes from at's word
      next.scales[r] = at / 4 * 4;
      word[r][0] = (row / 4 + min(lane % 4, (row % 4 + 7) / 4)) * 4;
      word[r][1] = (row / 4 + min(lane % 4, (row % 4 + last) / 4)) * 4;
    }
  };
  const uint64_t codes_stride = (INNER ? a.gate : a.down).codes.stride, code_rows = codes_stride * (INNER ? 16 : 32);
  const uint64_t scales_stride = (INNER ? a.gate : a.down).scales.stride, scale_rows = scales_stride * (INNER ? 16 : 32);
  auto forward = [&] {
    --next.left;
    if (--next.run) {
#pragma unroll
      for (int r = 0; r < M; ++r) next.codes[r] += code_rows, next.scales[r] += scale_rows;
    } else if (next.left) {
      next.tile = 0;
      if (++next.chunk == chunks) next.chunk = 0, ++next.slot;
      enter();
    }
  };
  const uint32_t codes_at = lds_address(codes) + wave * (NS * kCodes * 16);
  const uint32_t scales_at = lds_address(scales) + wave * (NS * kWords * 4);
  const uint32_t none_at = scalar(lds_address(none) + wave * 16);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint32_t c = (lane & 7) ^ (j * 4 + (lane >> 4)), row = (j * 8 + lane / 8) * (uint32_t)codes_stride;
    from[0][j] = row + c * 16, from[1][j] = row + min(c, last) * 16;
  }
  // Step u of the tile to the ring's place `at`.  Steps that the tile does not have are requests too, of one lane and to
  // nowhere, so that a wait can count on them.
  auto request = [&](uint32_t at, int u) {
    const int r = u / S, s = u % S;
    const GlobalBytes code = uniform(next.codes[r] + s * 8 * 128), scale = uniform(next.scales[r] + s * 8 * 8);
    const uint32_t to = scalar(codes_at + at * (kCodes * 16)), scales_to = scalar(scales_at + at * (kWords * 4));
    if (s < next.n) {
      const bool part = s == next.part;
#pragma unroll
      for (int j = 0; j < 2; ++j) dma16_once(code, part ? from[1][j] : from[0][j], to + j * 1024);
      dma4(scale, part ? word[r][1] : word[r][0], scales_to);
    } else if (lane == 0) {
#pragma unroll
      for (uint32_t j = 0; j < N; ++j) dma4(uniform(next.scales[r] - wave * 8), word[r][1], none_at);
    }
  };
  enter();
#pragma unroll
  for (uint32_t k = 0; k < NS; ++k)
    if (next.left) {
      request(k, k % U);
      if (k % U == U - 1) forward();
    }
  uint32_t ring = 0;  // where the tile's first step is
  auto wrapped = [](uint32_t at) { return at >= NS ? at - NS : at; };

  // Sums of a tile: every 2 * NC wavefronts in turn add them up, each of 16 columns two rows of every four.
  constexpr uint32_t kTurns = 4 / NC;
  static_assert(4 % NC == 0);
  const uint32_t turn = wave / (2 * NC), group = wave / 2 % NC, n_in = q * 4 + wave % 2 * 2;
  const uint32_t summed = lds_address(sums) + (group * 128 + wave % 2 * 64 + lane) * 8;
  const bool biased = INNER && (a.gate.bias || a.up.bias);
  u32x4 x[S][NC][8];
  // A block's scale among a step's eight, blocks past the row's end having the last one's.
  uint32_t pick[2][2], shift[M] = {};
#pragma unroll
  for (uint32_t h = 0; h < 2; ++h) pick[0][h] = (h * 4 + q) | 0x0C0C0C00, pick[1][h] = min(h * 4 + q, last) | 0x0C0C0C00;
  uint32_t e = 0, t0 = 0, tokens = 0, used = 0;
  bool fresh = true;
  while (left) {
    const uint32_t run = min(tiles - tile, left), mine = steps_of(chunk);
    if (fresh || chunk == 0) {  // the expert's pairs, in the order of the tokens; every wavefront writes the same
      e = scalar(slots[slot]), t0 = (e >> 16) * most, e &= 0xFFFF;
      int32_t pair = -1;
      if (lane < a.tokens)
        for (uint32_t k = 0; k < a.top_k; ++k)
          if (chosen[lane * a.top_k + k] == (int32_t)e) pair = (int32_t)(lane * a.top_k + k);
      const uint64_t mask = __ballot(pair >= 0);
      if (pair >= 0) list[__popcll(mask & ((1ull << lane) - 1))] = pair;
      tokens = min((uint32_t)__popcll(mask) - t0, most), used = (tokens + each - 1) / each;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
      for (int r = 0; r < M; ++r) {  // bytes from a word to the row's first scale
        const MxExperts& w = INNER ? (r ? a.up : a.gate) : a.down;
        shift[r] = (uint32_t)(w.scales.ptr + e * w.scales_expert + i * w.scales.stride) % 4;
      }
      fresh = false;
    }
    const uint32_t part = part_of(chunk, mine);
    const GlobalBytes x0 = global_bytes(INNER ? m.p.x : m.p.h);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (c < used) {
        uint32_t t = c * each + i / parts, p = i % parts;  // columns without a token repeat the first
        if (i >= each * parts || t >= tokens) t = 0, p = 0;
        const uint32_t pair = (uint32_t)list[t0 + t];
        const uint32_t row = INNER ? p * (uint32_t)a.tokens + pair / a.top_k : p * pairs + pair;
        const uint32_t at = row * x_len * 2 + (chunk * span + wave) * (kMoeStep * 2) + q * 16;
#pragma unroll
        for (int s = 0; s < S; ++s)
          if (s < mine)
#pragma unroll
            for (int u = 0; u < 8; ++u) x[s][c][u] = ld16(x0, at + s * 8 * (kMoeStep * 2) + u * 64);
      }
    }
    // where this lane's sums go: of the first part's column
    const uint32_t t = group * each + i / parts;
    const bool stores = i % parts == 0 && i / parts < each && t < tokens;
    const uint64_t pair = stores ? (uint32_t)list[t0 + t] : 0;
    const uint64_t out = INNER ? m.p.h + pair * m.p.h_len * 2 + chunk_at(n_in / 8) * 16 + n_in % 8 * 2
                               : m.p.y + ((chunk * (uint64_t)pairs + pair) * rows + n_in) * 4;
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0), here rather than before each tile's first product

    f32x2 v[M] = {};
    auto add_up = [&] {
      f32x2 terms[8][M];
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int r = 0; r < M; ++r)
          terms[k][r] = __builtin_bit_cast(f32x2, *(LdsPairs)(summed + (k * M + r) * NC * 1024));
#pragma unroll
      for (int r = 0; r < M; ++r) {
        v[r] = terms[0][r];
#pragma unroll
        for (int k = 1; k < 8; ++k) v[r] += terms[k][r];
      }
    };
    uint32_t bias0 = 0;
    auto store = [&](uint32_t tile) {
      // a token's parts are columns side by side
#pragma unroll
      for (int r = 0; r < M; ++r) {
        const f32x2 own = v[r];
        if (parts > 1) v[r] += f32x2{right<1>(own[0]), right<1>(own[1])};
        if (parts > 2) v[r] += f32x2{right<2>(own[0]), right<2>(own[1])};
      }
      if (!stores) return;
      if constexpr (INNER) {
        if (biased) {
          const uint32_t at = (tile - bias0) * 16 + n_in;
          v[0] += f32x2{biases[0][at], biases[0][at + 1]}, v[1] += f32x2{biases[1][at], biases[1][at + 1]};
        }
        store_h(out + chunk_at(tile * 2) * 16, (uint64_t)pairs * m.p.h_len * 2,
                f32x2{activated(v[0][0], v[1][0]), activated(v[0][1], v[1][1])});
      } else {
#pragma unroll
        for (int r = 0; r < M; ++r) st8(out + tile * 128 + r * 64, __builtin_bit_cast(uint64_t, v[r]));
      }
    };
    auto walk = [&](auto used_) {
      constexpr int used = used_;
      for (uint32_t k = 0; k < run; ++k) {
        bool open = k > 0 && (k - 1) % kTurns == turn && group < used;  // the last tile's sums are this wavefront's
        if (open) add_up();
        if (biased && k % kBiasTiles == 0) {
          if (open) store(tile + k - 1), open = false;  // with the biases before
          bias0 = tile + k;
          __syncthreads();
          const uint32_t n = bias0 * 16 + threadIdx.x;
          static_assert(kBiasTiles * 16 <= 512, "a thread a row");
          if (INNER && threadIdx.x < kBiasTiles * 16 && n < rows) {
#pragma unroll
            for (int r = 0; r < M; ++r) {
              float bias[1];
              biases_of(r ? a.up : a.gate, a.out_type, e, n, bias);
              biases[r][INNER ? threadIdx.x : 0] = bias[0];
            }
          }
          __syncthreads();
        }
        f32x4 acc[M][used] = {};
#pragma unroll
        for (int r = 0; r < M; ++r)
#pragma unroll
          for (int s = 0; s < S; ++s) {
            const uint32_t at = wrapped(ring + (r * S + s) % NS);
            if (s < mine) {
              if (next.left)
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 1) * N) : "memory");
              else
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
              const u32x4 words = *(LdsChunks)(scales_at + i * 16 + at * (kWords * 4));
              u32x4 w4[2];
#pragma unroll
              for (int h = 0; h < 2; ++h)
                w4[h] = *(LdsChunks)(codes_at + (i * 8 + ((h * 4 + q) ^ (i / 2))) * 16 + at * (kCodes * 16));
              asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
              if (next.left) request(at, (r * S + s + D) % U);  // in place of what has just been read
              const uint32_t low = __builtin_amdgcn_alignbyte(words[1], words[0], shift[r]);
              const uint32_t high = __builtin_amdgcn_alignbyte(words[2], words[1], shift[r]);
              float scale[2];
#pragma unroll
              for (int h = 0; h < 2; ++h)
                scale[h] = scale_f32(__builtin_amdgcn_perm(high, low, s == part ? pick[1][h] : pick[0][h]));
#pragma unroll
              for (int u = 0; u < 8; ++u) {
                const u32x4 w8 = weights8(w4[u / 4][u % 4], scale[u / 4]);
#pragma unroll
                for (int c = 0; c < used; ++c) acc[r][c] = mfma(w8, x[s][c][u], acc[r][c]);
              }
            } else if (next.left) {
              request(at, (r * S + s + D) % U);
            }
            if ((r * S + s + D) % U == U - 1 && next.left) forward();
          }
        ring = wrapped(ring + U % NS);
        if (open) store(tile + k - 1);
        // Sums to LDS, 16 columns at a time: lane l has rows 4 (l / 16) .. + 3 of column l % 16.
        __builtin_amdgcn_s_barrier();  // the ones before have been read
        asm volatile("" ::: "memory");
#pragma unroll
        for (int r = 0; r < M; ++r)
#pragma unroll
          for (int c = 0; c < used; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              sums[((wave * M + r) * NC + c) * 128 + h * 64 + lane] = f32x2{acc[r][c][2 * h], acc[r][c][2 * h + 1]};
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
      }
      if ((run - 1) % kTurns == turn && group < used) add_up(), store(tile + run - 1);
    };
    if (NC > 3 && used > 3)
      walk(std::integral_constant<int, NC>{});
    else if (NC > 2 && used > 2)
      walk(std::integral_constant<int, NC < 3 ? NC : 3>{});
    else if (NC > 1 && used > 1)
      walk(std::integral_constant<int, NC < 2 ? NC : 2>{});
    else
      walk(std::integral_constant<int, 1>{});
    left -= run, tile = 0;
    if (++chunk == chunks) chunk = 0, ++slot;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // for requests to nowhere, while the workgroup's LDS is its own
}

// The weighted sums of each token's experts, the largest weight first.  64 tokens of 4096, two experts in seven chunks:
// 5.7 us for 15 MB that lie in the last-level cache, the launch and one trip to memory.
__global__ __launch_bounds__(256) void moe_combine_kernel(MoeArgs m) {
  const MxMoeArgs& a = m.a;
  const uint32_t per = a.cols / 4, at = blockIdx.x * 256 + threadIdx.x, t = at / per, n = (at - t * per) * 4;
  if (t >= a.tokens) return;
  const uint64_t pairs = a.tokens * a.top_k;
  const uint32_t terms = a.top_k * m.chunks;
  constexpr uint32_t kAhead = 8;  // terms on their way at a time
  f32x4 v = {};
  for (uint32_t j0 = 0; j0 < terms; j0 += kAhead) {
    f32x4 y[kAhead];
    float weight[kAhead];
    int32_t e[kAhead];
#pragma unroll
    for (uint32_t j = 0; j < kAhead; ++j) {
      const uint32_t term = min(j0 + j, terms - 1), k = term / m.chunks;
      const uint64_t pair = t * a.top_k + k;
      e[j] = g_ld<int32_t>(m.p.chosen + pair * 4), weight[j] = g_ld<float>(m.p.weights + pair * 4);
      y[j] = __builtin_bit_cast(f32x4, ld16(m.p.y + (((term - k * m.chunks) * pairs + pair) * a.cols + n) * 4));
    }
#pragma unroll
    for (uint32_t j = 0; j < kAhead; ++j)
      if (j0 + j < terms && e[j] >= 0) v += weight[j] * y[j];
  }
  for (uint32_t k0 = 0; a.down.bias && k0 < a.top_k; k0 += 4) {
    float weight[4], bias[4][4];
    int32_t e[4];
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
      const uint64_t pair = t * a.top_k + min(k0 + k, a.top_k - 1);
      e[k] = g_ld<int32_t>(m.p.chosen + pair * 4), weight[k] = g_ld<float>(m.p.weights + pair * 4);
      biases_of(a.down, a.out_type, (uint32_t)max(e[k], 0), n, bias[k]);
    }
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k)
      if (k0 + k < a.top_k && e[k] >= 0)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += weight[k] * bias[k][i];
  }
  store_out(a, t, n, v);
}

template <bool INNER, bool ALL, int WR, int KG, int XC, int NS>
hipError_t product_of(const MoeArgs& m, bool dma, hipStream_t stream) {
  constexpr uint32_t kRows = 16 * WR;
  const uint64_t tiles = ((INNER ? m.a.inner : m.a.cols) + kRows - 1) / kRows, pairs = m.a.tokens * m.a.top_k;
  const uint64_t items = ALL ? 1 : pairs < m.a.experts ? pairs : m.a.experts;
  return launch(dma ? moe_product_kernel<INNER, ALL, WR, KG, XC, NS, true>
                    : moe_product_kernel<INNER, ALL, WR, KG, XC, NS, false>,
                items * tiles, 64 * WR * KG, m, stream);
}

template <bool INNER, int S, int NC>
hipError_t stream_of(const MoeArgs& m, hipStream_t stream) {
  return launch(moe_stream_kernel<INNER, S, NC>, kStreamGroups, 512, m, stream);
}

hipError_t logits_of(const MoeArgs& m, hipStream_t stream) {
  const uint64_t groups = m.a.experts * ((m.a.tokens + kLogitTokens - 1) / kLogitTokens) + m.a.tokens;
  switch (m.a.x_type) {
    case kTypeF32: return launch(moe_logits_kernel<kTypeF32>, groups, kLogitThreads, m, stream);
    case kTypeF16: return launch(moe_logits_kernel<kTypeF16>, groups, kLogitThreads, m, stream);
    case kTypeBf16: return launch(moe_logits_kernel<kTypeBf16>, groups, kLogitThreads, m, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

uint64_t mxfp4_moe_workspace(const MxMoeArgs& a) { return places_of(a).end - a.workspace; }

hipError_t launch_mxfp4_moe(const MxMoeArgs& a, hipStream_t stream) {
  return in_parts(a.tokens, kMoeTokens, [&](uint64_t first, uint64_t tokens) {
    MoeArgs m{a, places_of(a), 1, 1, false};
    m.a.tokens = tokens;
    m.a.x = rows_from(a.x, first, type_bytes(a.x_type)), m.a.out = rows_from(a.out, first, type_bytes(a.out_type));
    if (a.experts_out) m.a.experts_out += first * a.top_k * 4;
    if (a.weights_out) m.a.weights_out += first * a.top_k * 4;
    const MxMoeChoice k = choose_mxfp4_moe(m.a);
    m.routed = k.routed;
    hipError_t e = logits_of(m, stream);
    if (e == hipSuccess && k.routed) e = launch(moe_route_kernel, tokens, 64, m, stream);
    if (e != hipSuccess) return e;
    m.span = m.p.x_len / kMoeStep;
    switch (k.inner) {
      case MxMoeChoice::kRows16: e = product_of<true, false, 1, 4, 4, 2>(m, k.inner_dma, stream); break;
      case MxMoeChoice::kRows64: e = product_of<true, false, 4, 1, 16, 2>(m, k.inner_dma, stream); break;
      case MxMoeChoice::kStream2: e = stream_of<true, 2, 2>(m, stream); break;
      case MxMoeChoice::kStream4: e = stream_of<true, 4, 1>(m, stream); break;
    }
    if (e != hipSuccess) return e;
    m.span = k.span, m.chunks = k.chunks;
    switch (k.outer) {
      case MxMoeChoice::kSums1: return product_of<false, true, 1, 8, 4, 3>(m, k.outer_dma, stream);
      case MxMoeChoice::kSums2: return product_of<false, true, 1, 8, 6, 3>(m, k.outer_dma, stream);
      case MxMoeChoice::kRows: e = product_of<false, false, 4, 1, 16, 3>(m, k.outer_dma, stream); break;
      case MxMoeChoice::kChunks: e = stream_of<false, 1, 4>(m, stream); break;
    }
    if (e == hipSuccess) e = launch(moe_combine_kernel, (tokens * (a.cols / 4) + 255) / 256, 256, m, stream);
    return e;
  });
}

}  // namespace ptwm
