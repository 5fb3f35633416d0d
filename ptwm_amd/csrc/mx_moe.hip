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
//
// The products are of bf16 on the matrix unit.  Weights are widened to bf16,
// which is exact; x, and h, are the sum of one to three bf16 values (parts),
// each of which is a column of the product of its own, summed with its like at
// the end.  So an instruction's 16 columns are one to three columns a token,
// whatever the types, and few tokens in two parts cost no more than in one.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "mx_device.h"

namespace ptwm {
namespace {

constexpr uint32_t kTokens = 64;  // of a launch; longer calls run in several
constexpr uint32_t kStep = 256;   // values of a row that go through LDS together: a cache line of codes

// h's parts: 24 significant bits where the outputs have 24, else 16, the rounding of a 2^-8 or 2^-5 of the output's own.
constexpr uint32_t inner_parts(uint32_t out_type) { return out_type == kTypeF32 ? 3 : 2; }

// Where a launch's intermediate results lie in the workspace.  A pair is a token's k-th expert, token * top_k + k.
struct MoePlaces {
  uint64_t logits;   // f64 [tokens][experts]
  uint64_t x;        // bf16 [parts][tokens][x_len]
  uint64_t h;        // bf16 [parts][pairs][h_len]
  uint64_t y;        // f32 [pairs][cols]
  uint64_t chosen;   // int32 [pairs], -1 where a chosen expert is masked
  uint64_t weights;  // f32 [pairs]
  uint64_t end;
  uint32_t x_len, h_len;  // cols and inner in whole steps, zeros past their ends
};
MoePlaces places_of(const MxMoeArgs& a) {
  const uint64_t t = a.tokens < kTokens ? a.tokens : kTokens, pairs = t * a.top_k;
  uint64_t at = a.workspace;
  const auto take = [&](uint64_t bytes) {
    const uint64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  MoePlaces p;
  p.x_len = (a.cols + kStep - 1) / kStep * kStep, p.h_len = (a.inner + kStep - 1) / kStep * kStep;
  p.logits = take(t * a.experts * 8);
  p.x = take(parts_of(a.x_type) * t * p.x_len * 2);
  p.h = take(inner_parts(a.out_type) * pairs * p.h_len * 2);
  p.y = take(pairs * a.cols * 4);
  p.chosen = take(pairs * 4), p.weights = take(pairs * 4);
  p.end = at;
  return p;
}

struct MoeArgs {
  MxMoeArgs a;
  MoePlaces p;
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
__device__ __forceinline__ void store1_as(uint32_t type, uint64_t base, uint64_t at, float v) {
  if (type == kTypeBf16)
    store1<kTypeBf16>(base + at * 2, v);
  else if (type == kTypeF16)
    store1<kTypeF16>(base + at * 2, v);
  else
    store1<kTypeF32>(base + at * 4, v);
}
__device__ __forceinline__ float bias_of(const MxExperts& w, uint32_t type, uint32_t e, uint32_t n) {
  return w.bias ? load1_as(type, w.bias, e * w.bias_expert + n * w.bias_stride) : 0.0f;
}

// Logits of one expert and four tokens: the threads take turns along the rows.  Summed in 64 bits, in which products
// are exact, so that which of two near experts is chosen does not depend on the order of the additions.  The
// workgroups after these write x's parts, a token each.
constexpr uint32_t kLogitTokens = 4;
constexpr uint32_t kLogitThreads = 512;
template <uint32_t T>
__global__ __launch_bounds__(kLogitThreads) void moe_logits_kernel(MoeArgs m) {
  const MxMoeArgs& a = m.a;
  __shared__ double part[kLogitTokens][kLogitThreads];
  const uint32_t groups = ((uint32_t)a.tokens + kLogitTokens - 1) / kLogitTokens;
  if (blockIdx.x >= a.experts * groups) {
    const uint32_t t = blockIdx.x - a.experts * groups;
    for (uint32_t k = threadIdx.x * 8; k < m.p.x_len; k += kLogitThreads * 8) {
      u32x4 p[parts_of(T)] = {};
      if (k < a.cols) parts_of_raw<T>(load_raw8<T>(a.x.ptr + (t * a.x.stride + k) * type_bytes(T)), 1.0f, p);
#pragma unroll
      for (int j = 0; j < parts_of(T); ++j) st16(m.p.x + ((j * a.tokens + t) * m.p.x_len + k) * 2, p[j]);
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
#pragma unroll
  for (uint32_t t = 0; t < kLogitTokens; ++t) part[t][threadIdx.x] = sum[t];
  __syncthreads();
  const uint32_t t = threadIdx.x >> 6, lane = threadIdx.x & 63;  // a wavefront a token
  if (t >= kLogitTokens || t0 + t >= a.tokens) return;
  double v = 0;
#pragma unroll
  for (uint32_t k = 0; k < kLogitThreads; k += 64) v += part[t][k + lane];
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
  if (lane == 0) {
    if (a.router_bias) v += (double)load1_as(a.router_type, a.router_bias, e);
    g_st<double>(m.p.logits + ((uint64_t)(t0 + t) * a.experts + e) * 8, v);
  }
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

// The largest of a wavefront's values, in all lanes.
template <int CTRL>
__device__ __forceinline__ uint32_t larger_by(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = larger_by<0x111>(v), v = larger_by<0x112>(v), v = larger_by<0x114>(v), v = larger_by<0x118>(v);  // in rows of 16
  v = larger_by<0x142>(v), v = larger_by<0x143>(v);  // a row's last lane to the next rows
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
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
    uint32_t owner = (uint32_t)__ffsll((long long)at) - 1, low = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)most, (int)owner);
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

// Pairs whose experts the inner products' workgroups choose for themselves, each all of them.
constexpr uint32_t kFusedPairs = 32;

// Rows of one expert's products for its tokens (or, ALL, of the outer products
// of all experts of up to 64 pairs, weighted and added up).  WR wavefronts hold
// 16 * RP rows each, of gate and up (INNER) or of down, and share the columns;
// KG groups of them take turns in steps of 256 values along the rows and add up
// in LDS at the end.
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
// kDma 2: codes lie at multiples of 16 bytes and scales of 4, whole words of
// four blocks; 1: codes only, scales come byte by byte; 0: codes go through
// registers.
template <bool INNER, bool ALL, int WR, int KG, int RP, int XC, int NS, int kDma>
__global__ __launch_bounds__(64 * WR * KG) void moe_product_kernel(MoeArgs m) {
  static_assert(WR == 1 || KG == 1, "groups of several wavefronts meet at barriers of the whole workgroup");
  static_assert(!(INNER && ALL) && (!INNER || RP == 1) && (!ALL || XC <= 16), "one group of columns for all tokens");
  constexpr int M = INNER ? 2 : 1, RT = M * RP;               // matrices, 16s of rows
  constexpr int NC = (XC + 15) / 16, CW = XC < 16 ? XC : 16;  // groups of columns, columns of one
  constexpr uint32_t G = 64 * WR, kWaves = WR * KG, kRows = 16 * RP * WR;
  constexpr uint32_t kCodes = RT * 128, kColumns = XC * 32;  // chunks of a stage
  constexpr int JW = kCodes / 64, JX = kColumns / G, JS = kDma == 2 ? 1 : 2 * RT;
  constexpr int N = JX + (kDma > 0 ? JW : 0) + JS;  // requests of a step
  constexpr uint32_t kScales = JS * 64;                                          // words of a stage
  static_assert(kColumns % G == 0 && RT <= 2 && (NS - 2) * N < 64, "whole requests, and a wait that counts them");
  __shared__ u32x4 columns[KG * NS * kColumns], codes[KG * WR * NS * kCodes];
  __shared__ uint32_t scales[KG * WR * NS * kScales];
  __shared__ int32_t list[64], table[ALL ? 64 * CW : 1], fused[INNER ? kFusedPairs : 1];
  __shared__ float weights[ALL ? 64 : 1];
  const MxMoeArgs& a = m.a;
  const uint32_t lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
  const uint64_t below = (1ull << lane) - 1;  // lanes
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t group = wave / WR, wr = wave % WR, gi = wr * 64 + lane;
  const uint32_t rows = INNER ? a.inner : a.cols, length = INNER ? a.cols : a.inner, blocks = length / kMxBlock;
  const uint32_t x_len = INNER ? m.p.x_len : m.p.h_len, steps = x_len / kStep;
  const uint32_t tiles = ((INNER ? m.p.h_len : rows) + kRows - 1) / kRows;
  const uint32_t slot = blockIdx.x / tiles, n0 = blockIdx.x % tiles * kRows;
  const uint32_t parts = INNER ? parts_of(a.x_type) : inner_parts(a.out_type), each = CW / parts;  // tokens of CW columns
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
    for (uint32_t k = lane; k < experts * CW; k += 64) table[k] = -1;
    if (e >= 0) {
      const uint32_t k = __popcll(leaders & ((1ull << leader) - 1));
      table[k * CW + lane / a.top_k] = (int32_t)lane;
      if (leader == lane) list[k] = e;
    }
    __syncthreads();
    if (lane < experts) expert_k = list[lane];
  } else {
    const bool choosing = INNER && pairs <= kFusedPairs;
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
  auto row_of = [&](int r, uint32_t in) { return min(n0 + (wr * RP + (INNER ? 0 : r)) * 16 + in, rows - 1); };
  auto scales_of = [&](int r, uint32_t n) {
    const MxExperts& w = matrix(r);
    return w.scales.ptr + e0 * w.scales_expert + n * w.scales.stride;
  };
#pragma unroll
  for (int j = 0; j < JW; ++j) {
    const MxExperts& w = matrix(j / 2);
    w_at[j] = w.codes.ptr + e0 * w.codes_expert + row_of(j / 2, j % 2 * 8 + lane / 8) * w.codes.stride;
  }
  if constexpr (kDma == 2) {  // two words a row
    s_at[0] = RT == 2 && lane >= 32 ? scales_of(1, row_of(1, lane / 2 % 16)) : scales_of(0, row_of(0, lane / 2 % 16));
  } else {  // eight bytes a row
#pragma unroll
    for (int j = 0; j < JS; ++j) s_at[j] = scales_of(j / 2, row_of(j / 2, j % 2 * 8 + lane / 8));
  }
  const uint32_t columns_at = lds_address(columns) + group * (NS * kColumns * 16);
  const uint32_t codes_at = lds_address(codes) + wave * (NS * kCodes * 16);
  const uint32_t scales_at = lds_address(scales) + wave * (NS * kScales * 4);

  for (uint32_t t0 = 0; t0 < count; t0 += each * NC) {
    const uint32_t tokens = min(count - t0, each * NC), used = (tokens + each - 1) / each;  // groups of columns
    // A lane's chunks of the columns, as offsets: column c holds part c % parts of a token; columns without one repeat
    // the first.  (2^31 bytes hold 3 parts of 2048 pairs of the longest rows.)
    uint32_t x_at[JX], x_token[ALL ? JX : 1];
#pragma unroll
    for (int j = 0; j < JX; ++j) {
      const uint32_t column = (j * G + gi) / 32, c = column % CW;
      uint32_t t = column / CW * each + c / parts, part = c % parts;
      if (c >= each * parts || t >= tokens) t = 0, part = 0;
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
        if constexpr (kDma > 0)
          dma16(from, codes_at + (stage * kCodes + j * 64) * 16);
        else
          ((LdsChunks)(codes_at + (stage * kCodes + lane) * 16))[j * 64] = ld16(from);
      }
#pragma unroll
      for (int j = 0; j < JS; ++j) {
        const uint64_t from = s_at[j] + e * a.down.scales_expert;
        const uint32_t to = scales_at + (stage * kScales + j * 64) * 4;
        if constexpr (kDma == 2)
          dma4(from + min(u.step * 2 + (lane & 1), blocks / 4 - 1) * 4, to);
        else
          dma1(from + min(u.step * 8 + (lane & 7), blocks - 1), to);
      }
#pragma unroll
      for (int j = 0; j < JX; ++j) {
        if (NS == 2 && NC > 1 && j * G >= used * 512) break;  // a wait for all needs no count of them
        uint32_t from = x_at[j] + u.step * (kStep * 2);
        if constexpr (ALL) {
          // a token that did not choose the expert has another's h here, whose sums are left out
          const int32_t pair = table[u.k * CW + x_token[j]];
          from += (uint32_t)max(pair, 0) * x_len * 2;
        }
        dma16(x0, from, columns_at + (stage * kColumns + j * G + wr * 64) * 16);
      }
    };
    f32x4 acc[RT][NC] = {}, total[ALL ? RT : 1][NC] = {};
    auto compute = [&](uint32_t stage, auto used_) {
      constexpr int used = used_;
      u32x2 words[RT];
      if constexpr (kDma == 2) {
#pragma unroll
        for (int r = 0; r < RT; ++r) words[r] = *(LdsPairs)(scales_at + stage * (kScales * 4) + (r * 16 + i) * 8);
      }
      u32x4 wv[2][RT];
      float sf[2][RT];
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const uint32_t row = r * 16 + i, c = s * 4 + q;
          wv[s][r] = *(LdsChunks)(codes_at + (stage * kCodes + row * 8 + (c ^ (row / 2 & 7))) * 16);
          sf[s][r] = scale_f32(kDma == 2 ? words[r][s] >> 8 * q & 0xFF
                                         : *(LdsWord)(scales_at + (stage * kScales + row * 8 + c) * 4));
        }
      // columns are read a product ahead, and no further: eight products' are more than the registers
      u32x4 xv[2][used];
      auto read = [&](int u) {
#pragma unroll
        for (int c = 0; c < used; ++c) {
          const uint32_t column = c * 16 + i % CW, chunk = (u / 4 * 4 + q) * 4 + u % 4;
          xv[u & 1][c] = *(LdsChunks)(columns_at + (stage * kColumns + column * 32 + (chunk ^ (column & 15))) * 16);
        }
      };
      read(0);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        if (u < 7) read(u + 1);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const u32x4 w8 = weights8(wv[u / 4][r][u % 4], sf[u / 4][r]);
#pragma unroll
          for (int c = 0; c < used; ++c) acc[r][c] = mfma(w8, xv[u & 1][c], acc[r][c]);
        }
        if constexpr (used > 2) __builtin_amdgcn_sched_barrier(0);
      }
    };
    auto add_expert = [&](uint32_t k) {  // an expert's sums, weighted, for the tokens that chose it
      const uint32_t c = i % CW, t = c / parts;
      const int32_t pair = c < each * parts && t < tokens ? table[ALL ? k * CW + t : 0] : -1;
      const float weight = weights[ALL ? max(pair, 0) : 0];
#pragma unroll
      for (int r = 0; r < (ALL ? RT : 1); ++r) {
        const f32x4 more = total[r][0] + weight * acc[r][0];
        total[r][0] = pair >= 0 ? more : total[r][0];
        acc[r][0] = f32x4{};
      }
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
        if (NC > 1 && used > 1)
          compute(stage, std::integral_constant<int, NC < 2 ? NC : 2>{});
        else
          compute(stage, std::integral_constant<int, 1>{});
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
    static_assert(RT * NC * 64 <= NS * kCodes, "a wavefront's sums fit its codes");
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int c = 0; c < NC; ++c) sums[((wave * RT + r) * NC + c) * 64 + lane] = ALL ? total[ALL ? r : 0][c] : acc[r][c];
    __syncthreads();
    // of 16s `r` of wavefront w of a group, row `in`, token t: over its parts and the groups
    auto sum_of = [&](uint32_t w, uint32_t r, uint32_t in, uint32_t t) {
      const uint32_t c = t / each, column = t % each * parts;
      float v = 0;
#pragma unroll
      for (uint32_t g = 0; g < KG; ++g)
        for (uint32_t p = 0; p < parts; ++p)
          v += sums[(((g * WR + w) * RT + r) * NC + c) * 64 + in / 4 * 16 + column + p][in & 3];
      return v;
    };
    for (uint32_t at = threadIdx.x; at < tokens * kRows; at += 64 * kWaves) {
      const uint32_t t = at / kRows, in = at % kRows, w = in / (16 * RP), rp = in / 16 % RP, n = n0 + in;
      const uint64_t pair = ALL ? 0 : (uint32_t)list[t0 + t];
      if constexpr (INNER) {
        if (n >= m.p.h_len) continue;
        float h = 0;
        if (n < a.inner) {
          const float g = sum_of(w, 0, in % 16, t) + bias_of(a.gate, a.out_type, e0, n);
          const float u = sum_of(w, 1, in % 16, t) + bias_of(a.up, a.out_type, e0, n);
          h = g / (1.0f + expf(-g)) * u;
        }
        // parts as x's, but for the last, which is rounded
        const uint32_t hp = inner_parts(a.out_type);
        for (uint32_t p = 0; p < hp; ++p) {
          uint16_t b;
          if (p + 1 < hp) {
            const uint32_t cut = f32_bits(__builtin_amdgcn_fmed3f(h, -kBf16Max, kBf16Max)) & 0xFFFF0000u;
            h -= bits_f32(cut);
            b = (uint16_t)(cut >> 16);
          } else {
            b = (uint16_t)pack2<kTypeBf16>(h, 0.0f);
          }
          g_st<uint16_t>(m.p.h + (((uint64_t)p * pairs + pair) * m.p.h_len + n) * 2, b);
        }
      } else if (n < rows) {
        float v = sum_of(w, rp, in % 16, t);
        if constexpr (ALL) {
          for (uint32_t k = 0; a.down.bias && k < experts; ++k) {
            const int32_t pair = table[k * CW + t];
            if (pair >= 0) v += weights[pair] * bias_of(a.down, a.out_type, (uint32_t)list[k], n);
          }
          store1_as(a.out_type, a.out.ptr, t * a.out.stride + n, v);
        } else {
          g_st<float>(m.p.y + (pair * rows + n) * 4, v + bias_of(a.down, a.out_type, e0, n));
        }
      }
    }
  }
}

// The weighted sums of each token's experts, the largest weight first.
__global__ __launch_bounds__(256) void moe_combine_kernel(MoeArgs m) {
  const MxMoeArgs& a = m.a;
  const uint32_t per = a.cols / 4, at = blockIdx.x * 256 + threadIdx.x, t = at / per, n = (at - t * per) * 4;
  if (t >= a.tokens) return;
  f32x4 v = {};
  for (uint32_t k0 = 0; k0 < a.top_k; k0 += 4) {  // four at a time on their way
    f32x4 y[4];
    float weight[4];
    int32_t e[4];
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
      const uint64_t pair = (uint64_t)t * a.top_k + min(k0 + k, a.top_k - 1);
      e[k] = g_ld<int32_t>(m.p.chosen + pair * 4), weight[k] = g_ld<float>(m.p.weights + pair * 4);
      y[k] = __builtin_bit_cast(f32x4, ld16(m.p.y + (pair * a.cols + n) * 4));
    }
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k)
      if (k0 + k < a.top_k && e[k] >= 0) v += weight[k] * y[k];
  }
  const uint64_t to = t * a.out.stride + n;
  if (a.out_type == kTypeBf16)
    st8(a.out.ptr + to * 2, pack2<kTypeBf16>(v[0], v[1]) | (uint64_t)pack2<kTypeBf16>(v[2], v[3]) << 32);
  else if (a.out_type == kTypeF16)
    st8(a.out.ptr + to * 2, pack2<kTypeF16>(v[0], v[1]) | (uint64_t)pack2<kTypeF16>(v[2], v[3]) << 32);
  else
    st16(a.out.ptr + to * 4, __builtin_bit_cast(u32x4, v));
}

// How far the weights of one product go by DMA.
int dma_of(const MxExperts& w, uint32_t length, uint64_t experts) {
  const auto at = [&](const MxRows& r, uint64_t expert, uint64_t n) {
    return r.ptr % n == 0 && r.stride % n == 0 && (experts == 1 || expert % n == 0);
  };
  if (!at(w.codes, w.codes_expert, 16)) return 0;
  return length % 128 == 0 && at(w.scales, w.scales_expert, 4) ? 2 : 1;
}

template <bool INNER, bool ALL, int WR, int KG, int RP, int XC, int NS>
hipError_t product_of(const MoeArgs& m, int dma, hipStream_t stream) {
  constexpr uint32_t kRows = 16 * RP * WR;
  const uint64_t tiles = ((INNER ? m.p.h_len : m.a.cols) + kRows - 1) / kRows, pairs = m.a.tokens * m.a.top_k;
  const uint64_t items = ALL ? 1 : pairs < m.a.experts ? pairs : m.a.experts;
  return launch(dma == 2   ? moe_product_kernel<INNER, ALL, WR, KG, RP, XC, NS, 2>
                : dma == 1 ? moe_product_kernel<INNER, ALL, WR, KG, RP, XC, NS, 1>
                           : moe_product_kernel<INNER, ALL, WR, KG, RP, XC, NS, 0>,
                items * tiles, 64 * WR * KG, m, stream);
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
  const int gate = dma_of(a.gate, a.cols, a.experts), up = dma_of(a.up, a.cols, a.experts);
  const int inner = gate < up ? gate : up, outer = dma_of(a.down, a.inner, a.experts);
  return in_parts(a.tokens, kTokens, [&](uint64_t first, uint64_t tokens) {
    MoeArgs m{a, places_of(a)};
    m.a.tokens = tokens;
    m.a.x = rows_from(a.x, first, type_bytes(a.x_type)), m.a.out = rows_from(a.out, first, type_bytes(a.out_type));
    if (a.experts_out) m.a.experts_out += first * a.top_k * 4;
    if (a.weights_out) m.a.weights_out += first * a.top_k * 4;
    hipError_t e = logits_of(m, stream);
    const uint64_t pairs = tokens * a.top_k;
    const uint32_t xp = parts_of(a.x_type), hp = inner_parts(a.out_type);
    if (e == hipSuccess && pairs > kFusedPairs) e = launch(moe_route_kernel, tokens, 64, m, stream);
    if (e != hipSuccess) return e;
    // columns that an expert's tokens take on average
    const double inner_columns = (double)pairs / a.experts * xp, outer_columns = (double)pairs / a.experts * hp;
    if (tokens * xp <= 4)
      e = product_of<true, false, 1, 4, 1, 4, 2>(m, inner, stream);
    else if (tokens * xp <= 16 || inner_columns <= 8)
      e = product_of<true, false, 4, 1, 1, 16, 3>(m, inner, stream);
    else
      e = product_of<true, false, 4, 1, 1, 32, 2>(m, inner, stream);
    if (e != hipSuccess) return e;
    if (tokens * hp <= 4 && pairs <= 64) return product_of<false, true, 1, 8, 1, 4, 3>(m, outer, stream);
    if (tokens * hp <= 16 || outer_columns <= 8)
      e = product_of<false, false, 4, 1, 1, 16, 3>(m, outer, stream);
    else
      e = product_of<false, false, 4, 1, 2, 32, 2>(m, outer, stream);
    if (e == hipSuccess) e = launch(moe_combine_kernel, (tokens * (a.cols / 4) + 255) / 256, 256, m, stream);
    return e;
  });
}

}  // namespace ptwm
