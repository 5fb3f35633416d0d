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
//   route    (two tokens on) the choice, and the pairs of token and expert
//            sorted by expert
//   inner    gate and up products of an expert's tokens, h as bf16 parts
//   outer    the down products; of one token, their weighted sum at once
//   combine  (two tokens on) the weighted sums
// One token takes three launches: the inner products choose for themselves.
//
// The products are of bf16 on the matrix unit.  Weights are widened to bf16,
// which is exact; x, and h, are the sum of one to three bf16 values (parts),
// each of which is a column of the product of its own, summed with its like at
// the end.  So an instruction's 16 columns are one to three columns a token,
// whatever the types, and few tokens in two parts cost no more than in one.
#include <hip/hip_runtime.h>

#include "mx_device.h"

namespace ptwm {
namespace {

constexpr uint32_t kTokens = 64;  // of a launch; longer calls run in several
constexpr uint32_t kStep = 256;   // values of a row that go through LDS together: a cache line of codes

// h's parts: 24 significant bits where the outputs have 24, else 16, the rounding of a 2^-8 or 2^-5 of the output's own.
constexpr uint32_t inner_parts(uint32_t out_type) { return out_type == kTypeF32 ? 3 : 2; }

struct Active {  // an expert with tokens
  uint32_t expert, first, count, unused;
};

// Where a launch's intermediate results lie in the workspace.
struct MoePlaces {
  uint64_t logits;   // f64 [tokens][experts]
  uint64_t x;        // bf16 [parts][tokens][x_len]
  uint64_t h;        // bf16 [parts][tokens * top_k][h_len], rows sorted by expert
  uint64_t y;        // f32 [tokens * top_k][cols], rows as h's
  uint64_t chosen;   // int32 [tokens * top_k], -1 where a chosen expert is masked
  uint64_t weights;  // f32 [tokens * top_k]
  uint64_t place;    // int32 [tokens * top_k]: row of a pair in h and y, -1 without one
  uint64_t order;    // int32 [tokens * top_k]: the pair of a row
  uint64_t active;   // Active [experts with tokens]
  uint64_t actives;  // their number
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
  p.place = take(pairs * 4), p.order = take(pairs * 4);
  p.active = take((pairs < a.experts ? pairs : a.experts) * sizeof(Active));
  p.actives = take(4);
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

// Logits of one expert and four tokens: 256 threads take turns along the rows.  Summed in 64 bits, in which products
// are exact, so that which of two near experts is chosen does not depend on the order of the additions.  The
// workgroups after these write x's parts, a token each.
constexpr uint32_t kLogitTokens = 4;
template <uint32_t T>
__global__ __launch_bounds__(256) void moe_logits_kernel(MoeArgs m) {
  const MxMoeArgs& a = m.a;
  __shared__ double part[kLogitTokens][256];
  const uint32_t groups = ((uint32_t)a.tokens + kLogitTokens - 1) / kLogitTokens;
  if (blockIdx.x >= a.experts * groups) {
    const uint32_t t = blockIdx.x - a.experts * groups;
    for (uint32_t k = threadIdx.x * 8; k < m.p.x_len; k += 256 * 8) {
      u32x4 p[parts_of(T)] = {};
      if (k < a.cols) parts_of_raw<T>(load_raw8<T>(a.x.ptr + (t * a.x.stride + k) * type_bytes(T)), 1.0f, p);
#pragma unroll
      for (int j = 0; j < parts_of(T); ++j) st16(m.p.x + ((j * a.tokens + t) * m.p.x_len + k) * 2, p[j]);
    }
    return;
  }
  const uint32_t e = blockIdx.x / groups, t0 = blockIdx.x % groups * kLogitTokens;
  double sum[kLogitTokens] = {};
  for (uint32_t k = threadIdx.x * 8; k < a.cols; k += 256 * 8) {
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
  const uint32_t t = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (t0 + t >= a.tokens) return;
  double v = (part[t][lane] + part[t][lane + 64]) + (part[t][lane + 128] + part[t][lane + 192]);
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
__device__ __forceinline__ uint64_t larger_by(uint64_t v) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, 0xF, 0xF, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, 0xF, 0xF, false);
  const uint64_t other = lo | (uint64_t)hi << 32;
  return other > v ? other : v;
}
__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
  v = larger_by<0x111>(v), v = larger_by<0x112>(v), v = larger_by<0x114>(v), v = larger_by<0x118>(v);  // in rows of 16
  v = larger_by<0x142>(v), v = larger_by<0x143>(v);  // a row's last lane to the next rows
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, 63);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), 63);
  return lo | (uint64_t)hi << 32;
}

// A token's experts in the order of their logits, by one wavefront: the largest that is left, the lowest expert of equal
// ones.
struct Choice {
  uint64_t key[kMoeMaxExperts / 64];
  uint64_t best;  // the last one taken
  __device__ __forceinline__ Choice(const MoeArgs& m, uint32_t t) {
    const uint32_t lane = threadIdx.x & 63;
#pragma unroll
    for (uint32_t j = 0; j < kMoeMaxExperts / 64; ++j) {
      const uint32_t e = j * 64 + lane;
      key[j] = e < m.a.experts ? order_of(g_ld<double>(m.p.logits + ((uint64_t)t * m.a.experts + e) * 8)) : 0;
    }
  }
  __device__ __forceinline__ uint32_t next(uint32_t experts) {
    uint64_t most = 0;
#pragma unroll
    for (uint32_t j = 0; j < kMoeMaxExperts / 64; ++j)
      if (j * 64 < experts) most = key[j] > most ? key[j] : most;
    best = wave_max(most);
    uint32_t e = 0;
    bool found = false;
#pragma unroll
    for (uint32_t j = 0; j < kMoeMaxExperts / 64; ++j) {
      if (j * 64 >= experts || found) continue;
      const uint64_t at = __ballot(key[j] == best);
      if (!at) continue;
      found = true;
      const uint32_t lane = (uint32_t)__ffsll((long long)at) - 1;
      e = j * 64 + lane;
      if ((threadIdx.x & 63) == lane) key[j] = 0;
    }
    return e;
  }
};

// Chooses a token's experts: lane k returns the k-th, with its weight.  An expert at minus infinity has none, not even
// among its like.
struct Chosen {
  uint32_t expert;
  float weight;
  bool masked;
};
__device__ __forceinline__ Chosen choose(const MoeArgs& m, uint32_t t) {
  const uint32_t lane = threadIdx.x & 63;
  Choice c(m, t);
  Chosen mine{0, 0, false};
  double logit = 0, top = 0;
  for (uint32_t k = 0; k < m.a.top_k; ++k) {
    const uint32_t e = c.next(m.a.experts);
    const double l = logit_of(c.best);
    if (k == 0) top = l;
    if (k == lane) mine.expert = e, logit = l;
  }
  const bool in = lane < m.a.top_k;
  mine.masked = logit == -__builtin_inf();
  const float w = in && !mine.masked ? expf((float)(logit - top)) : 0.0f;
  float sum = w;
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) sum += __shfl_xor(sum, d, 64);
  mine.weight = mine.masked ? 0.0f : w / sum;
  if (in) {
    const uint64_t at = (uint64_t)t * m.a.top_k + lane;
    g_st<int32_t>(m.p.chosen + at * 4, mine.masked ? -1 : (int32_t)mine.expert);
    g_st<float>(m.p.weights + at * 4, mine.weight);
    if (m.a.experts_out) g_st<int32_t>(m.a.experts_out + at * 4, (int32_t)mine.expert);
    if (m.a.weights_out) g_st<float>(m.a.weights_out + at * 4, mine.weight);
  }
  return mine;
}

// The choice of all tokens and the pairs sorted by expert, then token, by one workgroup: a mask of tokens for each
// expert, whose counts say where its pairs start.
__global__ __launch_bounds__(1024) void moe_route_kernel(MoeArgs m) {
  const MxMoeArgs& a = m.a;
  __shared__ unsigned long long mask[kMoeMaxExperts];
  __shared__ uint32_t first[kMoeMaxExperts], sums[16][2];
  __shared__ int16_t chosen[kTokens * kMoeMaxTopK];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  mask[threadIdx.x] = 0;
  __syncthreads();
  for (uint32_t t = wave; t < a.tokens; t += 16) {
    const Chosen c = choose(m, t);
    if (lane < a.top_k) {
      chosen[t * a.top_k + lane] = c.masked ? -1 : (int16_t)c.expert;
      if (!c.masked) atomicOr(&mask[c.expert], 1ull << t);
    }
  }
  __syncthreads();
  // running sums over the experts: of their pairs, and of those that have any
  const uint32_t count = __popcll(mask[threadIdx.x]);
  uint32_t pairs = count, actives = count ? 1 : 0;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t p = __shfl_up(pairs, d, 64), q = __shfl_up(actives, d, 64);
    if (lane >= (uint32_t)d) pairs += p, actives += q;
  }
  if (lane == 63) sums[wave][0] = pairs, sums[wave][1] = actives;
  __syncthreads();
  for (uint32_t w = 0; w < wave; ++w) pairs += sums[w][0], actives += sums[w][1];
  first[threadIdx.x] = pairs - count;
  if (count) {
    const uint64_t to = m.p.active + (uint64_t)(actives - 1) * sizeof(Active);
    st16(to, u32x4_make(threadIdx.x, pairs - count, count, 0));
  }
  if (threadIdx.x == 1023) g_st<uint32_t>(m.p.actives, actives);
  __syncthreads();
  for (uint32_t p = threadIdx.x; p < a.tokens * a.top_k; p += 1024) {
    const int e = chosen[p];
    int32_t at = -1;
    if (e >= 0) {
      at = (int32_t)(first[e] + __popcll(mask[e] & ((1ull << p / a.top_k) - 1)));
      g_st<int32_t>(m.p.order + (uint64_t)at * 4, (int32_t)p);
    }
    g_st<int32_t>(m.p.place + (uint64_t)p * 4, at);
  }
}

// Rows of one expert's products for its tokens.  WR wavefronts hold 16 rows of
// gate and of up each (INNER), or 32 rows of down, and share the columns; KG
// groups of them take turns in steps of 256 values along the rows and add up in
// LDS at the end.  ONE: the call has one token; its outer products add up over
// all its experts at once, 16 rows a workgroup.
//
// Codes, scales and columns go through LDS by DMA, NS - 1 steps ahead: the
// matrix instruction's order, a row a lane, would cost the address unit a cycle
// a lane, and the requests need no registers.  A wavefront's codes and scales
// are its own; the columns of a group are loaded by all of it.  16-byte chunks of a row of
// codes (8) or of a column (32) lie at chunk ^ (row / 2 % 8) and chunk ^ (column
// % 16), so that the 16 lanes that read together meet every bank once.  In a
// product lane l takes block l / 16 of row (column) l % 16, values 8f .. 8f+7
// with product f of four.
//
// kDma 2: codes lie at multiples of 16 bytes and scales of 4, whole words of
// four blocks; 1: codes only, scales are loaded to registers a step ahead, which
// waits for all that is on its way; 0: codes go through registers too.
template <bool INNER, bool ONE, int WR, int KG, int XC, int NS, int kDma>
__global__ __launch_bounds__(64 * WR * KG) void moe_product_kernel(MoeArgs m) {
  static_assert(WR == 1 || KG == 1, "groups of several wavefronts meet at barriers of the whole workgroup");
  constexpr bool kAll = ONE && !INNER;                // over all experts
  constexpr int RP = INNER || ONE ? 1 : 2;            // 16s of rows of a matrix
  constexpr int M = INNER ? 2 : 1, RT = M * RP;       // matrices, 16s of rows
  constexpr int NC = (XC + 15) / 16, CW = XC < 16 ? XC : 16;  // groups of columns, columns of one
  constexpr uint32_t G = 64 * WR, kRows = 16 * RP * WR;
  constexpr uint32_t kCodes = RT * 128, kColumns = XC * 32;  // chunks of a stage
  constexpr int JW = kCodes / 64, JX = kColumns / G, N = JX + (kDma > 0 ? JW : 0) + (kDma == 2 ? 1 : 0);
  static_assert(kColumns % G == 0 && (NS - 2) * N < 64, "whole requests, and a wait that counts them");
  __shared__ u32x4 columns[KG * NS * kColumns], codes[KG * WR * NS * kCodes];
  __shared__ uint32_t scales[KG * WR * NS * 64];
  __shared__ int32_t list[kAll ? 2 * kMoeMaxTopK : 1];  // the experts that take part and their slots
  const MxMoeArgs& a = m.a;
  const uint32_t lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t group = wave / WR, wr = wave % WR, gi = wr * 64 + lane;
  const uint32_t rows = INNER ? a.inner : a.cols, length = INNER ? a.cols : a.inner, blocks = length / kMxBlock;
  const uint32_t x_len = INNER ? m.p.x_len : m.p.h_len, steps = x_len / kStep;
  const uint32_t tiles = ((INNER ? m.p.h_len : rows) + kRows - 1) / kRows;
  const uint32_t slot = blockIdx.x / tiles, n0 = blockIdx.x % tiles * kRows;
  const uint32_t parts = INNER ? parts_of(a.x_type) : inner_parts(a.out_type);
  // the expert and its tokens
  Active item{0, 0, 1, 0};
  uint32_t units = steps;
  uint32_t experts = 0;  // that take part (kAll); lane k holds the k-th and its slot
  int32_t expert_k = 0, slot_k = 0;
  if constexpr (kAll) {
    const int32_t e = lane < a.top_k ? g_ld<int32_t>(m.p.chosen + lane * 4) : -1;
    const uint64_t in = __ballot(e >= 0);
    experts = __popcll(in);
    const uint32_t k = __popcll(in & ((1ull << lane) - 1));
    if (e >= 0) list[2 * k] = e, list[2 * k + 1] = (int32_t)lane;  // the same by every wavefront
    __syncthreads();
    if (lane < experts) expert_k = list[2 * lane], slot_k = list[2 * lane + 1];
    units = experts * steps;
  } else if constexpr (ONE) {
    if (slot + 1 == a.top_k && n0 == 0) {
      // of all wavefronts that choose, these also write the choice
      const Chosen c = choose(m, 0);
      item.expert = (uint32_t)__builtin_amdgcn_readlane((int)c.expert, (int)slot);
      if (__builtin_amdgcn_readlane((int)c.masked, (int)slot)) return;
    } else {
      Choice c(m, 0);
      for (uint32_t k = 0; k <= slot; ++k) item.expert = c.next(a.experts);
      if (logit_of(c.best) == -__builtin_inf()) return;
    }
    item.first = slot;
  } else {
    if (slot >= g_ld<uint32_t>(m.p.actives)) return;
    const u32x4 v = ld16(m.p.active + (uint64_t)slot * sizeof(Active));
    item = Active{v[0], v[1], v[2], 0};
  }
  const uint32_t e0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)item.expert);
  const uint32_t first = (uint32_t)__builtin_amdgcn_readfirstlane((int)item.first);
  const uint32_t count = (uint32_t)__builtin_amdgcn_readfirstlane((int)item.count);

  // Rows past the last one take its place; their sums are not stored, or as zeros.
  uint64_t w_at[JW], s_at;
  auto matrix = [&](int r) -> const MxExperts& { return INNER ? (r ? a.up : a.gate) : a.down; };
  auto row_of = [&](int r, uint32_t in) { return min(n0 + (wr * RP + (INNER ? 0 : r)) * 16 + in, rows - 1); };
#pragma unroll
  for (int j = 0; j < JW; ++j) {
    const MxExperts& w = matrix(j / 2);
    w_at[j] = w.codes.ptr + (kAll ? 0 : e0 * w.codes_expert) + row_of(j / 2, j % 2 * 8 + lane / 8) * w.codes.stride;
  }
  {
    const int r = RT == 2 && lane >= 32;
    const uint32_t n = row_of(r, lane / 2 % 16);
    s_at = r == 0 ? matrix(0).scales.ptr + (kAll ? 0 : e0 * matrix(0).scales_expert) + n * matrix(0).scales.stride
                  : matrix(1).scales.ptr + (kAll ? 0 : e0 * matrix(1).scales_expert) + n * matrix(1).scales.stride;
  }
  uint64_t byte_at[RT];  // of the lane's row, for scales by the byte
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const MxExperts& w = matrix(r);
    byte_at[r] = w.scales.ptr + (kAll ? 0 : e0 * w.scales_expert) + row_of(r, i) * w.scales.stride;
  }
  const uint32_t columns_at = lds_address(columns) + group * (NS * kColumns * 16);
  const uint32_t codes_at = lds_address(codes) + wave * (NS * kCodes * 16);
  const uint32_t words_at = lds_address(scales) + wave * (NS * 64 * 4);

  const uint32_t each = CW / parts;  // tokens of a group of columns
  for (uint32_t t0 = 0; t0 < count; t0 += each * NC) {
    const uint32_t tokens = min(count - t0, each * NC);
    // A lane's chunks of the columns: column c holds part c % parts of a token; columns without one repeat the first.
    uint64_t x_at[JX];
#pragma unroll
    for (int j = 0; j < JX; ++j) {
      const uint32_t column = (j * G + gi) / 32, c = column % CW;
      uint32_t t = column / CW * each + c / parts, part = c % parts;
      if (c >= each * parts || t >= tokens) t = 0, part = 0;
      uint64_t row = first + t0 + t;
      if constexpr (INNER) row = ONE ? 0 : (uint32_t)g_ld<int32_t>(m.p.order + row * 4) / a.top_k;
      const uint32_t chunk = (gi & 31) ^ (column & 15);
      x_at[j] = (INNER ? m.p.x + (part * a.tokens + row) * x_len * 2
                       : m.p.h + (part * a.tokens * a.top_k + (kAll ? 0 : row)) * x_len * 2) + chunk * 16;
    }
    // Where along its way a group is: a step, of the k-th expert.
    struct Unit {
      uint32_t step, k;
    };
    auto forward = [&](Unit& u) {
      u.step += KG;
      while (kAll && u.step >= steps) u.step -= steps, ++u.k;
    };
    auto expert_of = [&](const Unit& u) { return (uint64_t)(uint32_t)__builtin_amdgcn_readlane(expert_k, (int)u.k); };
    auto slot_of = [&](const Unit& u) { return (uint32_t)__builtin_amdgcn_readlane(slot_k, (int)u.k); };
    auto request = [&](const Unit& u, uint32_t stage) {
      const uint64_t e = kAll ? expert_of(u) : 0;
#pragma unroll
      for (int j = 0; j < JW; ++j) {
        const uint32_t chunk = (lane & 7) ^ (j * 4 + (lane >> 4) & 7);
        const uint64_t from = w_at[j] + e * a.down.codes_expert + min(u.step * 8 + chunk, blocks - 1) * 16;
        if constexpr (kDma > 0)
          dma16(from, codes_at + (stage * kCodes + j * 64) * 16);
        else
          ((LdsChunks)(codes_at + (stage * kCodes + lane) * 16))[j * 64] = ld16(from);
      }
      if constexpr (kDma == 2)
        dma4(s_at + e * a.down.scales_expert + min(u.step * 2 + (lane & 1), blocks / 4 - 1) * 4,
             words_at + stage * 256);
#pragma unroll
      for (int j = 0; j < JX; ++j)
        dma16(x_at[j] + (kAll ? (uint64_t)slot_of(u) * x_len * 2 : 0) + u.step * (kStep * 2),
              columns_at + (stage * kColumns + j * G + wr * 64) * 16);
    };
    uint32_t bytes[RT][2] = {}, bytes_next[RT][2] = {};
    auto load_bytes = [&](const Unit& u) {
      const uint64_t e = kAll ? expert_of(u) : 0;
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int s = 0; s < 2; ++s)
          bytes_next[r][s] = g_ld<uint8_t>(byte_at[r] + e * a.down.scales_expert +
                                           min(u.step * 8 + s * 4 + q, blocks - 1));
    };
    f32x4 acc[RT][NC] = {}, total[kAll ? RT : 1][NC] = {};
    auto compute = [&](uint32_t stage) {
      u32x2 words[RT];
      if constexpr (kDma == 2) {
#pragma unroll
        for (int r = 0; r < RT; ++r) words[r] = *(LdsPairs)(words_at + stage * 256 + (r * 16 + i) * 8);
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        u32x4 wv[RT];
        float sf[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const uint32_t row = r * 16 + i, c = s * 4 + q;
          wv[r] = *(LdsChunks)(codes_at + (stage * kCodes + row * 8 + (c ^ (row / 2 & 7))) * 16);
          sf[r] = scale_f32(kDma == 2 ? words[r][s] >> 8 * q & 0xFF : bytes[r][s]);
        }
#pragma unroll
        for (int f = 0; f < 4; ++f) {
          u32x4 xv[NC];
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            const uint32_t column = c * 16 + i % CW, chunk = (s * 4 + q) * 4 + f;
            xv[c] = *(LdsChunks)(columns_at + (stage * kColumns + column * 32 + (chunk ^ (column & 15))) * 16);
          }
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            const u32x4 w8 = weights8(wv[r][f], sf[r]);
#pragma unroll
            for (int c = 0; c < NC; ++c) acc[r][c] = mfma(w8, xv[c], acc[r][c]);
          }
        }
      }
    };
    auto add_expert = [&](uint32_t k) {  // an expert's sums, weighted
      const float weight = g_ld<float>(m.p.weights + k * 4);
#pragma unroll
      for (int r = 0; r < (kAll ? RT : 1); ++r)
#pragma unroll
        for (int c = 0; c < NC; ++c) total[r][c] += weight * acc[r][c], acc[r][c] = f32x4{};
    };
    const uint32_t n = group < units ? (units - group + KG - 1) / KG : 0;  // of this group
    if (t0) __syncthreads();  // before LDS is used again
    if (n) {
      Unit now{group, 0};
      while (kAll && now.step >= steps) now.step -= steps, ++now.k;
      if constexpr (kDma < 2) load_bytes(now);
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
        if constexpr (kDma < 2) {
#pragma unroll
          for (int r = 0; r < RT; ++r) bytes[r][0] = bytes_next[r][0], bytes[r][1] = bytes_next[r][1];
          if (k + 1 < n) load_bytes(next);
        }
        if (k + NS - 1 < n) {
          request(ahead, into);
          forward(ahead);
        }
        compute(stage);
        if constexpr (kAll) {
          if (k + 1 == n || next.k != now.k) add_expert(slot_of(now));
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
      for (int c = 0; c < NC; ++c) sums[((wave * RT + r) * NC + c) * 64 + lane] = kAll ? total[kAll ? r : 0][c] : acc[r][c];
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
    for (uint32_t at = threadIdx.x; at < tokens * kRows; at += 64 * WR * KG) {
      const uint32_t t = at / kRows, in = at % kRows, w = in / (16 * RP), rp = in / 16 % RP, nn = n0 + in;
      const uint64_t row = first + t0 + t;
      if constexpr (INNER) {
        if (nn >= m.p.h_len) continue;
        float h = 0;
        if (nn < a.inner) {
          const float g = sum_of(w, 0, in % 16, t) + bias_of(a.gate, a.out_type, e0, nn);
          const float u = sum_of(w, 1, in % 16, t) + bias_of(a.up, a.out_type, e0, nn);
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
          g_st<uint16_t>(m.p.h + ((p * a.tokens * a.top_k + row) * m.p.h_len + nn) * 2, b);
        }
      } else if (nn < rows) {
        float v = sum_of(w, rp, in % 16, t);
        if constexpr (kAll) {
          for (uint32_t k = 0; a.down.bias && k < experts; ++k)
            v += g_ld<float>(m.p.weights + list[2 * k + 1] * 4) * bias_of(a.down, a.out_type, (uint32_t)list[2 * k], nn);
          store1_as(a.out_type, a.out.ptr, nn, v);
        } else {
          g_st<float>(m.p.y + (row * rows + nn) * 4, v + bias_of(a.down, a.out_type, e0, nn));
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
  for (uint32_t k = 0; k < a.top_k; ++k) {
    const uint64_t pair = (uint64_t)t * a.top_k + k;
    const int32_t row = g_ld<int32_t>(m.p.place + pair * 4);
    if (row >= 0) v += g_ld<float>(m.p.weights + pair * 4) * __builtin_bit_cast(f32x4, ld16(m.p.y + ((uint64_t)row * a.cols + n) * 4));
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

template <bool INNER, bool ONE, int WR, int KG, int XC, int NS>
hipError_t product_of(const MoeArgs& m, int dma, hipStream_t stream) {
  constexpr uint32_t kRows = 16 * (INNER || ONE ? 1 : 2) * WR;
  const uint64_t tiles = ((INNER ? m.p.h_len : m.a.cols) + kRows - 1) / kRows, pairs = m.a.tokens * m.a.top_k;
  const uint64_t items = ONE ? (INNER ? m.a.top_k : 1) : pairs < m.a.experts ? pairs : m.a.experts;
  return launch(dma == 2   ? moe_product_kernel<INNER, ONE, WR, KG, XC, NS, 2>
                : dma == 1 ? moe_product_kernel<INNER, ONE, WR, KG, XC, NS, 1>
                           : moe_product_kernel<INNER, ONE, WR, KG, XC, NS, 0>,
                items * tiles, 64 * WR * KG, m, stream);
}

hipError_t logits_of(const MoeArgs& m, hipStream_t stream) {
  const uint64_t groups = m.a.experts * ((m.a.tokens + kLogitTokens - 1) / kLogitTokens) + m.a.tokens;
  switch (m.a.x_type) {
    case kTypeF32: return launch(moe_logits_kernel<kTypeF32>, groups, 256, m, stream);
    case kTypeF16: return launch(moe_logits_kernel<kTypeF16>, groups, 256, m, stream);
    case kTypeBf16: return launch(moe_logits_kernel<kTypeBf16>, groups, 256, m, stream);
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
    if (tokens == 1) {
      if (e == hipSuccess) e = product_of<true, true, 1, 4, 4, 3>(m, inner, stream);
      if (e == hipSuccess) e = product_of<false, true, 1, 8, 4, 4>(m, outer, stream);
      return e;
    }
    if (e == hipSuccess) e = launch(moe_route_kernel, 1, 1024, m, stream);
    if (e == hipSuccess) e = product_of<true, false, 4, 1, 16, 3>(m, inner, stream);
    if (e == hipSuccess) e = product_of<false, false, 4, 1, 16, 3>(m, outer, stream);
    if (e == hipSuccess) e = launch(moe_combine_kernel, (tokens * (a.cols / 4) + 255) / 256, 256, m, stream);
    return e;
  });
}

}  // namespace ptwm
