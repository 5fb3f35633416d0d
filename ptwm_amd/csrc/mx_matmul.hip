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

#include <type_traits>

#include "mx_choice.h"
#include "mx_device.h"

namespace ptwm {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// 16 weight rows and 16 tokens, 128 values of each: lane l holds row (token) l % 16 and block l / 16, and its scale.
__device__ __forceinline__ f32x4 mfma_mx4(u32x4 w, uint32_t ws, u32x4 x, uint32_t xs, f32x4 c) {
  const i32x8 wv = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
  const i32x8 xv = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, xv, c, 4, 4, 0, (int)ws, 0, (int)xs);
}

// Small products, and rows too far apart for a tile's 32-bit offsets: a 16x16
// tile of outputs by one workgroup, whose wavefronts take turns in steps of 128
// values along the rows and add up in LDS, operands straight from memory; bound
// by one way to memory (16x4096x256 2.4 us).
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

// 32 weight rows and 32 tokens, 64 values of each: lane l holds row (token) l % 32 and block l / 32.  OP: the byte of the
// words of scales.
template <int OP>
__device__ __forceinline__ f32x16 mfma_mx4_32(u32x4 w, uint32_t ws, u32x4 x, uint32_t xs, f32x16 c) {
  const i32x8 wv = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
  const i32x8 xv = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wv, xv, c, 4, 4, OP, (int)ws, OP, (int)xs);
}

// The scale bytes of a row of `blocks` blocks from block `first` on, 16 of them, and zeros past its end.  Without a branch
// where there are 16 at all: the last 16 are loaded, in parts() moved to the front.
struct Scales16 {
  u32x4 v;
  __device__ __forceinline__ void load(uint64_t row, uint32_t first, uint32_t blocks) {
    v = ld16(row + min(first, blocks - 16));
  }
  __device__ __forceinline__ void gather(uint64_t row, uint32_t blocks) {  // of a row of fewer, byte by byte
    v = u32x4{};
    for (uint32_t k = 0; k < blocks; ++k) {
      const uint32_t byte = (uint32_t)g_ld<uint8_t>(row + k) << 8 * (k & 3);
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) v[j] |= k / 4 == j ? byte : 0;
    }
  }
  __device__ __forceinline__ u32x4 from(uint32_t first, uint32_t blocks) const {
    const uint32_t skip = first + 16 > blocks && blocks >= 16 ? first + 16 - blocks : 0;
    u32x4 w = v;
    w = skip & 8 ? u32x4{w[2], w[3], 0, 0} : w;
    w = skip & 4 ? u32x4{w[1], w[2], w[3], 0} : w;
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = __builtin_amdgcn_alignbyte(k < 3 ? w[k + 1 < 4 ? k + 1 : 3] : 0u, w[k], skip & 3);
    return w;
  }
};

// A tile of 32 * RT * WR weight rows and 32 * CT * WC tokens by one workgroup
// of WR * WC * KG wavefronts: a wavefront holds the sums of RT x CT squares of
// 32, WR x WC of them share the operands, and KG groups take turns in quads of
// 512 values along the rows and add up in LDS at the end.
//
// Both operands go through LDS by DMA, in steps of 256 values: 128 bytes of a
// row, a cache line where rows lie at multiples of it.  There are NS stages,
// each requested again as soon as all have read the step before it there.  A
// row's eight 16-byte chunks lie at chunk ^ (row / 2 % 8), so the 16 lanes that
// read a chunk of 16 rows at a time meet every bank once.  A product takes 64
// values: lane l holds of a row the blocks of even (l < 32) or odd number.  The
// operands of a product are read while the one before it runs.
//
// The scales of a quad are 16 bytes of a row.  Where these lie at multiples of
// 16 they take the codes' way (kDma 2); elsewhere a thread loads them a quad
// ahead and hands them on through LDS, which waits for all that is on its way
// once a quad.  Codes that do not lie at multiples of 16 bytes (kDma 0) go
// through registers to the same places, so results do not depend on how
// operands lie.  Offsets within a tile are 32 bits on top of uniform addresses.
//
// What bounds the largest tile, 256 x 256 by 2 x 4 wavefronts, is the clock
// under full load, and then waits within the tile.  2048x8192x4096, a tile a
// CU: 32768 cycles of the matrix unit within 57000 to 65000 (48000 to 55000 in
// the loop, the rest for the first bytes and the stores), at 1.8 GHz in a
// launch alone and 1.3 to 1.6 GHz in launches one after the other (2.3 with a
// single tile at work): 37 to 43 us, 38 without any request to memory.  While
// the matrix unit is busy, LDS gives 96 of its 128 bytes a cycle and takes the
// requests' 32.  Steps of 64 bytes of a row instead of 128 took every cache
// line twice: 2048x14336x4096 86 us, 77 this way.  Smaller tiles are bound by
// the way to memory; four stages shorten it (128x14336x4096, 128 x 64 tiles:
// 13.7 us with two stages, 10.7 with four).
template <int RT, int CT, int WR, int WC, int KG, int NS, int kDma>
__global__ __launch_bounds__(64 * WR * WC * KG, 1) void mxfp4_matmul_tiles_kernel(MxLinearArgs a) {
  static_assert(KG == 1 || WR * WC == 1, "groups of several wavefronts meet at barriers of the whole workgroup");
  constexpr uint32_t R = 32 * RT * WR, T = 32 * CT * WC, G = 64 * WR * WC;
  constexpr uint32_t kStage = (R + T) * 8;       // 16-byte chunks of a step
  constexpr int J = kStage / G, JR = R * 8 / G;  // a thread's chunks of a step, of them the weights'
  constexpr int SE = (R + T + G - 1) / G;        // rows whose scales a thread loads
  constexpr int NQ = NS / 2 + 1;                 // quads whose scales are held
  static_assert(NS == 2 || NS == 4, "whole quads of two steps");
  static_assert(R * 8 % G == 0 && kStage % G == 0, "a load is of one operand");
  __shared__ u32x4 stages[KG * NS * kStage];
  __shared__ u32x4 scales[KG * NQ * SE * G];
  __shared__ float bias[KG == 1 ? R : 1];  // of the tile, in 32 bits
  const uint32_t lane = threadIdx.x & 63, h = lane >> 5, i = lane & 31;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t group = wave / (WR * WC), wr = wave % (WR * WC) / WC, wc = wave % WC;
  const uint32_t gw = wave % (WR * WC) * 64, gi = gw + lane;  // a thread of its group
  // Tiles one after the other share their weights; each of the eight chiplets takes a run of them, for its own cache.
  const uint32_t row_tiles = (a.rows + R - 1) / R, token_tiles = (uint32_t)((a.tokens + T - 1) / T);
  const uint32_t all = row_tiles * token_tiles, part = all / 8, more = all % 8;
  const uint32_t chiplet = blockIdx.x % 8, turn = blockIdx.x / 8;
  const uint32_t tile = chiplet * part + min(chiplet, more) + turn;
  const uint32_t n0 = tile / token_tiles * R;
  const uint64_t t0 = (uint64_t)(tile % token_tiles) * T;
  const uint32_t rows = min(a.rows - n0, R), tokens = (uint32_t)min(a.tokens - t0, (uint64_t)T);
  const uint32_t blocks = a.cols / kMxBlock, quads = (blocks + 15) / 16;
  // rows and tokens past the last one take the last one's place and are not stored
  const GlobalBytes w0 = uniform(a.weight.ptr + n0 * a.weight.stride), x0 = uniform(a.x.ptr + t0 * a.x.stride);
  const uint64_t ws0 = a.scales.ptr + n0 * a.scales.stride, xs0 = a.x_scales.ptr + t0 * a.x_scales.stride;
  uint32_t at[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const uint32_t t = (j * G + gi) / 8;
    at[j] = j < JR ? min(t, rows - 1) * (uint32_t)a.weight.stride : min(t - R, tokens - 1) * (uint32_t)a.x.stride;
  }
  uint64_t scales_at[SE];
#pragma unroll
  for (int k = 0; k < SE; ++k) {
    const uint32_t t = min(k * G + gi, R + T - 1);
    scales_at[k] = t < R ? ws0 + min(t, rows - 1) * a.scales.stride : xs0 + min(t - R, tokens - 1) * a.x_scales.stride;
  }
  // the group's parts of LDS, by their addresses
  const uint32_t own_stages = lds_address(stages) + group * (NS * kStage * 16);
  const uint32_t own_scales = lds_address(scales) + group * (NQ * SE * G * 16);
  u32x4 held[J];  // on their way through registers
  // Requests step d of a quad; past the row's end its last block again.
  auto request = [&](uint32_t quad, int d, uint32_t slot, int from, int to) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (j < from || j >= to) continue;
      const uint32_t chunk = (gi & 7) ^ ((gi >> 4) + j * (G / 16) & 7);
      const uint32_t offset = at[j] + min(quad * 16 + d * 8 + chunk, blocks - 1) * 16;
      const GlobalBytes p = j < JR ? w0 : x0;
      if constexpr (kDma > 0)
        dma16(p, offset, own_stages + (slot * kStage + j * G + gw) * 16);
      else
        held[j] = ld16(p, offset);
    }
  };
  auto store = [&](uint32_t slot) {
    if constexpr (kDma == 0) {
#pragma unroll
      for (int j = 0; j < J; ++j) ((LdsChunks)(own_stages + (slot * kStage + gi) * 16))[j * G] = held[j];
    }
  };
  Scales16 loaded[SE];
  auto load_scales = [&](uint32_t quad) {
#pragma unroll
    for (int k = 0; k < SE; ++k) loaded[k].load(scales_at[k], quad * 16, blocks);
  };
  auto store_scales = [&](uint32_t quad, uint32_t slot) {
#pragma unroll
    for (int k = 0; k < SE; ++k)
      ((LdsChunks)(own_scales + (slot * SE * G + gi) * 16))[k * G] = loaded[k].from(quad * 16, blocks);
  };
  auto request_scales = [&](uint32_t quad, uint32_t slot) {
#pragma unroll
    for (int k = 0; k < SE; ++k) dma16(scales_at[k] + quad * 16, own_scales + (slot * SE * G + k * G + gw) * 16);
  };
  // scales of a step and of the next one: words of four blocks, the lane's in bytes 0 and 2
  u32x2 ws[2][RT], xs[2][CT];
  auto read_scales = [&](int d, uint32_t slot) {
    const LdsPairs w = (LdsPairs)(own_scales + slot * (SE * G * 16) + (wr * RT * 32 + i) * 16 + d * 8);
    const LdsPairs x = (LdsPairs)(own_scales + slot * (SE * G * 16) + (R + wc * CT * 32 + i) * 16 + d * 8);
#pragma unroll
    for (int r = 0; r < RT; ++r) ws[d][r] = w[r * 64];
#pragma unroll
    for (int c = 0; c < CT; ++c) xs[d][c] = x[c * 64];
  };
  auto turn_scales = [&](int d) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int r = 0; r < RT; ++r) ws[d][r][k] >>= 8 * h;
#pragma unroll
      for (int c = 0; c < CT; ++c) xs[d][c][k] >>= 8 * h;
    }
  };
  // What the wavefront wrote, and all that it requested but for the newest `requests`, is there, and all have come.
  auto meet = [&](auto requests) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((int)requests) : "memory");
    if constexpr (WR * WC > 1)
      __builtin_amdgcn_s_barrier();
    else
      __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
  };
  u32x4 wv[2][RT], xv[2][CT];
  // addresses of the chunks of product q in the first of the wavefront's rows and tokens
  uint32_t w_read[4], x_read[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint32_t chunk = (2 * q + h) ^ (i >> 1 & 7);
    w_read[q] = own_stages + ((wr * RT * 32 + i) * 8 + chunk) * 16;
    x_read[q] = own_stages + ((R + wc * CT * 32 + i) * 8 + chunk) * 16;
  }
  auto read = [&](uint32_t slot, int q, int k) {  // operand k of product q of a step, what is used first first
    if (k < CT)
      xv[q & 1][k] = ((LdsChunks)(x_read[q] + slot * (kStage * 16)))[k * 256];
    else
      wv[q & 1][k - CT] = ((LdsChunks)(w_read[q] + slot * (kStage * 16)))[(k - CT) * 256];
  };
  f32x16 acc[RT][CT] = {};
  // Where the pipeline is: the step's and the next one's stages, the quad's and the next one's scales, the stage's
  // next quad.
  struct Place {
    uint32_t quad, later;         // of this step, of the step NS steps on
    uint32_t slot, next;          // stages
    uint32_t scales, scales_next;  // of this quad and the next one
  };
  // `left`: steps that are left from this one on where they are few, 0: more than NS.  Of the last two a row's end may
  // cut blocks off.
  auto product = [&](auto d_, auto q_, const Place& p, auto left) {
    constexpr int d = d_, q = q_, kNext = (q + 1) & 3;
    constexpr bool kEnd = left == 1 && q == 3;
    // two stages alternate with the steps of a quad
    const uint32_t slot = NS == 2 ? d : p.slot, next = NS == 2 ? d ^ 1 : p.next;
    if constexpr (kDma < 2 && (left == 1 || left == 2)) {
      const uint32_t keep = p.quad * 16 + d * 8 + 2 * q + h < blocks ? ~0u : 0u;
#pragma unroll
      for (int r = 0; r < RT; ++r) wv[q & 1][r] &= keep;
    }
    if constexpr (q == 3 && !kEnd) read_scales(d ^ 1, d ? p.scales_next : p.scales);
    if constexpr (q == 3 && left == 0 && kDma == 2 && ((d + NS) & 1) == 0) {
      // of the quad that starts NS steps on, in place of the one before this one
      request_scales(p.later, p.scales ? p.scales - 1 : NQ - 1);
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      if constexpr (!kEnd) {
#pragma unroll
        for (int k = r * (RT + CT) / RT; k < (r + 1) * (RT + CT) / RT; ++k) read(q == 3 ? next : slot, kNext, k);
      }
      if constexpr (q == 3 && left == 0) request(p.later, (d + NS) & 1, slot, r * J / RT, (r + 1) * J / RT);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int c = 0; c < CT; ++c)
        acc[r][c] = mfma_mx4_32<2 * (q & 1)>(wv[q & 1][r], ws[d][r][q / 2], xv[q & 1][c], xs[d][c][q / 2], acc[r][c]);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (q == 3 && !kEnd) turn_scales(d ^ 1);
  };
  // requests of the steps `from` to `to` - 1 after this one
  auto requests = [](int d, int from, int to) constexpr {
    int n = 0;
    for (int k = from; k < to; ++k) n += J + (kDma == 2 && ((d + k) & 1) == 0 ? SE : 0);
    return n;
  };
  auto step = [&](auto d_, Place& p, auto left) {
    constexpr int d = d_;
    product(d_, std::integral_constant<int, 0>{}, p, left);
    product(d_, std::integral_constant<int, 1>{}, p, left);
    product(d_, std::integral_constant<int, 2>{}, p, left);
    if constexpr (left != 1) {
      if constexpr (left == 0 || left == NS) store(NS == 2 ? d ^ 1 : p.slot ? p.slot - 1 : NS - 1);  // requested a step ago
      if constexpr (kDma < 2 && d == 1) store_scales(p.quad + KG, p.scales_next);
      meet(std::integral_constant<int, kDma == 0 ? 0 : requests(d, 2, left ? left : NS)>{});
      if constexpr (kDma < 2 && d == 0 && left != 2) load_scales(p.quad + KG);
    }
    product(d_, std::integral_constant<int, 3>{}, p, left);
    p.slot = p.next, p.next = p.next + 1 == NS ? 0 : p.next + 1;
    if constexpr (d == 1) {
      p.quad += KG, p.later += KG;
      p.scales = p.scales_next, p.scales_next = p.scales_next + 1 == NQ ? 0 : p.scales_next + 1;
    }
  };
  auto pair = [&](Place& p, auto left) {
    step(std::integral_constant<int, 0>{}, p, left);
    step(std::integral_constant<int, 1>{}, p, std::integral_constant<int, left ? left - 1 : 0>{});
  };
  if (KG == 1 || group < quads) {
    uint32_t n = (quads - group + KG - 1) / KG;  // quads of this group
    if constexpr (kDma < 2) {
      if (blocks >= 16) {
        load_scales(group);
      } else {
#pragma unroll
        for (int k = 0; k < SE; ++k) loaded[k].gather(scales_at[k], blocks);
      }
    }
#pragma unroll
    for (int k = 0; k < NS; ++k) {
      if (k >= 2 && (uint32_t)k / 2 >= n) break;
      if constexpr (kDma == 2) {
        if (k % 2 == 0) request_scales(group + k / 2 * KG, k / 2);
      }
      request(group + k / 2 * KG, k & 1, k, 0, J);
      if (k < NS - 1) store(k);
    }
    if constexpr (kDma < 2) store_scales(group, 0);
    if (kDma > 0 && 2 * n >= NS)
      meet(std::integral_constant<int, requests(0, 1, NS)>{});
    else
      meet(std::integral_constant<int, 0>{});
    Place p{group, group + NS / 2 * KG, 0, 1, 0, 1};
    read_scales(0, 0);
#pragma unroll
    for (int k = 0; k < RT + CT; ++k) read(0, 0, k);
    turn_scales(0);
    for (; n > NS / 2; --n) pair(p, std::integral_constant<int, 0>{});
    if constexpr (NS == 4) {
      if (n == 2) pair(p, std::integral_constant<int, 4>{});
    }
    pair(p, std::integral_constant<int, 2>{});
  }

  // lane l holds token l % 32 and rows 8 j + 4 (l / 32) .. + 3, j = 0 .. 3
  auto quad_of = [&](int r, int c, int j) {
    return f32x4{acc[r][c][4 * j], acc[r][c][4 * j + 1], acc[r][c][4 * j + 2], acc[r][c][4 * j + 3]};
  };
  const uint64_t tw = t0 + wc * CT * 32;
  const uint32_t nw = n0 + wr * RT * 32;
  if constexpr (KG == 1) {
    __syncthreads();
    if (a.bias) {
      for (uint32_t k = threadIdx.x; k < R; k += G) {
        const uint32_t n = min(n0 + k, a.rows - 1);
        bias[k] = a.out_type == kTypeBf16  ? load1<kTypeBf16>(a.bias + (uint64_t)n * 2)
                  : a.out_type == kTypeF16 ? load1<kTypeF16>(a.bias + (uint64_t)n * 2)
                                           : load1<kTypeF32>(a.bias + (uint64_t)n * 4);
      }
      __syncthreads();
    }
    // Through LDS, so that consecutive lanes store a token's outputs, and not a lane 8 or 16 bytes of them.
    u32x4* const turn = stages + wave * 32 * RT * 4;
    constexpr uint32_t kRow = RT * 4;  // chunks of a token and pass
    static_assert(WR * WC * 32 * kRow <= NS * kStage, "the stages hold a pass of all wavefronts");
    auto rows_first = [&](auto type) {
      constexpr uint32_t OT = type;
      constexpr int P = OT == kTypeF32 ? 2 : 1, RP = RT / P;  // passes over the rows of a column of tokens
#pragma unroll
      for (int pass = 0; pass < CT * P; ++pass) {
        const int c = pass / P, r0 = pass % P * RP;
#pragma unroll
        for (int r = 0; r < RP; ++r)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            f32x4 v = quad_of(r0 + r, c, j);
            if (a.bias) v += *reinterpret_cast<const f32x4*>(bias + (wr * RT + r0 + r) * 32 + j * 8 + h * 4);
            if constexpr (OT == kTypeF32) {
              turn[i * kRow + ((r * 8 + 2 * j + h) ^ (i & (kRow - 1)))] = __builtin_bit_cast(u32x4, v);
            } else {
              const uint64_t two = pack2<OT>(v[0], v[1]) | (uint64_t)pack2<OT>(v[2], v[3]) << 32;
              reinterpret_cast<uint64_t*>(turn)[2 * (i * kRow + ((r * 4 + j) ^ (i & (kRow - 1)))) + h] = two;
            }
          }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // other lanes' values
#pragma unroll
        for (uint32_t k = 0; k < 32 * kRow / 64; ++k) {
          const uint32_t t = (k * 64 + lane) / kRow, q = lane % kRow;
          const u32x4 v = turn[t * kRow + (q ^ (t & (kRow - 1)))];
          const uint64_t to = tw + c * 32 + t;
          constexpr uint32_t kEach = 16 / type_bytes(OT);
          const uint32_t n = nw + r0 * 32 + q * kEach;
          const uint64_t at = a.out.ptr + (to * a.out.stride + n) * type_bytes(OT);
          if (to >= a.tokens || n >= a.rows) continue;
          if (n + kEach <= a.rows) {
            st16(at, v);
          } else {
#pragma unroll
            for (uint32_t k = 0; k < kEach; ++k) {
              if (n + k >= a.rows) break;
              if constexpr (OT == kTypeF32)
                g_st<uint32_t>(at + 4 * k, v[k]);
              else
                g_st<uint16_t>(at + 2 * k, (uint16_t)(v[k / 2] >> 16 * (k & 1)));
            }
          }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // before the next pass writes there
      }
    };
    if (a.out_type == kTypeBf16)
      rows_first(std::integral_constant<uint32_t, kTypeBf16>{});
    else if (a.out_type == kTypeF16)
      rows_first(std::integral_constant<uint32_t, kTypeF16>{});
    else
      rows_first(std::integral_constant<uint32_t, kTypeF32>{});
  } else {
    // the groups' sums take the place of the stages, in the order of the groups
    constexpr int kQuads = RT * CT * 4;
    constexpr uint32_t kFit = kStage / 64;
    static_assert(kQuads <= NS * kFit, "the stages hold the sums");
    __syncthreads();
#pragma unroll
    for (uint32_t q = 0; q < kQuads; ++q)
      stages[group * NS * kStage + q * 64 + lane] = __builtin_bit_cast(u32x4, quad_of(q / (CT * 4), q / 4 % CT, q % 4));
    __syncthreads();
    for (uint32_t q = wave; q < kQuads; q += KG) {
      f32x4 v = {};
#pragma unroll
      for (int g = 0; g < KG; ++g) v += __builtin_bit_cast(f32x4, stages[g * NS * kStage + q * 64 + lane]);
      const uint64_t t = t0 + q / 4 % CT * 32 + i;
      const uint32_t n = n0 + q / (CT * 4) * 32 + q % 4 * 8 + h * 4;
      if (t < a.tokens && n < a.rows) store4(a, t, n, v);
    }
  }
}

template <int RT, int CT, int WR, int WC, int KG, int NS>
hipError_t tiles_of(const MxLinearArgs& a, int dma, hipStream_t stream) {
  return launch_tiles<1, 32 * RT * WR, 32 * CT * WC>(dma == 2   ? mxfp4_matmul_tiles_kernel<RT, CT, WR, WC, KG, NS, 2>
                                                     : dma == 1 ? mxfp4_matmul_tiles_kernel<RT, CT, WR, WC, KG, NS, 1>
                                                                : mxfp4_matmul_tiles_kernel<RT, CT, WR, WC, KG, NS, 0>,
                                                     64 * WR * WC * KG, a, stream);
}

}  // namespace

hipError_t launch_mxfp4_matmul(const MxLinearArgs& a, hipStream_t stream) {
  const MxMatmulChoice k = choose_mxfp4_matmul(a);
  switch (k.kind) {
    case MxMatmulChoice::k256x256: return tiles_of<4, 2, 2, 4, 1, 2>(a, k.dma, stream);
    case MxMatmulChoice::k256x128: return tiles_of<2, 2, 4, 2, 1, 2>(a, k.dma, stream);
    case MxMatmulChoice::k128x128: return tiles_of<2, 1, 2, 4, 1, 4>(a, k.dma, stream);
    case MxMatmulChoice::k128x64: return tiles_of<2, 1, 2, 2, 1, 4>(a, k.dma, stream);
    case MxMatmulChoice::k64x64: return tiles_of<2, 1, 1, 2, 1, 4>(a, k.dma, stream);
    case MxMatmulChoice::k32x32by8: return tiles_of<1, 1, 1, 1, 8, 2>(a, k.dma, stream);
    case MxMatmulChoice::k32x32by4: return tiles_of<1, 1, 1, 1, 4, 2>(a, k.dma, stream);
    default: return launch_tiles<1, 16, 16>(mxfp4_matmul_kernel, 256, a, stream);
  }
}

}  // namespace ptwm
