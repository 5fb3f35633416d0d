// mx_choice.h -- which kernel takes a product with MXFP4 weights, of two MXFP4
// matrices, and the products of a mixture-of-experts layer: rules on sizes,
// types and alignment, on the host.  The times beside them are microseconds on
// an MI355X.
#pragma once

#include "mx_ops.h"

namespace ptwm {

struct MxLinearChoice {
  enum Kind : uint32_t { kSmall, kFew, kTiles } kind;
  uint32_t tokens;        // kFew: up to this many
  uint32_t rows, ct;      // kTiles: rows of a wavefront, 32-token columns of a tile,
  uint32_t rg, kg;        // groups of rows, groups that share the length of the rows
  bool aligned;           // what goes to LDS as it is lies at multiples of 16 bytes
};

// LDS that the few tokens' kernel takes: nt tokens in 32 bits, whole steps.
constexpr uint64_t mx_few_bytes(uint64_t cols, uint64_t nt) { return (cols + 127) / 128 * 128 * nt * 4; }

// Tokens of a large tile in 32s: registers hold 128, but not with f16's two ways, nor with f32's split values.
constexpr uint32_t mx_large_columns(uint32_t type) { return type == kTypeF32 ? 1 : type == kTypeF16 ? 2 : 4; }

// Wavefronts that share the length of the rows: as many as LDS holds stages for.
constexpr uint32_t mx_sharing(uint32_t type) { return type == kTypeF32 ? 4 : 8; }

// Whether `count` rows that lie `stride` elements apart, and `tail` bytes from the last one's start, are within 32-bit
// offsets of the first.  A single row's stride is of no account: tensors leave anything there, as a batch of one that is
// cut from longer ones (hidden[:, -1]) does.
inline bool mx_within_reach(uint64_t count, uint64_t stride, uint32_t element, uint32_t tail) {
  return count <= 1 || (stride <= 0xFFFFFFFFu && (count - 1) * stride * element + tail <= 0xFFFFFFFFu);
}

// Up to how many tokens the few tokens' kernel takes the call with, 0 if it does not.  Its LDS is kept to 60 KiB.  One
// token where there are few rows: measured (this kernel and the tiles) 1x4096x14336 e4m3 9.0 and 11.2, 1x1024x4096 bf16
// 3.7 and 5.1, 1x8192x8192 10.7 and 10.5, 1x14336x4096 9.5 and 8.0.  Up to four of f32, whose splitting costs the tiles
// most: 1x14336x4096 9.6 and 29, 2x1024x4096 4.8 and 15, 4x1024x3584 6.5 and 13 (bf16 6.5 and 5.5).
inline uint32_t mx_few_tokens(uint32_t type, const MxLinearArgs& a) {
  const auto fits = [&](uint64_t nt) { return a.tokens <= nt && mx_few_bytes(a.cols, nt) <= 60 * 1024; };
  // 16 rows of a workgroup, whole; tokens are addressed in 64 bits
  const uint64_t rows = a.rows < 16 ? a.rows : 16;
  if (!fits(1) && !fits(2) && !fits(4)) return 0;
  if (!mx_within_reach(rows, a.weight.stride, 1, a.cols / 2) || !mx_within_reach(rows, a.scales.stride, 1, a.cols / 32))
    return 0;
  if (fits(1) && (type == kTypeF32 || a.rows <= 6144)) return 1;
  if (type == kTypeF32) return fits(2) ? 2 : fits(4) ? 4 : 0;
  return 0;
}

// A tile, or the kernel without 32-bit offsets where a wavefront's rows or a tile's tokens are too far apart for them:
// a step of a row is 512 bytes at most.
inline MxLinearChoice mx_tile(uint32_t type, const MxLinearArgs& a, uint32_t rows, uint32_t ct, uint32_t rg, uint32_t kg) {
  const uint64_t n = a.rows < rows ? a.rows : rows, t = a.tokens < 32 * ct ? a.tokens : 32 * ct;
  if (!mx_within_reach(n, a.weight.stride, 1, 512) || !mx_within_reach(n, a.scales.stride, 1, 512) ||
      !mx_within_reach(t, a.x.stride, type_bytes(type), 512) ||
      (type == kTypeE4m3 && !mx_within_reach(t, a.x_scales.stride, 1, 512)))
    return {MxLinearChoice::kSmall, 0, 0, 0, 0, 0, false};
  // the large tile of f32 splits its values on their way, so they may lie anywhere
  const bool raw = type != kTypeF32 || rg == 1;
  const bool aligned = a.weight.ptr % 16 == 0 && (n <= 1 || a.weight.stride % 16 == 0) &&
                       (!raw || (a.x.ptr % 16 == 0 && (t <= 1 || a.x.stride * type_bytes(type) % 16 == 0)));
  return {MxLinearChoice::kTiles, 0, rows, ct, rg, kg, aligned};
}

inline MxLinearChoice mx_tile_by_size(uint32_t type, const MxLinearArgs& a) {
  const uint32_t CT = mx_large_columns(type), KG = mx_sharing(type);
  const auto tile = [&](uint32_t rows, uint32_t ct, uint32_t rg, uint32_t kg) { return mx_tile(type, a, rows, ct, rg, kg); };
  const auto count = [&](uint64_t rows, uint64_t tokens) {
    return ((a.rows + rows - 1) / rows) * ((a.tokens + tokens - 1) / tokens);
  };
  // Tiles of 256 rows where there are enough for the 256 CUs, with half the tokens where there are not, then smaller
  // ones whose wavefronts share the length of the rows: measured (256 rows and 128 tokens, 64 tokens, shared)
  // 512x14336x4096 bf16 (224 tiles of 128) 62, 68, 98; 256x14336x4096 bf16 (112 of 128, 224 of 64) 52, 36, 55;
  // 1024x4096x4096 bf16 (128, 256) 50, 38, 54; 128x14336x4096 bf16 (56, 112) 49, 32, 30; 200x5000x5120 e4m3 (40, 80)
  // 61, 41, 24.
  if (count(256, 32 * CT) >= 160) return tile(64, CT, 4, 1);
  // Rows of two steps at most leave nothing to share, and the products are soon over: a wavefront a tile.  300x5001x128
  // bf16 4.8 and 8.7 with tiles as below, 64x4704x256 3.8 and 4.7; 700x3000x128 5.4 with 64 rows, 6.2 with 32.
  if (type != kTypeF32 && a.cols <= 256) return count(32, 32) > 1600 ? tile(64, 1, 1, 1) : tile(32, 1, 1, 1);
  if (CT == 4 && count(256, 64) >= 160) return tile(64, 2, 4, 1);
  // As many wavefronts to a tile as LDS holds where each tile has a CU of its own, the smaller tile if it still has:
  // 45x1354x960 bf16 (86 tiles of 32 rows) 4.0 and 4.8 with four wavefronts, 32x5120x4096 bf16 (160) 7.2 and 9.3 with
  // 64 rows, 64x4096x4096 e4m3 (256) 6.8 and 8.9; 96x4096x4096 bf16 (384 of 32 rows, 192 of 64) 11.3 and 9.7.
  if (count(32, 32) <= 256) return tile(32, 1, 1, KG);
  // Few tokens read each weight once, and more, smaller tiles keep more of them in flight: 1x14336x4096 bf16 7.7 and
  // 8.2 with 64 rows.
  if (a.tokens <= 16 && count(32, 32) <= 512) return tile(32, 1, 1, 4);
  if (count(64, 32) <= 256) return tile(64, 1, 1, KG);
  // Two workgroups share a CU's LDS with 64 tokens of e4m3, with 32 of the others: 700x3000x2048 bf16 21 and 26 with
  // 64 tokens, 256x14336x4096 e4m3 41 and 48 with 32.
  if (type == kTypeE4m3 && a.tokens > 32) return tile(64, 2, 1, 4);
  return tile(64, 1, 1, 4);
}

inline MxLinearChoice choose_mxfp4_linear(uint32_t type, const MxLinearArgs& a) {
  const uint64_t tiles = (uint64_t)((a.rows + 15) / 16) * ((a.tokens + 15) / 16);
  // Small products end sooner without stages in LDS, each wavefront a step of a small tile: 16x4096x256 bf16 2.8 and
  // 4.0 with tiles, 2x1024x96 2.6 and 4.1, 100x1024x512 3.5 and 4.1, 16x4096x256 f32 3.4 and 5.2; 64x4704x512 bf16 (4704
  // steps) 5.5 and 4.8.
  const bool small = a.cols <= 512 && tiles * ((a.cols + 127) / 128) <= 2048;
  if (const uint32_t nt = mx_few_tokens(type, a)) return {MxLinearChoice::kFew, nt, 0, 0, 0, 0, false};
  return small ? MxLinearChoice{MxLinearChoice::kSmall, 0, 0, 0, 0, 0, false} : mx_tile_by_size(type, a);
}

struct MxMatmulChoice {
  // rows and tokens of a tile; by: wavefronts that share the length of the rows
  enum Kind : uint32_t { kSmall, k256x256, k256x128, k128x128, k128x64, k64x64, k32x32by8, k32x32by4 } kind;
  int dma;  // what goes to LDS by DMA: nothing, the codes (1), the scales too (2)
};

// The product of two MXFP4 matrices; x.stride and weight.stride in bytes.
inline MxMatmulChoice choose_mxfp4_matmul(const MxLinearArgs& a) {
  const auto count = [&](uint64_t rows, uint64_t tokens) {
    return ((a.rows + rows - 1) / rows) * ((a.tokens + tokens - 1) / tokens);
  };
  const auto tile = [&](MxMatmulChoice::Kind kind, uint64_t rows, uint64_t tokens) -> MxMatmulChoice {
    const uint64_t n = a.rows < rows ? a.rows : rows, t = a.tokens < tokens ? a.tokens : tokens;
    if (!mx_within_reach(n, a.weight.stride, 1, a.cols / 2) || !mx_within_reach(t, a.x.stride, 1, a.cols / 2))
      return {MxMatmulChoice::kSmall, 0};
    const auto whole = [](const MxRows& r, uint64_t count) { return r.ptr % 16 == 0 && (count <= 1 || r.stride % 16 == 0); };
    if (!whole(a.weight, n) || !whole(a.x, t)) return {kind, 0};
    // whole quads, so that no scales are read past a row's end
    return {kind, a.cols % 512 == 0 && whole(a.scales, n) && whole(a.x_scales, t) ? 2 : 1};
  };
  // Small products of one quad of steps end sooner without stages in LDS: 16x4096x256 2.4 and 3.4, 64x4704x256 3.1 and
  // 4.5, 100x1024x512 2.9 and 3.6.
  if (a.cols <= 512 && count(16, 16) * ((a.cols + 127) / 128) <= 2048) return {MxMatmulChoice::kSmall, 0};
  // The largest tile of which there are enough for the 256 CUs: measured (256x256, 256x128, 128x128, 128x64)
  // 1024x14336x4096 (224, 448, 896, 1792 tiles) 36, 42, 50, 59; 512x14336x4096 (112, 224, 448, 896) 29, 22, 26, 35;
  // 300x14336x4096 (112, 168, 336, 560) 27, 19, 23, 25; 200x14336x4096 (56, 112, 224, 448) 27, 19, 14, 18;
  // 700x3000x2048 (36, 72, 144, 264) 16, 11, 8, 11; 400x4096x4096 (32, 64, 128, 224) 26, 18, 12, 10.
  if (count(256, 256) >= 160) return tile(MxMatmulChoice::k256x256, 256, 256);
  if (count(256, 128) >= 144) return tile(MxMatmulChoice::k256x128, 256, 128);
  if (count(128, 128) >= 136) return tile(MxMatmulChoice::k128x128, 128, 128);
  // Few tokens or rows: wavefronts share the length of the rows, eight where each tile has a CU of its own: measured
  // (eight, four, 64x64 tiles) 64x4096x4096 (256 tiles of 32) 4.7, 5.0, 7.9; 1x4096x14336 (128) 8.6, 10.9, 16;
  // 37x5001x3360 (314) 7.5, 5.9, 9.2; 1x14336x4096 (448) 8.4, 7.4, 8.0; 33x14336x4096 (896) 12.8, 9.9, 8.5.
  if (a.cols > 512) {
    if (count(32, 32) <= 256) return tile(MxMatmulChoice::k32x32by8, 32, 32);
    if (count(32, 32) <= 512) return tile(MxMatmulChoice::k32x32by4, 32, 32);
  }
  // 64x14336x4096 (224 tiles of 64x64, 112 of 128x64) 8.7 and 10.0, 128x14336x4096 (448, 224) 11.6 and 10.7.
  if (count(64, 64) <= 256) return tile(MxMatmulChoice::k64x64, 64, 64);
  return tile(MxMatmulChoice::k128x64, 128, 64);
}

constexpr uint32_t kMoeUnits = 256;   // compute units
constexpr uint32_t kMoeChunks = 16;   // that the outer products' rows are cut into at most
constexpr uint32_t kMoeFusedPairs = 32;

// How the products of a mixture-of-experts layer are made, for up to kMoeTokens tokens.
struct MxMoeChoice {
  // gate and up: 16 rows a workgroup, four wavefronts along them; 64 rows; columns in registers, two or four steps of a
  // row a wavefront
  enum Inner : uint32_t { kRows16, kRows64, kStream2, kStream4 } inner;
  // down: 16 rows a workgroup and the weighted sums of one or two tokens at once; 64 rows; columns in registers, by chunks
  enum Outer : uint32_t { kSums1, kSums2, kRows, kChunks } outer;
  bool inner_dma, outer_dma;  // codes lie at multiples of 16 bytes; else they go through registers
  bool routed;                // the choice of experts is a launch of its own, not the inner products' workgroups'
  uint32_t span, chunks;      // kChunks: steps of a chunk, chunks of a row; else one
};

inline MxMoeChoice choose_mxfp4_moe(const MxMoeArgs& a) {
  const auto whole = [&](const MxExperts& w) {
    return w.codes.ptr % 16 == 0 && w.codes.stride % 16 == 0 && (a.experts == 1 || w.codes_expert % 16 == 0);
  };
  // 16 rows as 32-bit offsets
  const auto near = [](const MxExperts& w) { return w.codes.stride < 1ull << 27 && w.scales.stride < 1ull << 27; };
  const auto steps_of = [](uint32_t length) { return (length + kMoeStep - 1) / kMoeStep; };
  const uint64_t tokens = a.tokens, pairs = tokens * a.top_k, served = pairs < a.experts ? pairs : a.experts;
  const uint32_t x_steps = steps_of(a.cols), h_steps = steps_of(a.inner), parts = parts_of(a.x_type);
  // columns of the matrix instruction that an expert's tokens take, on average
  const double inner_columns = (double)pairs / a.experts * parts, outer_columns = (double)pairs / a.experts * kMoeInnerParts;
  MxMoeChoice k{};
  k.inner_dma = whole(a.gate) && whole(a.up), k.outer_dma = whole(a.down);
  k.span = k.chunks = 1;
  // Few tokens are chosen for by the inner products' workgroups themselves, each for all of them, a wavefront two tokens:
  // 16 experts of 1024x2048, 4 tokens 22 and 26 with a launch for the choice; 64 experts, 32 tokens 49 and 37.
  k.routed = tokens > 8 || pairs > kMoeFusedPairs;
  // Columns in registers where rows keep most of eight wavefronts busy: measured (so, and by 64 rows) 8 experts of
  // 4096x14336, 64 tokens 97 and 134, 8 tokens 86 and 95; 32 of 4096x2048, 16 tokens 51 and 59; 8192 columns, 64 tokens
  // 78 and 99; 128 of 2048x768, 16 tokens 36 and 30.  Or half of them where an expert's tokens would take the other
  // kernel several passes: 2 experts of 1024x2048, 64 tokens 12 and 19; 10 of 640x5984, 17 tokens of f32 each 62 and 50.
  if (tokens > 1 && k.inner_dma && a.cols > (inner_columns > 32 ? 768 : 2048) && x_steps <= 32 && near(a.gate) &&
      near(a.up) && a.gate.codes.stride == a.up.codes.stride && a.gate.scales.stride == a.up.scales.stride)
    k.inner = x_steps <= 16 ? MxMoeChoice::kStream2 : MxMoeChoice::kStream4;
  // 16 rows where 64 would leave compute units idle, for the four columns that they hold: measured (16 rows, 64)
  // 128 experts of 2048x768, one token 10.2 and 14.3, two 12.6 and 14.5, two of f16 13.1 and 14.9, one of f32 11.6 and
  // 14.5; 16 of 1024x2048, three tokens 9.0 and 10.2; 8 of 1024x512, four 6.7 and 10.0; 8 of 4096x14336, one (448 of 64)
  // 31 and 27.
  else if (tokens * parts <= 4 && served * ((a.inner + 63) / 64) < kMoeUnits)
    k.inner = MxMoeChoice::kRows16;
  else
    k.inner = MxMoeChoice::kRows64;
  // The weighted sums at once, without a launch of their own of 3 to 4, unless few workgroups have much to do: measured
  // (at once, before the sums) 8 experts of 4096x14336, one token 15.0 and 17.4, two 23.9 and 22.6; 16 of 1024x2048, one
  // 5.4 and 6.8, two 7.2 and 6.8; 128 of 2048x768, two 9.3 and 5.4; 6 of 53 of 512x6080, one 17.9 and 9.6.
  if (tokens <= 2 && pairs <= 64 && (a.cols >= 2048 || pairs * h_steps <= 64)) {
    k.outer = tokens == 1 ? MxMoeChoice::kSums1 : MxMoeChoice::kSums2;
    return k;
  }
  // Columns in registers as above, and for shorter rows where there are more of them than the other kernel's workgroups
  // do in one round, or where an expert's tokens would take the other kernel four passes: measured (so, and by 64 rows)
  // 8 experts of 4096x14336, 64 tokens 105 and 222, 8 tokens 47 and 51; 34 of 256x12096, 9 tokens 17 and 26; 32 of
  // 2048x1536, 64 tokens with eight each 35 and 55; 8 of 2048x1536, 64 tokens 19 and 17; 11 of 1120x1504, 7 tokens 9.3 and
  // 6.0; 4 of 2048x800, 64 tokens 15 and 22.
  const uint32_t least = outer_columns > 48 ? 768 : served * ((a.cols + 63) / 64) > 2 * kMoeUnits ? 1024 : 2048;
  const uint32_t chunks = (h_steps + 7) / 8;  // a wavefront of eight has one step of each
  if (k.outer_dma && a.inner > least && chunks <= kMoeChunks && near(a.down)) {
    k.outer = MxMoeChoice::kChunks;
    k.span = (h_steps + chunks - 1) / chunks, k.chunks = (h_steps + k.span - 1) / k.span;
  } else {
    k.outer = MxMoeChoice::kRows;
  }
  return k;
}

}  // namespace ptwm
