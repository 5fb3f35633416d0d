// mx_choice.h -- which kernel takes a product with MXFP4 weights: rules on
// sizes, types and alignment, on the host.  The times beside them are
// microseconds on an MI355X.
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

}  // namespace ptwm
