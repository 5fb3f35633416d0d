// mx_linear.hip -- out = x * W^T (+ bias) with MXFP4 weights W, read as a
// decode restores them.
//
//   out[t, n] = sum_k x[t, k] * e2m1(W[n, k]) * 2^(S[n, k/32] - 127) + bias[n]
//
// The weights are the matrix instruction's first operand (16 rows), the
// tokens its second, and sums are held in 32 bits.  Both operands are widened
// to bf16, in which every value is exact, and so are products in 32 bits:
//   - a weight, a code times its scale, has 2 significant bits and 8 exponent
//     bits (v_cvt_scalef32_pk_bf16_fp4, subnormals included);
//   - x in e4m3 with scales has 4 significant bits
//     (v_cvt_scalef32_pk_bf16_fp8);
//   - x in f16 or f32 is split into two or three bf16 values whose sum is x,
//     one product each; where the weights' scales allow it, f16 is multiplied
//     as it is, by weights in f16.
// The instruction that takes codes and scales as they lie in memory
// (v_mfma_scale_f32_16x16x128_f8f6f4) would halve the matrix time with 8-bit
// x, but it adds the products of eight neighbours with 13 bits below the
// largest of them: measured, sums are off by 1.2e-5 of their norm with
// normal activations, against 2.5e-8 here, and by 2^-12 of the sum of
// magnitudes where codes spread over e4m3's whole range.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "mx_choice.h"
#include "mx_device.h"

namespace ptwm {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// bf16 parts that hold a value of type T exactly.
constexpr int parts_of(uint32_t type) { return type == kTypeF32 ? 3 : type == kTypeF16 ? 2 : 1; }

__device__ __forceinline__ uint32_t bf16_of_e4m3(uint32_t w, float scale, bool high) {
  return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
}

// Eight values as bf16 parts, each cut from what the ones before it leave
// (truncation, so nothing rounds up to infinity).  The parts before the last
// are finite, so an infinity or NaN is the last one, where it stays what it
// is: NaN's highest mantissa bit is set by the subtraction.  scale: of e4m3
// codes, read for its exponent only (byte 0 is 2^-127, 255 is NaN).
constexpr float kBf16Max = 0x1.FEp127f;
template <uint32_t T>
__device__ __forceinline__ void parts_of_raw(const Raw8<T>& r, float scale, u32x4 (&p)[parts_of(T)]) {
  if constexpr (T == kTypeBf16) {
    p[0] = r.w[0];
  } else if constexpr (T == kTypeE4m3) {
    const uint32_t lo = (uint32_t)r.w, hi = (uint32_t)(r.w >> 32);
    p[0] = u32x4_make(bf16_of_e4m3(lo, scale, false), bf16_of_e4m3(lo, scale, true), bf16_of_e4m3(hi, scale, false),
                      bf16_of_e4m3(hi, scale, true));
  } else {
    float v[8];
    values_of<T>(r, v);
#pragma unroll
    for (int j = 0; j < parts_of(T); ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t b[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float& x = v[2 * i + e];
          if (j + 1 < parts_of(T)) {
            b[e] = f32_bits(__builtin_amdgcn_fmed3f(x, -kBf16Max, kBf16Max)) & 0xFFFF0000u;
            x -= bits_f32(b[e]);
          } else {
            b[e] = f32_bits(x);
          }
        }
        p[j][i] = __builtin_amdgcn_perm(b[1], b[0], 0x07060302u);
      }
    }
  }
}

// Eight weights of one block as bf16.
__device__ __forceinline__ u32x4 weights8(uint32_t w, float scale) {
  return u32x4_make(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3)));
}

// The same as f16, where they are in its range.
__device__ __forceinline__ u32x4 weights8_f16(uint32_t w, float scale) {
  return u32x4_make(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 0)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 1)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 2)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 3)));
}

// Whether every byte of a word of scales is in 104 .. 135: code times scale, 2^-24 to 6 * 2^8 in magnitude, is then
// exact in f16.  (A byte that carries into the next one is itself out of range.)
__device__ __forceinline__ bool scales_fit_f16(uint32_t s) {
  return ((s + 0x18181818u) & 0xE0E0E0E0u) == 0x80808080u;
}

__device__ __forceinline__ float scale_f32(uint32_t byte) { return bits_f32(byte << 23); }

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <bool F16>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Outputs n .. n+3 of token t with their bias, those that exist.
template <uint32_t OT>
__device__ __forceinline__ void store4_as(const MxLinearArgs& a, uint64_t t, uint32_t n, f32x4 v) {
  const uint64_t at = a.out.ptr + (t * a.out.stride + n) * type_bytes(OT);
  if (n + 3 < a.rows) {
    if (a.bias) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += load1<OT>(a.bias + (uint64_t)(n + j) * type_bytes(OT));
    }
    if constexpr (OT == kTypeF32)
      st16(at, __builtin_bit_cast(u32x4, v));
    else
      st8(at, pack2<OT>(v[0], v[1]) | (uint64_t)pack2<OT>(v[2], v[3]) << 32);
  } else {
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (n + j < a.rows)
        store1<OT>(at + j * type_bytes(OT),
                   a.bias ? v[j] + load1<OT>(a.bias + (uint64_t)(n + j) * type_bytes(OT)) : v[j]);
  }
}
__device__ __forceinline__ void store4(const MxLinearArgs& a, uint64_t t, uint32_t n, f32x4 v) {
  if (a.out_type == kTypeBf16)
    store4_as<kTypeBf16>(a, t, n, v);
  else if (a.out_type == kTypeF16)
    store4_as<kTypeF16>(a, t, n, v);
  else
    store4_as<kTypeF32>(a, t, n, v);
}

// Small products, and rows too far apart for a tile's 32-bit offsets: a 16x16 tile of
// outputs by one workgroup, whose wavefronts take turns in steps of 128 values
// (four blocks) along the rows and add up in LDS, operands straight from
// memory; bound by one way to memory (16x4096x256 bf16 2.8 us).  Lane l
// holds weight row l % 16 and block l / 16 of the step, and token l % 16.
template <uint32_t T>
__global__ __launch_bounds__(256) void mxfp4_linear_kernel(MxLinearArgs a) {
  __shared__ float part[4][16][17];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, i = lane & 15;
  const uint32_t row_tiles = (a.rows + 15) / 16;
  const uint32_t n0 = blockIdx.x % row_tiles * 16;
  const uint64_t t0 = (uint64_t)(blockIdx.x / row_tiles) * 16;
  const uint32_t blocks = a.cols / kMxBlock;
  // past the last row or token the last one is computed again and not stored
  const uint64_t n = min(n0 + i, a.rows - 1);
  const uint64_t t = min(t0 + i, a.tokens - 1);
  const uint64_t w = a.weight.ptr + n * a.weight.stride;
  const uint64_t s = a.scales.ptr + n * a.scales.stride;
  const uint64_t x = a.x.ptr + t * a.x.stride * type_bytes(T);
  const uint64_t xs = a.x_scales.ptr + t * a.x_scales.stride;
  f32x4 acc = {};
  for (uint32_t k = wave * 4; k < blocks; k += 16) {
    const bool in = k + q < blocks;  // the last step may be short: zero codes there
    u32x4 wv = {};
    uint32_t sv = 127;
    if (in) {
      wv = ld16(w + (uint64_t)(k + q) * 16);
      sv = g_ld<uint8_t>(s + k + q);
    }
    float x_scale = 1.0f;
    if constexpr (T == kTypeE4m3)
      if (in) x_scale = scale_f32(g_ld<uint8_t>(xs + k + q));
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      u32x4 p[parts_of(T)] = {};
      if (in) parts_of_raw<T>(load_raw8<T>(x + ((uint64_t)(k + q) * 32 + f * 8) * type_bytes(T)), x_scale, p);
      const u32x4 w8 = weights8(wv[f], scale_f32(sv));
#pragma unroll
      for (int j = parts_of(T) - 1; j >= 0; --j) acc = mfma(w8, p[j], acc);
    }
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

// A tile of ROWS * RG weight rows and 32 * CT tokens by one workgroup of
// RG * KG wavefronts: RG groups of ROWS rows each, and KG groups that take
// turns in steps of 128 values (four blocks) along the rows and add up in LDS
// at the end.  ROWS is 64 or 32.
//
// The tokens' share of a step goes through LDS; the RG wavefronts of a K group
// load it together and each reads all of it (with RG = 1 a wavefront waits for
// nobody until the end).  Values go there one step ahead, as they are, and are
// widened or split as they are read (RAW), or through registers as bf16 parts,
// where several wavefronts would split the same f32 values.  Rows are
// held in 16-byte chunks, chunk ^ row in place (place()), so the 16 lanes that
// read one chunk of 16 rows at a time meet every bank once.
//
// The weights of a wavefront are its own.  Their codes go to LDS by DMA one
// step ahead, four lanes to a row's 64 bytes, and are read and widened in the
// matrix instruction's order, a row a lane: loading them in that order
// straight to registers costs the address unit a cycle a lane (measured: 16
// bytes a cycle and CU, against 60 this way).  A row's scales of a step are one
// word, loaded by one lane and exchanged between the halves.  Within a step
// the order along k is free as long as both operands follow it: lane l's share
// of weight row l % 32 is blocks l / 32 and 2 + l / 32, and product f of four
// takes a block's values 8f .. 8f+7.
//
// What goes to LDS as it is goes by DMA where it lies at multiples of 16 bytes
// (ALIGNED) and through registers otherwise, to the same places: results do
// not depend on how operands lie.  Offsets within a tile are 32 bits on top of uniform addresses
// (mx_tile()), which is what leaves registers for the operands in flight.

// The place of 16-byte chunk c of row t among rows of S chunks.
template <uint32_t S>
__device__ __forceinline__ uint32_t place(uint32_t t, uint32_t c) {
  constexpr uint32_t per = S < 16 ? 16 / S : 1;  // rows that meet all banks together
  return t * S + (c ^ (t / per & (S < 16 ? S - 1 : 15)));
}

template <uint32_t T, int ROWS, int CT, int RG, int KG, bool RAW, bool ALIGNED>
__global__ __launch_bounds__(64 * RG * KG, RG * KG <= 4 ? 1 + (ROWS * CT * RG >= 512) : RG * KG / 4)
void mxfp4_linear_tiles_kernel(MxLinearArgs a) {
  static_assert(RAW || parts_of(T) > 1, "what needs no split goes as it is");
  constexpr int P = parts_of(T), RT = ROWS / 32, R16 = ROWS / 16;
  constexpr uint32_t kTokens = 32 * CT, kRows = ROWS * RG, kLoaders = 64 * RG;
  constexpr uint32_t S = RAW ? 8 * type_bytes(T) : 16;       // 16-byte chunks of a row (and part) in LDS
  constexpr uint32_t kStage = (RAW ? 1 : P) * kTokens * S;   // chunks of a stage
  // a thread's pieces of the tokens' share: a chunk as it is, or eight values to split
  constexpr uint32_t kPer = RAW ? S : 16;                     // pieces of a token
  constexpr uint32_t kPiece = RAW ? 16 : 8 * type_bytes(T);  // bytes of a piece
  constexpr uint32_t kBlockPieces = kMxBlock * type_bytes(T) / kPiece;
  constexpr int J = kTokens * kPer / kLoaders;
  constexpr uint32_t kTokenStep = kLoaders / kPer;
  constexpr uint32_t kCodes = ROWS * 4;  // chunks of a wavefront's weight codes
  constexpr int XS = CT < 2 ? 1 : CT / 2;   // words of token scales of a lane
  // variables of their own, so that a read of one does not wait for what is on its way to another
  __shared__ u32x4 even_all[KG * kStage], odd_all[KG * kStage], codes_all[RG * KG * kCodes];
  const uint32_t lane = threadIdx.x & 63, h = lane >> 5, i = lane & 31;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t group = wave / RG, rg = wave % RG, loader = rg * 64 + lane;
  u32x4* const even = even_all + group * kStage;
  u32x4* const odd = odd_all + group * kStage;
  u32x4* const codes = codes_all + wave * kCodes;
  const uint32_t row_tiles = (a.rows + kRows - 1) / kRows;
  const uint32_t n0 = blockIdx.x % row_tiles * kRows + rg * ROWS;
  const uint64_t t0 = (uint64_t)(blockIdx.x / row_tiles) * kTokens;
  const uint32_t tokens = (uint32_t)min(a.tokens - t0, (uint64_t)kTokens);
  const uint32_t blocks = a.cols / kMxBlock, steps = (blocks + 3) / 4, rounds = (steps + KG - 1) / KG;
  // a wavefront past the last row, or a lane's row or token past it, takes the last one and stores nothing
  const uint32_t nb = min(n0, a.rows - 1);
  const GlobalBytes w0 = global_bytes(a.weight.ptr + nb * a.weight.stride);
  const GlobalBytes s0 = global_bytes(a.scales.ptr + nb * a.scales.stride);
  const GlobalBytes x0 = global_bytes(a.x.ptr + t0 * a.x.stride * type_bytes(T));
  const GlobalBytes c0 = global_bytes(a.x_scales.ptr + t0 * a.x_scales.stride);
  uint32_t wo[R16], xo[J], co[XS];
  const uint32_t code_chunk = (lane & 3) ^ (lane >> 4);
#pragma unroll
  for (int r = 0; r < R16; ++r)
    wo[r] = min(r * 16 + lane / 4, a.rows - 1 - nb) * (uint32_t)a.weight.stride;
  uint32_t so = min(RT == 2 ? lane : i, a.rows - 1 - nb) * (uint32_t)a.scales.stride;
#pragma unroll
  for (int c = 0; c < XS; ++c)
    if constexpr (T == kTypeE4m3)
      co[c] = min(CT < 2 ? i : c * 64 + lane, tokens - 1) * (uint32_t)a.x_scales.stride;
  // by DMA a piece's place in LDS is the lane's and the piece follows from it, through registers the other way round
  const uint32_t token = loader / kPer;
  auto token_of = [&](int j) { return token + j * kTokenStep; };
  auto piece_of = [&](int j) {
    return RAW ? place<S>(token_of(j), loader % kPer) - token_of(j) * S : loader % kPer;
  };
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const uint32_t t = min(token_of(j), tokens - 1);
    xo[j] = t * (uint32_t)a.x.stride * type_bytes(T) + piece_of(j) * kPiece;
  }
  const uint32_t loads = (tokens + kTokenStep - 1) / kTokenStep;  // of J, the ones with a token
  // In the last round a group's step may end past the row or lie past it.  Loads then repeat the row's last step and
  // block, and what they bring is cleared at its use; a word of scales ends where the row does.
  struct Step {
    uint32_t at;    // the step that is loaded
    uint32_t left;  // blocks of it that count, up to four
    uint32_t in;    // blocks of it that exist, one to four
  };
  auto step_of = [&](uint32_t round) {
    const uint32_t want = round * KG + group;
    Step p;
    p.at = min(want, steps - 1);
    p.in = min(blocks - p.at * 4, 4u);
    p.left = want < steps ? p.in : 0;
    return p;
  };
  u32x4 wr[R16];        // codes on their way through registers
  uint32_t sv, cv[XS];  // scales of a row and of tokens, a byte a block
  Raw8<T> raw[J];  // values on their way through registers
  u32x4 xr[J];
  // request k of the kRequests that bring a step: the words of scales, the codes, the tokens' pieces
  constexpr int kScales = 1 + (T == kTypeE4m3 ? XS : 0), kRequests = kScales + R16 + J;
  auto request = [&](int k, const Step& p, u32x4* stage) {
    if (k < kScales) {
      GlobalBytes g = (k ? c0 : s0) + ((uint64_t)p.at * 4 + p.in - 4);
      asm("" : "+s"(g));  // kept uniform: otherwise the loop carries a 64-bit address for every load and lane
      if (k == 0) {
        asm("" : "+v"(so));
        sv = ld4(g, so);
      } else {
        asm("" : "+v"(co[k - 1]));
        cv[k - 1] = ld4(g, co[k - 1]);
      }
    } else if (k < kScales + R16) {
      const int r = k - kScales;
      GlobalBytes w = w0 + (uint64_t)p.at * 64;
      asm("" : "+s"(w));
      asm("" : "+v"(wo[r]));
      const uint32_t at = wo[r] + min(code_chunk, p.in - 1) * 16;
      if constexpr (ALIGNED)
        __builtin_amdgcn_global_load_lds(w + at, (__attribute__((address_space(3))) void*)(codes + r * 64), 16, 0, 0);
      else
        wr[r] = ld16(w, at);
    } else {
      const int j = k - kScales - R16;
      if (RAW && ALIGNED && RG == 1 && j && (uint32_t)j >= loads) return;  // no token of the batch
      GlobalBytes x = x0 + (uint64_t)p.at * (128 * type_bytes(T));
      asm("" : "+s"(x));
      asm("" : "+v"(xo[j]));
      const uint32_t b = piece_of(j) / kBlockPieces;
      const uint32_t over = b - min(b, p.in - 1);  // blocks to go back: at least as many lie before
      const uint32_t at = xo[j] - over * (kMxBlock * type_bytes(T));
      if constexpr (RAW && ALIGNED)
        __builtin_amdgcn_global_load_lds(
            x + at, (__attribute__((address_space(3))) void*)(stage + j * kLoaders + rg * 64), 16, 0, 0);
      else if constexpr (RAW)
        xr[j] = ld16(x, at);
      else
        raw[j] = load_raw8<T>(x, at);
    }
  };
  auto store = [&](u32x4* stage) {  // what came through registers
    if constexpr (!ALIGNED) {
#pragma unroll
      for (int r = 0; r < R16; ++r) codes[r * 64 + lane] = wr[r];
    }
    if constexpr (RAW && !ALIGNED) {
#pragma unroll
      for (int j = 0; j < J; ++j) stage[j * kLoaders + loader] = xr[j];
    }
    if constexpr (!RAW) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        u32x4 p[P];
        parts_of_raw<T>(raw[j], 1.0f, p);
#pragma unroll
        for (int part = 0; part < P; ++part)
          stage[part * kTokens * S + place<S>(token_of(j), piece_of(j))] = p[part];
      }
    }
  };
  auto meet = [&] {
    // a barrier waits for no DMA: each wavefront waits for its own, requested a step ago, before all meet
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if constexpr (RG > 1)
      __syncthreads();
    else
      __builtin_amdgcn_wave_barrier();
  };
  f32x16 acc[RT][CT] = {};
  // one step from one stage, while the next one's operands are on their way; the last step stands alone, so that the
  // loop has no branch at which all loads in flight would be waited for
  auto multiply = [&](uint32_t round, u32x4* now, u32x4* next, auto last) {
    meet();
    const Step p = step_of(round);
    if constexpr (last) {
      if (p.left < 4) {
        constexpr uint32_t kBlockChunks = S / 4;
        for (uint32_t at = loader; at < kStage; at += kLoaders) {
          const uint32_t t = at / S % kTokens;
          if ((place<S>(t, at % S) - t * S) / kBlockChunks >= p.left) now[at] = u32x4{};
        }
        if constexpr (RG > 1) __syncthreads();
      }
    }
    u32x4 wv[2][RT];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int r = 0; r < RT; ++r) wv[m][r] = codes[(r * 32 + i) * 4 + ((2 * m + h) ^ (i >> 2 & 3))];
    // the word of row or token 32 k + l % 32 in lane l, from the lanes that loaded it
    uint32_t sn[RT], cn[CT];
    if constexpr (RT == 2) {
      const auto both = __builtin_amdgcn_permlane32_swap(sv, sv, false, false);
      sn[0] = both[0], sn[1] = both[1];
    } else {
      sn[0] = sv;
    }
    if constexpr (T == kTypeE4m3) {
#pragma unroll
      for (int k = 0; k < XS; ++k) {
        if constexpr (CT < 2) {
          cn[0] = cv[0];
        } else {
          const auto both = __builtin_amdgcn_permlane32_swap(cv[k], cv[k], false, false);
          cn[2 * k] = both[0], cn[2 * k + 1] = both[1];
        }
      }
    }
    // Product u of eight takes values 8 (u % 4) .. of block pair u / 4.  Chunks are read one ahead: G of them for
    // every kEach products (two for f32; one of e4m3 serves two), P times in parts.
    constexpr int G = RAW && T == kTypeF32 ? 2 : 1, kEach = T == kTypeE4m3 ? 2 : 1;
    constexpr int kParts = RAW ? 1 : P, kReads = 8 / kEach * kParts;
    u32x4 x8[2][CT][G];
    auto read = [&](int v) {
      const int u = v / kParts * kEach, part = kParts - 1 - v % kParts;
      const uint32_t chunk = ((u / 4 * 2 + h) * 4 + u % 4) * G / kEach;
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int g = 0; g < G; ++g)
          x8[v & 1][c][g] = now[part * kTokens * S + place<S>(c * 32 + i, chunk + g)];
    };
    read(0);
    if constexpr (!last) {
      // the codes are in registers before new ones may arrive in their place
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    const Step q = step_of(round + 1);
    auto products = [&](auto f16) {
      u32x4 w8[2][RT];
      float sf[RT], cf[CT];
      auto widen = [&](int u) {  // the weights of product u
        const int m = u / 4;
        const bool in = !last || 2 * m + h < p.left;
        const uint32_t shift = 8 * ((2 * m + h + (last ? 4 - p.in : 0)) & 3);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          if (u % 4 == 0) sf[r] = scale_f32(in ? sn[r] >> shift & 0xFF : 127);
          const uint32_t w = in ? wv[m][r][u & 3] : 0;
          w8[u & 1][r] = f16 ? weights8_f16(w, sf[r]) : weights8(w, sf[r]);
        }
      };
      widen(0);
#pragma unroll
      for (int v = 0; v < 8 * kParts; ++v) {
        const int u = v / kParts, m = u / 4, rd = v / kEach;
        // what is requested stays ahead of the products it hides behind
        if (v % kEach == 0 && rd + 1 < kReads) read(rd + 1);
        if constexpr (!last) {
          // Large tiles spread the next step's requests over the first half of the products: all at once they hold the
          // wavefront up, and its products with it, until the address unit has taken them (512x14336x4096 bf16: 71 us,
          // 62 this way).  Where the weights' way from memory is what takes time they go out at once.
          // What comes through registers is spread over all of them, which holds fewer registers at a time: over the
          // first half 54 of bf16's, 23 of f16's and 5 of e4m3's went to scratch memory, this way 14, 15 and none
          // (unaligned 2048x14336x4096 bf16 346 us -> 251, f16 352 -> 309, e4m3 223 -> 221; with half the wavefronts
          // a SIMD, none at all, 280, 355, 244).
          constexpr int kOver = (RG > 1 ? ALIGNED ? 4 : 8 : 1) * kParts;
#pragma unroll
          for (int k = v * kRequests / kOver; k < (v + 1) * kRequests / kOver && k < kRequests; ++k) request(k, q, next);
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (T == kTypeE4m3) {
          const bool in = !last || 2 * m + h < p.left;
          const uint32_t shift = 8 * ((2 * m + h + (last ? 4 - p.in : 0)) & 3);
#pragma unroll
          for (int c = 0; c < CT; ++c)
            if (u % 4 == 0) cf[c] = scale_f32(in ? cn[c] >> shift & 0xFF : 127);
        }
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          if constexpr (RAW && !f16) {
            Raw8<T> r8;
            if constexpr (T == kTypeE4m3) {
              const uint32_t lo = x8[rd & 1][c][0][u % 2 * 2], hi = x8[rd & 1][c][0][u % 2 * 2 + 1];
              r8.w = lo | (uint64_t)hi << 32;
            } else {
#pragma unroll
              for (int g = 0; g < G; ++g) r8.w[g] = x8[rd & 1][c][g];
            }
            u32x4 b[P];
            parts_of_raw<T>(r8, cf[c], b);
#pragma unroll
            for (int part = P - 1; part >= 0; --part)
#pragma unroll
              for (int r = 0; r < RT; ++r) acc[r][c] = mfma32<false>(w8[u & 1][r], b[part], acc[r][c]);
          } else {
#pragma unroll
            for (int r = 0; r < RT; ++r) acc[r][c] = mfma32<f16>(w8[u & 1][r], x8[rd & 1][c][0], acc[r][c]);
          }
        }
        // the next product's weights are widened while the matrix unit works: an instruction of it takes the time of
        // about six others, and the wavefront is free in between
        if (v % kParts == kParts - 1 && u < 7) widen(u + 1);
#pragma unroll
        for (int k = 0; k < CT * RT * (RAW && !f16 ? P : 1); ++k) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a matrix instruction
          __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);  // up to four others
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    // f16 needs no split where the weights are exact in f16 as well, which their scales tell
    if constexpr (T == kTypeF16) {
      if (__all(scales_fit_f16(sv)))
        products(std::true_type{});
      else
        products(std::false_type{});
    } else {
      products(std::false_type{});
    }
    if constexpr (!last) store(next);
  };
  // Rows of less than a step have their scales gathered, bytes past the word's start left as 2^0.
  auto gather = [&](GlobalBytes g, uint32_t at) {
    uint32_t word = 0x7F7F7F7Fu;
    for (uint32_t b = 0; b < blocks; ++b) word = word >> 8 | (uint32_t)g[at + b] << 24;
    return word;
  };
#pragma unroll
  for (int k = 0; k < kRequests; ++k)
    if (k >= kScales || blocks >= 4) request(k, step_of(0), even);
  if (blocks < 4) {
    sv = gather(s0, so);
    if constexpr (T == kTypeE4m3) {
#pragma unroll
      for (int c = 0; c < XS; ++c) cv[c] = gather(c0, co[c]);
    }
  }
  store(even);
  uint32_t round = 0;
  for (; round + 2 < rounds; round += 2) {
    multiply(round, even, odd, std::false_type{});
    multiply(round + 1, odd, even, std::false_type{});
  }
  u32x4* stage = even;
  if (round + 2 == rounds) {
    multiply(round++, even, odd, std::false_type{});
    stage = odd;
  }
  multiply(round, stage, stage, std::true_type{});

  // lane l holds token l % 32 and rows 8 j + 4 (l / 32) .. + 3, j = 0 .. 3
  constexpr int kQuads = RT * CT * 4;
  auto write = [&](int quad, f32x4 v) {
    const int r = quad / (CT * 4), c = quad / 4 % CT, j = quad % 4;
    const uint64_t t = t0 + c * 32 + i;
    if (t < a.tokens) store4(a, t, n0 + r * 32 + j * 8 + h * 4, v);
  };
  auto quad_of = [&](int quad) {
    const int r = quad / (CT * 4), c = quad / 4 % CT, j = quad % 4;
    return f32x4{acc[r][c][4 * j], acc[r][c][4 * j + 1], acc[r][c][4 * j + 2], acc[r][c][4 * j + 3]};
  };
  if constexpr (KG == 1) {
    if (ROWS == 64 && n0 + ROWS <= a.rows) {
      // Through the wavefront's own codes' LDS, so that eight lanes store 128 bytes of a token's outputs, and not a
      // lane 8 of them: 1039x11937x96 bf16 15 us, 20 without; 512x14336x1024 bf16 19.7 and 22.1; 2048x14336x4096 e4m3
      // 195 and 202, f16 236 and 245.
      auto rows_first = [&](auto type) {
        constexpr uint32_t OT = type;
        constexpr int R = OT == kTypeF32 ? 1 : RT;  // groups of 32 rows in 128 bytes
        f32x4 bias[RT][4] = {};
        if (a.bias) {
#pragma unroll
          for (int k = 0; k < RT * 16; ++k)
            bias[k / 16][k / 4 % 4][k % 4] =
                load1<OT>(a.bias + (uint64_t)(n0 + k / 16 * 32 + k / 4 % 4 * 8 + h * 4 + k % 4) * type_bytes(OT));
        }
#pragma unroll
        for (int pass = 0; pass < RT * CT / R; ++pass) {
          const int c = pass * R / RT, r0 = pass * R % RT;
#pragma unroll
          for (int k = 0; k < R * 4; ++k) {
            const int r = r0 + k / 4, j = k % 4;
            const f32x4 v = quad_of((r * CT + c) * 4 + j) + bias[r][j];
            if constexpr (OT == kTypeF32) {
              codes[i * 8 + ((2 * j + h) ^ (i & 7))] = __builtin_bit_cast(u32x4, v);
            } else {
              const uint64_t two = pack2<OT>(v[0], v[1]) | (uint64_t)pack2<OT>(v[2], v[3]) << 32;
              reinterpret_cast<uint64_t*>(codes)[2 * (i * 8 + (k ^ (i & 7))) + h] = two;
            }
          }
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // other lanes' values
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t t = k * 8 + lane / 8;
            const u32x4 v = codes[t * 8 + ((lane & 7) ^ (t & 7))];
            const uint64_t at = t0 + c * 32 + t;
            if (at < a.tokens)
              st16(a.out.ptr + (at * a.out.stride + n0 + r0 * 32) * type_bytes(OT) + (lane & 7) * 16, v);
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
      return;
    }
#pragma unroll
    for (int quad = 0; quad < kQuads; ++quad) write(quad, quad_of(quad));
  } else {
    // the groups' sums take the place of their stages, in the order of the groups
    constexpr uint32_t kFit = kStage / 64;
    static_assert(RG == 1 && kQuads <= 2 * kFit, "a K group is a wavefront");
    __syncthreads();
#pragma unroll
    for (uint32_t quad = 0; quad < kQuads; ++quad)
      (quad < kFit ? even + quad * 64 : odd + (quad - kFit) * 64)[lane] = __builtin_bit_cast(u32x4, quad_of(quad));
    __syncthreads();
    for (uint32_t quad = wave; quad < kQuads; quad += KG) {
      const u32x4* from = quad < kFit ? even_all + quad * 64 : odd_all + (quad - kFit) * 64;
      f32x4 v = {};
#pragma unroll
      for (int g = 0; g < KG; ++g) v += __builtin_bit_cast(f32x4, from[g * kStage + lane]);
      write(quad, v);
    }
  }
}

// One or a few tokens (NT): 16 weight rows by one workgroup of W wavefronts,
// without the matrix instruction, whose other columns would be idle.  The
// tokens lie in LDS in 32 bits, zeros past their ends.  A wavefront takes every
// W-th step of 128 values; a lane holds block l % 4 of it in row l / 4, so that
// codes and scales come from memory in the order in which they lie, straight
// to registers, kDepth steps ahead.  A lane's 32 products are summed by fused
// multiply-adds in 32 bits, in eight sums, the four lanes of a row and the
// wavefronts at the end.
//
// The weights are read once.  16 widening instructions and 32 * NT
// multiply-adds for 1 KiB of codes (a wavefront's 64 lanes) let a CU take 15
// bytes a cycle with one token, more than its share of what memory gives; what
// is left above that time is the way of the first and the last bytes.
constexpr int kFewWaves = 8;

template <uint32_t T, int NT>
__global__ __launch_bounds__(64 * kFewWaves) void mxfp4_linear_few_kernel(MxLinearArgs a) {
  constexpr int kDepth = 4, W = kFewWaves;
  extern __shared__ f32x4 few_x[];  // NT rows of whole steps
  __shared__ float part[W][NT][16];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane & 3;
  const uint32_t n0 = blockIdx.x * 16;
  const uint32_t blocks = a.cols / kMxBlock, steps = (blocks + 3) / 4;
  const GlobalBytes w0 = global_bytes(a.weight.ptr + n0 * a.weight.stride);
  const GlobalBytes s0 = global_bytes(a.scales.ptr + n0 * a.scales.stride);
  const uint32_t row = min(lane / 4, a.rows - 1 - n0);
  const uint32_t wo = row * (uint32_t)a.weight.stride, so = row * (uint32_t)a.scales.stride;
  u32x4 wv[kDepth];
  uint32_t sv[kDepth];
  auto request = [&](int d, uint32_t step) {
    const uint32_t b = min(step * 4 + q, blocks - 1);  // past the end the last block again, against zeros
    wv[d] = ld16(w0, wo + b * 16);
    sv[d] = s0[so + b];
  };
  // the tokens' first values are asked for before the weights, behind which they would wait
  Raw8<T> raw[NT];
  uint32_t byte[NT];
  auto ask = [&](uint32_t k) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const uint64_t at = min((uint64_t)t, a.tokens - 1);
      const uint32_t c = min(k, a.cols - 8);
      raw[t] = load_raw8<T>(a.x.ptr + (at * a.x.stride + c) * type_bytes(T));
      if constexpr (T == kTypeE4m3) byte[t] = g_ld<uint8_t>(a.x_scales.ptr + at * a.x_scales.stride + c / kMxBlock);
    }
  };
  auto take = [&](uint32_t k) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float v[8];
      if constexpr (T == kTypeE4m3) {
        u32x4 p[1];
        parts_of_raw<T>(raw[t], scale_f32(byte[t]), p);
        values_of<kTypeBf16>(Raw8<kTypeBf16>{{p[0]}}, v);
      } else {
        values_of<T>(raw[t], v);
      }
      const bool in = k < a.cols;
      f32x4* const to = few_x + t * steps * 32 + k / 4;
      to[0] = in ? f32x4{v[0], v[1], v[2], v[3]} : f32x4{};
      to[1] = in ? f32x4{v[4], v[5], v[6], v[7]} : f32x4{};
    }
  };
  uint32_t k = threadIdx.x * 8;
  ask(k);
#pragma unroll
  for (int d = 0; d < kDepth; ++d) request(d, wave + d * W);
  while (k < steps * 128) {
    take(k);
    k += 64 * W * 8;
    if (k < steps * 128) ask(k);
  }
  __syncthreads();
  f32x4 acc[NT][2] = {};
  for (uint32_t step = wave; step < steps; step += kDepth * W) {
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      const uint32_t now = step + d * W;
      if (now >= steps) break;
      const bool in = now * 4 + q < blocks;
      const u32x4 wn = wv[d];
      const float sf = scale_f32(in ? sv[d] : 127);
      request(d, now + kDepth * W);
#pragma unroll
      for (int f = 0; f < 4; ++f) {  // eight values
        f32x4 x[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            x[t][e] = few_x[t * steps * 32 + now * 32 + q * 8 + f * 2 + e];
        const uint32_t c = wn[f];
        const f32x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, sf, 0);
        const f32x2 p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, sf, 1);
        const f32x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, sf, 2);
        const f32x2 p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, sf, 3);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            acc[t][e][0] = __builtin_fmaf(e ? p2[0] : p0[0], x[t][e][0], acc[t][e][0]);
            acc[t][e][1] = __builtin_fmaf(e ? p2[1] : p0[1], x[t][e][1], acc[t][e][1]);
            acc[t][e][2] = __builtin_fmaf(e ? p3[0] : p1[0], x[t][e][2], acc[t][e][2]);
            acc[t][e][3] = __builtin_fmaf(e ? p3[1] : p1[1], x[t][e][3], acc[t][e][3]);
          }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const f32x4 s4 = acc[t][0] + acc[t][1];
    float v = (s4[0] + s4[1]) + (s4[2] + s4[3]);
    v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0xB1, 0xF, 0xF, true));
    v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x4E, 0xF, 0xF, true));
    if (q == 0) part[wave][t][lane / 4] = v;
  }
  __syncthreads();
  if (threadIdx.x < 4 * NT) {
    const uint32_t t = threadIdx.x / 4, n = threadIdx.x % 4 * 4;
    f32x4 v = {};
#pragma unroll
    for (int g = 0; g < W; ++g)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += part[g][t][n + j];
    if (t < a.tokens) store4(a, t, n0 + n, v);
  }
}

// The outputs of rows first .. first + rows - 1, and of tokens.
MxLinearArgs some_rows(const MxLinearArgs& a, uint64_t first, uint64_t rows) {
  MxLinearArgs p = a;
  const uint64_t skip = first * type_bytes(a.out_type);
  p.weight = rows_from(a.weight, first, 1), p.scales = rows_from(a.scales, first, 1);
  p.out.ptr += skip, p.bias = a.bias ? a.bias + skip : 0;
  p.rows = (uint32_t)rows;
  return p;
}
template <uint32_t T>
MxLinearArgs some_tokens(const MxLinearArgs& a, uint64_t first, uint64_t tokens) {
  MxLinearArgs p = a;
  p.x = rows_from(a.x, first, type_bytes(T)), p.x_scales = rows_from(a.x_scales, first, 1);
  p.out = rows_from(a.out, first, type_bytes(a.out_type));
  p.tokens = tokens;
  return p;
}

// Workgroups of TR rows and TT tokens each, rows first, in as few launches as hold them.
template <uint32_t T, uint32_t TR, uint32_t TT>
hipError_t launch_tiles(void (*kernel)(MxLinearArgs), uint32_t threads, const MxLinearArgs& a, hipStream_t stream,
                        uint32_t shared = 0) {
  const uint64_t most = kMaxThreads / threads;
  return in_parts(a.rows, most * TR, [&](uint64_t row, uint64_t rows) {
    const uint64_t row_tiles = (rows + TR - 1) / TR;
    return in_parts(a.tokens, most / row_tiles * TT, [&](uint64_t token, uint64_t tokens) {
      return launch(kernel, row_tiles * ((tokens + TT - 1) / TT), threads,
                    some_tokens<T>(some_rows(a, row, rows), token, tokens), stream, shared);
    });
  });
}

template <uint32_t T, int ROWS, int CT, int RG, int KG, bool RAW>
hipError_t tiles_of(const MxLinearArgs& a, bool aligned, hipStream_t stream) {
  return launch_tiles<T, ROWS * RG, 32 * CT>(aligned ? mxfp4_linear_tiles_kernel<T, ROWS, CT, RG, KG, RAW, true>
                                                     : mxfp4_linear_tiles_kernel<T, ROWS, CT, RG, KG, RAW, false>,
                                             64 * RG * KG, a, stream);
}

template <uint32_t T, int NT>
hipError_t few_of(const MxLinearArgs& a, hipStream_t stream) {
  return launch_tiles<T, 16, NT>(mxfp4_linear_few_kernel<T, NT>, 64 * kFewWaves, a, stream,
                                 (uint32_t)mx_few_bytes(a.cols, NT));
}

template <uint32_t T>
hipError_t linear_of(const MxLinearArgs& a, hipStream_t stream) {
  const MxLinearChoice k = choose_mxfp4_linear(T, a);
  if (k.kind == MxLinearChoice::kFew) {
    if (k.tokens == 1) return few_of<T, 1>(a, stream);
    if constexpr (T == kTypeF32) {
      if (k.tokens == 2) return few_of<T, 2>(a, stream);
      if (k.tokens == 4) return few_of<T, 4>(a, stream);
    }
    return hipErrorInvalidValue;
  }
  if (k.kind == MxLinearChoice::kTiles) {
    constexpr int CT = mx_large_columns(T), KG = mx_sharing(T);
    const auto is = [&](uint32_t rows, uint32_t ct, uint32_t rg, uint32_t kg) {
      return k.rows == rows && k.ct == ct && k.rg == rg && k.kg == kg;
    };
    if (is(64, CT, 4, 1)) return tiles_of<T, 64, CT, 4, 1, T != kTypeF32>(a, k.aligned, stream);
    if (is(32, 1, 1, KG)) return tiles_of<T, 32, 1, 1, KG, true>(a, k.aligned, stream);
    if (is(64, 1, 1, KG)) return tiles_of<T, 64, 1, 1, KG, true>(a, k.aligned, stream);
    if constexpr (T != kTypeF32) {
      if (is(32, 1, 1, 4)) return tiles_of<T, 32, 1, 1, 4, true>(a, k.aligned, stream);
      if (is(64, 1, 1, 4)) return tiles_of<T, 64, 1, 1, 4, true>(a, k.aligned, stream);
      if (is(32, 1, 1, 1)) return tiles_of<T, 32, 1, 1, 1, true>(a, k.aligned, stream);
      if (is(64, 1, 1, 1)) return tiles_of<T, 64, 1, 1, 1, true>(a, k.aligned, stream);
    }
    if constexpr (CT == 4)
      if (is(64, 2, 4, 1)) return tiles_of<T, 64, 2, 4, 1, true>(a, k.aligned, stream);
    if constexpr (T == kTypeE4m3)
      if (is(64, 2, 1, 4)) return tiles_of<T, 64, 2, 1, 4, true>(a, k.aligned, stream);
    return hipErrorInvalidValue;
  }
  return launch_tiles<T, 16, 16>(mxfp4_linear_kernel<T>, 256, a, stream);
}

}  // namespace

hipError_t launch_mxfp4_linear(uint32_t x_type, const MxLinearArgs& a, hipStream_t stream) {
  switch (x_type) {
    case kTypeF32: return linear_of<kTypeF32>(a, stream);
    case kTypeF16: return linear_of<kTypeF16>(a, stream);
    case kTypeBf16: return linear_of<kTypeBf16>(a, stream);
    case kTypeE4m3: return linear_of<kTypeE4m3>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace ptwm
