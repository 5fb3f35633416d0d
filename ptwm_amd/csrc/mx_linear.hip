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
//     one product each.
// The instruction that takes codes and scales as they lie in memory
// (v_mfma_scale_f32_16x16x128_f8f6f4) would halve the matrix time with 8-bit
// x, but it adds the products of eight neighbours with 13 bits below the
// largest of them: measured, sums are off by 1.2e-5 of their norm with
// normal activations, against 2.5e-8 here, and by 2^-12 of the sum of
// magnitudes where codes spread over e4m3's whole range.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "mx_device.h"

namespace ptwm {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// bf16 parts that hold a value of type T exactly.
constexpr int parts_of(uint32_t type) { return type == kTypeF32 ? 3 : type == kTypeF16 ? 2 : 1; }

// Eight values of type T as they lie in memory.
template <uint32_t T>
struct Raw8 {
  u32x4 w[T == kTypeF32 ? 2 : 1];
};
template <>
struct Raw8<kTypeE4m3> {
  uint64_t w;
};
template <uint32_t T>
__device__ __forceinline__ Raw8<T> load_raw8(uint64_t a) {
  Raw8<T> r;
  if constexpr (T == kTypeE4m3) {
    r.w = ld8(a);
  } else {
    r.w[0] = ld16(a);
    if constexpr (T == kTypeF32) r.w[1] = ld16(a + 16);
  }
  return r;
}

template <uint32_t T>
__device__ __forceinline__ Raw8<T> load_raw8(GlobalBytes p, uint32_t at) {
  Raw8<T> r;
  r.w[0] = ld16(p, at);
  if constexpr (T == kTypeF32) r.w[1] = ld16(p, at + 16);
  return r;
}

__device__ __forceinline__ uint32_t bf16_of_e4m3(uint32_t w, float scale, bool high) {
  return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
}

// Eight values as bf16 parts, each cut from what the ones before it leave
// (truncation, so nothing rounds up to infinity); the rest of an infinity or
// NaN is zero, which keeps it what it is in the sum.  scale: of e4m3 codes,
// read for its exponent only (byte 0 is 2^-127, 255 is NaN).
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
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (T == kTypeF32) {
        const uint32_t a = r.w[0][i], b = r.w[1][i];
        v[i] = bits_f32(a), v[4 + i] = bits_f32(b);
      } else {
        const uint32_t both = r.w[0][i];
        const f16x2 h = __builtin_bit_cast(f16x2, both);
        v[2 * i] = (float)h[0], v[2 * i + 1] = (float)h[1];
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)  // a NaN whose cut would read as an infinity
      if (v[i] != v[i]) v[i] = bits_f32(0x7FC00000u);
#pragma unroll
    for (int j = 0; j < parts_of(T); ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t b0 = f32_bits(v[2 * i]), b1 = f32_bits(v[2 * i + 1]);
        p[j][i] = __builtin_amdgcn_perm(b1, b0, 0x07060302u);
        if (j + 1 < parts_of(T)) {
          const float h0 = bits_f32(b0 & 0xFFFF0000u), h1 = bits_f32(b1 & 0xFFFF0000u);
          v[2 * i] = __builtin_isfinite(h0) ? v[2 * i] - h0 : 0.0f;
          v[2 * i + 1] = __builtin_isfinite(h1) ? v[2 * i + 1] - h1 : 0.0f;
        }
      }
    }
  }
}

// Eight weights of one block as bf16.
__device__ __forceinline__ bf16x8 weights8(uint32_t w, float scale) {
  const u32x4 r = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3))};
  return __builtin_bit_cast(bf16x8, r);
}

__device__ __forceinline__ float scale_f32(uint32_t byte) { return bits_f32(byte << 23); }

__device__ __forceinline__ f32x4 mfma(bf16x8 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ f32x16 mfma32(bf16x8 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// The bias of outputs n .. n+3, zero past the last one or without a bias.
template <uint32_t OT>
__device__ __forceinline__ void load_bias(const MxLinearArgs& a, uint32_t n, float (&b)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    b[j] = a.bias && n + j < a.rows ? load1<OT>(a.bias + (uint64_t)(n + j) * type_bytes(OT)) : 0.0f;
}

// Outputs n .. n+3 of token t, those that exist.
template <uint32_t OT>
__device__ __forceinline__ void store4(const MxLinearArgs& a, uint64_t t, uint32_t n, f32x4 v, const float (&b)[4]) {
  const uint64_t at = a.out.ptr + (t * a.out.stride + n) * type_bytes(OT);
  float o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) o[j] = v[j] + b[j];
  if (n + 3 < a.rows) {
    if constexpr (OT == kTypeF32)
      st16(at, u32x4_make(f32_bits(o[0]), f32_bits(o[1]), f32_bits(o[2]), f32_bits(o[3])));
    else
      st8(at, pack2<OT>(o[0], o[1]) | (uint64_t)pack2<OT>(o[2], o[3]) << 32);
  } else {
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (n + j < a.rows) store1<OT>(at + j * type_bytes(OT), o[j]);
  }
}

// A 16x16 tile of outputs by one workgroup, whose wavefronts take turns in
// steps of 128 values (four blocks) along the rows and add up in LDS.  Lane l
// holds weight row l % 16 and block l / 16 of the step, and token l % 16.
template <uint32_t T, uint32_t OT>
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
      const bf16x8 w8 = weights8(wv[f], scale_f32(sv));
#pragma unroll
      for (int j = parts_of(T) - 1; j >= 0; --j) acc = mfma(w8, p[j], acc);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) part[wave][i][q * 4 + j] = acc[j];
  __syncthreads();
  const uint32_t on = threadIdx.x & 15, ot = threadIdx.x >> 4;
  if (n0 + on < a.rows && t0 + ot < a.tokens) {
    float v = part[0][ot][on] + part[1][ot][on] + part[2][ot][on] + part[3][ot][on];
    if (a.bias) v += load1<OT>(a.bias + (uint64_t)(n0 + on) * type_bytes(OT));
    store1<OT>(a.out.ptr + ((t0 + ot) * a.out.stride + n0 + on) * type_bytes(OT), v);
  }
}

// Many tokens: a tile of 128 * RT weight rows and 32 * CT tokens by one
// workgroup of four wavefronts, 32 * RT rows each.
//
// A step takes 128 values (four blocks) of every row.  The tokens' share goes
// through LDS as bf16 parts, two steps deep; every wavefront reads all of it.
// bf16 whose rows lie at multiples of 16 bytes goes there by itself (DMA),
// other types through registers, both while the step before is multiplied.
// The weights of a wavefront are its own: they go from memory to registers as
// codes, one step ahead, and are widened there.  Within a step the order
// along k is free as long as both operands follow it: lane l's share of
// weight row l % 32 is blocks l / 32 and 2 + l / 32, a 16-byte load each, and
// product f of four takes a block's values 8f .. 8f+7.  A token's 16 chunks of
// eight values (256 bytes, every bank once) are stored at chunk ^ token % 16,
// so 16 lanes that read one chunk of 16 tokens meet 16 different groups of
// four banks.
//
// A row's 64 bytes of codes are requested in one go and its four scales as
// one word: requests to the L2, a segment of one row each, bound an earlier
// form that took them piece by piece.  Offsets within a tile are 32 bits on
// top of uniform addresses (tiles_fit()), which is what leaves registers for
// the operands in flight.
template <uint32_t T, uint32_t OT, int RT, int CT, bool DMA>
__global__ __launch_bounds__(256, 2) void mxfp4_linear_tiles_kernel(MxLinearArgs a) {
  constexpr int P = parts_of(T);
  constexpr uint32_t kTokens = 32 * CT, kRows = 128 * RT;
  // a thread's pieces of the tokens' share: 16 e4m3 codes (two chunks) or one chunk each
  constexpr int C8 = T == kTypeE4m3 ? 2 : 1, J = 2 * CT / C8;
  constexpr uint32_t kPer = 16 / C8;  // pieces of a token
  // two variables, so that a read of one does not wait for what is on its way to the other
  __shared__ u32x4 even[P * kTokens * 16], odd[P * kTokens * 16];
  const uint32_t lane = threadIdx.x & 63, h = lane >> 5, i = lane & 31;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t row_tiles = (a.rows + kRows - 1) / kRows;
  const uint32_t n0 = blockIdx.x % row_tiles * kRows + wave * 32 * RT;
  const uint64_t t0 = (uint64_t)(blockIdx.x / row_tiles) * kTokens;
  const uint32_t blocks = a.cols / kMxBlock, steps = (blocks + 3) / 4, tail = blocks & 3;
  // a wavefront past the last row, or a lane's row or token past it, takes the last one and stores nothing
  const uint32_t nb = min(n0, a.rows - 1);
  GlobalBytes w = global_bytes(a.weight.ptr + nb * a.weight.stride);
  GlobalBytes s = global_bytes(a.scales.ptr + nb * a.scales.stride);
  GlobalBytes x = global_bytes(a.x.ptr + t0 * a.x.stride * type_bytes(T));
  GlobalBytes xsc = global_bytes(a.x_scales.ptr + t0 * a.x_scales.stride);
  uint32_t wo[RT], so[RT], xo[J], xso[J];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const uint32_t n = min(r * 32 + i, a.rows - 1 - nb);
    wo[r] = n * (uint32_t)a.weight.stride;
    so[r] = n * (uint32_t)a.scales.stride;
  }
  // through registers, thread by thread: its chunk's place in LDS is swizzled; by DMA the place is the lane's and the
  // chunk is swizzled
  const uint32_t token = threadIdx.x / kPer;
  const uint32_t chunk = DMA ? (threadIdx.x & 15) ^ (token & 15) : threadIdx.x % kPer * C8;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const uint32_t t = (uint32_t)min((uint64_t)(token + j * (256 / kPer)), a.tokens - 1 - t0);
    xo[j] = (t * (uint32_t)a.x.stride + chunk * 8) * type_bytes(T);
    if constexpr (T == kTypeE4m3) xso[j] = t * (uint32_t)a.x_scales.stride + chunk / 4;
  }
  u32x4 wv[2][2][RT];
  uint32_t sv[2][RT];
  // past a row's end, in the last step, its last block is loaded again, and cleared at its use; a word of scales
  // ends where the row does
  const uint32_t w_at[2] = {tail ? min(h, tail - 1) * 16 : h * 16, tail ? min(2 + h, tail - 1) * 16 : 32 + h * 16};
  const uint32_t s_over = tail ? 4 - tail : 0;
  const uint32_t x_over = tail && chunk / 4 >= tail ? chunk / 4 + 1 - tail : 0;  // never more blocks than lie before
  auto load_weights = [&](int set, bool last) {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      asm("" : "+v"(wo[r]), "+v"(so[r]));
#pragma unroll
      for (int m = 0; m < 2; ++m) wv[set][m][r] = ld16(w, wo[r] + (last ? w_at[m] : h * 16 + m * 32));
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) sv[set][r] = ld4(last ? s - s_over : s, so[r]);
  };
  Raw8<T> raw[J][C8];
  uint32_t xs[J];
  auto load_tokens = [&](u32x4* stage, bool last) {
    const uint32_t over = last ? x_over : 0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      asm("" : "+v"(xo[j]));
      const uint32_t at = xo[j] - over * (kMxBlock * type_bytes(T));
      if constexpr (DMA) {
        __builtin_amdgcn_global_load_lds(x + at, (__attribute__((address_space(3))) void*)(stage + j * 256 + wave * 64),
                                         16, 0, 0);
      } else if constexpr (T == kTypeE4m3) {
        asm("" : "+v"(xso[j]));
        const u32x4 v = ld16(x, at);
        raw[j][0].w = v[0] | (uint64_t)v[1] << 32;
        raw[j][1].w = v[2] | (uint64_t)v[3] << 32;
        xs[j] = xsc[xso[j] - over];
      } else {
        raw[j][0] = load_raw8<T>(x, at);
      }
    }
  };
  auto store_tokens = [&](u32x4* stage) {
    if constexpr (!DMA) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const uint32_t t = token + j * (256 / kPer);
#pragma unroll
        for (int g = 0; g < C8; ++g) {
          u32x4 p[P];
          parts_of_raw<T>(raw[j][g], T == kTypeE4m3 ? scale_f32(xs[j]) : 1.0f, p);
#pragma unroll
          for (int part = 0; part < P; ++part)
            stage[(part * kTokens + t) * 16 + ((chunk + g) ^ (t & 15))] = p[part];
        }
      }
    }
  };
  f32x16 acc[RT][CT] = {};
  // one step from one stage, while the next one's operands are on their way to the other; the last step stands alone,
  // so that the loop has no branch at which all loads in flight would be waited for
  auto multiply = [&](uint32_t step, auto set, u32x4* now, u32x4* next, auto last) {
    const bool next_last = step + 2 == steps;
    w += 64, s += 4, x += 128 * type_bytes(T), xsc += 4;  // of the next step
    // kept uniform: without this the loop carries a 64-bit address for every load and lane
    asm("" : "+s"(w), "+s"(s), "+s"(x), "+s"(xsc));
    // a barrier waits for no DMA: each wavefront waits for its own, requested a step ago, before all meet
    if constexpr (DMA) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if constexpr (last)
      if (tail) {  // what lies past the rows' ends
        for (uint32_t at = threadIdx.x; at < P * kTokens * 16; at += 256)
          if (((at & 15) ^ (at >> 4 & 15)) >= tail * 4) now[at] = u32x4{};
        __syncthreads();
      }
    if constexpr (!last) {
      load_tokens(next, next_last);
      load_weights(set ^ 1, next_last);
    }
    // part p of product u of eight (block pair u / 4, values 8 (u % 4) ..): read one ahead
    u32x4 x8[2][CT];
    auto read = [&](int v) {
      const int u = v / P, part = P - 1 - v % P;
#pragma unroll
      for (int c = 0; c < CT; ++c)
        x8[v & 1][c] = now[(part * kTokens + c * 32 + i) * 16 + (((u / 4 * 2 + h) * 4 + u % 4) ^ (i & 15))];
    };
    read(0);
    bf16x8 w8[RT];
    float sf[RT];
#pragma unroll
    for (int v = 0; v < 8 * P; ++v) {
      const int u = v / P, m = u / 4;
      // what is requested stays ahead of the products it hides behind
      if (v + 1 < 8 * P) read(v + 1);
      if (v % P == 0) {
        const bool in = !last || tail == 0 || 2 * m + h < tail;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          if (u % 4 == 0) {
            const uint32_t byte = 2 * m + h + (last ? s_over : 0);
            sf[r] = scale_f32(in ? sv[set][r] >> (8 * (byte & 3)) & 0xFF : 127);
          }
          w8[r] = weights8(in ? wv[set][m][r][u & 3] : 0, sf[r]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int r = 0; r < RT; ++r) acc[r][c] = mfma32(w8[r], x8[v & 1][c], acc[r][c]);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (!last) store_tokens(next);
  };
  constexpr std::integral_constant<int, 0> k0{};
  constexpr std::integral_constant<int, 1> k1{};
  load_tokens(even, steps == 1);
  load_weights(0, steps == 1);
  store_tokens(even);
  uint32_t step = 0;
  for (; step + 2 < steps; step += 2) {
    multiply(step, k0, even, odd, std::false_type{});
    multiply(step + 1, k1, odd, even, std::false_type{});
  }
  u32x4* stage = even;
  if (step + 2 == steps) {
    multiply(step++, k0, even, odd, std::false_type{});
#pragma unroll
    for (int r = 0; r < RT; ++r) wv[0][0][r] = wv[1][0][r], wv[0][1][r] = wv[1][1][r], sv[0][r] = sv[1][r];
    stage = odd;
  }
  multiply(step, k0, stage, stage, std::true_type{});
  // lane l holds token l % 32 and rows 8 j + 4 (l / 32) .. + 3, j = 0 .. 3
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t n = n0 + r * 32 + j * 8 + h * 4;
      float bias[4];
      load_bias<OT>(a, n, bias);
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        const uint64_t t = t0 + c * 32 + i;
        const f32x4 v = {acc[r][c][4 * j], acc[r][c][4 * j + 1], acc[r][c][4 * j + 2], acc[r][c][4 * j + 3]};
        if (t < a.tokens) store4<OT>(a, t, n, v, bias);
      }
    }
}

// Whether a tile's rows and tokens lie within 32-bit offsets, and a row's scales fill a word.
bool tiles_fit(const MxLinearArgs& a) {
  return a.cols >= 128 && a.weight.stride < (1u << 23) && a.x.stride < (1u << 23) && a.scales.stride < (1u << 23) &&
         a.x_scales.stride < (1u << 23);
}

template <uint32_t T, int RT, int CT>
hipError_t tiles_of(uint32_t out_type, const MxLinearArgs& a, hipStream_t stream) {
  const uint64_t tiles =
      (uint64_t)((a.rows + 128 * RT - 1) / (128 * RT)) * ((a.tokens + 32 * CT - 1) / (32 * CT));
  if (tiles > 0x7FFFFFFFu) return hipErrorInvalidValue;
  const dim3 grid((uint32_t)tiles), block(256);
  if constexpr (T == kTypeBf16) {
    if (a.x.ptr % 16 == 0 && a.x.stride % 8 == 0)
      switch (out_type) {
        case kTypeF32: hipLaunchKernelGGL((mxfp4_linear_tiles_kernel<T, kTypeF32, RT, CT, true>), grid, block, 0, stream, a); return hipGetLastError();
        case kTypeF16: hipLaunchKernelGGL((mxfp4_linear_tiles_kernel<T, kTypeF16, RT, CT, true>), grid, block, 0, stream, a); return hipGetLastError();
        case kTypeBf16: hipLaunchKernelGGL((mxfp4_linear_tiles_kernel<T, kTypeBf16, RT, CT, true>), grid, block, 0, stream, a); return hipGetLastError();
        default: return hipErrorInvalidValue;
      }
  }
  switch (out_type) {
    case kTypeF32: hipLaunchKernelGGL((mxfp4_linear_tiles_kernel<T, kTypeF32, RT, CT, false>), grid, block, 0, stream, a); break;
    case kTypeF16: hipLaunchKernelGGL((mxfp4_linear_tiles_kernel<T, kTypeF16, RT, CT, false>), grid, block, 0, stream, a); break;
    case kTypeBf16: hipLaunchKernelGGL((mxfp4_linear_tiles_kernel<T, kTypeBf16, RT, CT, false>), grid, block, 0, stream, a); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

// 32s of tokens of a workgroup's tile, by the LDS that their parts take.
template <uint32_t T>
constexpr int kTileTokens = T == kTypeF32 ? 1 : T == kTypeF16 ? 2 : 4;

template <uint32_t T>
hipError_t linear_of(uint32_t out_type, const MxLinearArgs& a, hipStream_t stream) {
  if (a.tokens > 64 && tiles_fit(a)) return tiles_of<T, 2, kTileTokens<T>>(out_type, a, stream);
  const uint64_t tiles = (uint64_t)((a.rows + 15) / 16) * ((a.tokens + 15) / 16);
  if (tiles > 0x7FFFFFFFu) return hipErrorInvalidValue;
  const dim3 grid((uint32_t)tiles), block(256);
  switch (out_type) {
    case kTypeF32: hipLaunchKernelGGL((mxfp4_linear_kernel<T, kTypeF32>), grid, block, 0, stream, a); break;
    case kTypeF16: hipLaunchKernelGGL((mxfp4_linear_kernel<T, kTypeF16>), grid, block, 0, stream, a); break;
    case kTypeBf16: hipLaunchKernelGGL((mxfp4_linear_kernel<T, kTypeBf16>), grid, block, 0, stream, a); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_mxfp4_linear(uint32_t x_type, uint32_t out_type, const MxLinearArgs& a, hipStream_t stream) {
  switch (x_type) {
    case kTypeF32: return linear_of<kTypeF32>(out_type, a, stream);
    case kTypeF16: return linear_of<kTypeF16>(out_type, a, stream);
    case kTypeBf16: return linear_of<kTypeBf16>(out_type, a, stream);
    case kTypeE4m3: return linear_of<kTypeE4m3>(out_type, a, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace ptwm
