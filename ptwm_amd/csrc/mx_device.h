// mx_device.h -- device helpers of the MX operators: loads and stores of
// eight values, the quantisation of a block to e4m3 codes, and what the
// products share (values as bf16 parts, widened weights, stores of outputs).
#pragma once

#include "mx_ops.h"

namespace ptwm {

// A launch holds fewer than 2^32 threads: what goes past them would not run, and no error would say so.
constexpr uint64_t kMaxThreads = 0xFFFFFFFF;

// One launch with one argument; the triple chevrons' way keeps a stack of configurations besides.
template <typename A>
hipError_t launch(void (*kernel)(A), uint64_t groups, uint32_t threads, const A& a, hipStream_t stream,
                  uint32_t shared = 0) {
  if (groups > kMaxThreads / threads) return hipErrorInvalidValue;
  void* args[] = {const_cast<A*>(&a)};
  return hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3((uint32_t)groups), dim3(threads), args, shared,
                         stream);
}

// The rows of an operand from row `first` on.
inline MxRows rows_from(const MxRows& r, uint64_t first, uint32_t element) {
  return {r.ptr ? r.ptr + first * r.stride * element : 0, r.stride};
}

// Calls f(first, count) for parts of `most` rows, one after the other, until all are served or one fails.
template <typename F>
hipError_t in_parts(uint64_t rows, uint64_t most, F&& f) {
  for (uint64_t first = 0; first < rows; first += most) {
    const hipError_t e = f(first, rows - first < most ? rows - first : most);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Rows start at any multiple of the element's size, so vector accesses are
// declared at byte alignment: gfx950 takes them as they are.
struct __attribute__((packed)) Bytes16 {
  u32x4 v;
};
struct __attribute__((packed)) Bytes8 {
  uint64_t v;
};
struct __attribute__((packed)) Bytes4 {
  uint32_t v;
};
__device__ __forceinline__ u32x4 ld16(uint64_t a) {
  return ((const __attribute__((address_space(1))) Bytes16*)(uintptr_t)a)->v;
}
__device__ __forceinline__ uint64_t ld8(uint64_t a) {
  return ((const __attribute__((address_space(1))) Bytes8*)(uintptr_t)a)->v;
}
__device__ __forceinline__ void st16(uint64_t a, u32x4 v) {
  ((__attribute__((address_space(1))) Bytes16*)(uintptr_t)a)->v = v;
}
__device__ __forceinline__ void st8(uint64_t a, uint64_t v) {
  ((__attribute__((address_space(1))) Bytes8*)(uintptr_t)a)->v = v;
}
__device__ __forceinline__ void st4(uint64_t a, uint32_t v) {
  ((__attribute__((address_space(1))) Bytes4*)(uintptr_t)a)->v = v;
}

// A uniform address and 32-bit offsets from it.
typedef const __attribute__((address_space(1))) uint8_t* GlobalBytes;
__device__ __forceinline__ GlobalBytes global_bytes(uint64_t a) { return (GlobalBytes)(uintptr_t)a; }
__device__ __forceinline__ u32x4 ld16(GlobalBytes p, uint32_t at) {
  return ((const __attribute__((address_space(1))) Bytes16*)(p + at))->v;
}
__device__ __forceinline__ uint32_t ld4(GlobalBytes p, uint32_t at) {
  return ((const __attribute__((address_space(1))) Bytes4*)(p + at))->v;
}

// An address that is the same in all lanes, in scalar registers.
__device__ __forceinline__ GlobalBytes uniform(uint64_t a) {
  // the builtin's result is signed
  const uint32_t low = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a);
  const uint32_t high = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32));
  return global_bytes(low | (uint64_t)high << 32);
}

// DMA of 16 bytes a lane from a uniform address and the lane's offset to consecutive places in LDS from `to` (uniform)
// on.  Written out, because the compiler waits for all that is on its way before it reads LDS.  Nothing but a wait on
// vmcnt says that the bytes have come.
__device__ __forceinline__ void dma16(GlobalBytes from, uint32_t offset, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(from)
               : "memory", "m0");
}
__device__ __forceinline__ void dma16(uint64_t from, uint32_t to) {  // from the lane's own address
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory", "m0");
}
// Of bytes that nobody reads again: they leave L2 first, and what is being written there stays until its lines are full.
__device__ __forceinline__ void dma16_once(GlobalBytes from, uint32_t offset, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(to), "v"(offset), "s"(from)
               : "memory", "m0");
}
__device__ __forceinline__ void dma16_once(uint64_t from, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt" ::"s"(to), "v"(from) : "memory", "m0");
}

// DMA of 4 bytes a lane, from multiples of 4.
__device__ __forceinline__ void dma4(GlobalBytes from, uint32_t offset, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(to), "v"(offset), "s"(from)
               : "memory", "m0");
}
__device__ __forceinline__ void dma4(uint64_t from, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(to), "v"(from) : "memory", "m0");
}

// LDS by its byte address, which takes a known offset along in the instruction.
typedef __attribute__((address_space(3))) u32x4* LdsChunks;
typedef __attribute__((address_space(3))) u32x2* LdsPairs;
template <typename T>
__device__ __forceinline__ uint32_t lds_address(T* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) T*)p;
}

__device__ __forceinline__ float bits_f32(uint32_t b) { return __builtin_bit_cast(float, b); }
__device__ __forceinline__ uint32_t f32_bits(float f) { return __builtin_bit_cast(uint32_t, f); }

// Eight consecutive values of type T as they lie in memory, and in 32 bits.
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
template <uint32_t T>
__device__ __forceinline__ void values_of(const Raw8<T>& r, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a = r.w[0][i];
    if constexpr (T == kTypeF32) {
      const uint32_t b = r.w[1][i];
      v[i] = bits_f32(a), v[4 + i] = bits_f32(b);
    } else if constexpr (T == kTypeBf16) {
      v[2 * i] = bits_f32(a << 16);
      v[2 * i + 1] = bits_f32(a & 0xFFFF0000u);
    } else {
      const f16x2 h = __builtin_bit_cast(f16x2, a);
      v[2 * i] = (float)h[0], v[2 * i + 1] = (float)h[1];
    }
  }
}
template <uint32_t T>
__device__ __forceinline__ void load8(uint64_t a, float (&v)[8]) {
  values_of<T>(load_raw8<T>(a), v);
}

// Two values rounded to nearest even in a 16-bit type.
template <uint32_t T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (T == kTypeBf16) {
    const bf16x2 r = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, r);
  } else {
    const f16x2 r = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, r);
  }
}

template <uint32_t T>
__device__ __forceinline__ void store8(uint64_t a, const float (&v)[8]) {
  if constexpr (T == kTypeF32) {
    st16(a, u32x4_make(f32_bits(v[0]), f32_bits(v[1]), f32_bits(v[2]), f32_bits(v[3])));
    st16(a + 16, u32x4_make(f32_bits(v[4]), f32_bits(v[5]), f32_bits(v[6]), f32_bits(v[7])));
  } else {
    st16(a, u32x4_make(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7])));
  }
}

template <uint32_t T>
__device__ __forceinline__ void store1(uint64_t a, float v) {
  if constexpr (T == kTypeF32) {
    g_st<float>(a, v);
  } else {
    g_st<uint16_t>(a, (uint16_t)pack2<T>(v, 0.0f));
  }
}
template <uint32_t T>
__device__ __forceinline__ float load1(uint64_t a) {
  if constexpr (T == kTypeF32) return g_ld<float>(a);
  const uint16_t b = g_ld<uint16_t>(a);
  if constexpr (T == kTypeBf16) return bits_f32((uint32_t)b << 16);
  return (float)__builtin_bit_cast(_Float16, b);
}

// The e4m3 codes of eight values, the quad's four lanes holding one block,
// and the block's scale byte (the same in the four lanes).
//
// The scale is the smallest power of two 2^(b-127), b >= 0, with
// max|v| <= 448 * 2^(b-127), so nothing saturates.  448 is 1.75 * 2^8, and
// with max|v| = 1.m * 2^(E-127) that is b = E - 8, plus one where 1.m > 1.75.
// The multiplication by 2^(127-b) is exact, and one rounding to nearest even
// remains.  A block with an infinity or NaN gets the scale NaN and NaN codes.
__device__ __forceinline__ uint32_t quantise8(const float (&v)[8], uint32_t& lo, uint32_t& hi) {
  uint32_t m = 0;  // magnitudes compare as integers, infinities and NaN last
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, f32_bits(v[i]) & 0x7FFFFFFFu);
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xF, 0xF, true));  // lanes 1 0 3 2
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xF, 0xF, true));  // lanes 2 3 0 1
  const bool broken = m >= 0x7F800000u;
  const int b = max((int)(m >> 23) - 8 + ((m & 0x7FFFFFu) > 0x600000u ? 1 : 0), 0);
  const float inv = bits_f32((uint32_t)(254 - b) << 23);
  int a = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, 0, false);
  a = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, a, true);
  int c = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * inv, v[5] * inv, 0, false);
  c = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * inv, v[7] * inv, c, true);
  lo = broken ? 0x7F7F7F7Fu : (uint32_t)a;
  hi = broken ? 0x7F7F7F7Fu : (uint32_t)c;
  return broken ? 255u : (uint32_t)b;
}

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

__device__ __forceinline__ float scale_f32(uint32_t byte) { return bits_f32(byte << 23); }

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
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

// The outputs of rows first .. first + rows - 1, and of tokens.
inline MxLinearArgs some_rows(const MxLinearArgs& a, uint64_t first, uint64_t rows) {
  MxLinearArgs p = a;
  const uint64_t skip = first * type_bytes(a.out_type);
  p.weight = rows_from(a.weight, first, 1), p.scales = rows_from(a.scales, first, 1);
  p.out.ptr += skip, p.bias = a.bias ? a.bias + skip : 0;
  p.rows = (uint32_t)rows;
  return p;
}
inline MxLinearArgs some_tokens(const MxLinearArgs& a, uint32_t x_element, uint64_t first, uint64_t tokens) {
  MxLinearArgs p = a;
  p.x = rows_from(a.x, first, x_element), p.x_scales = rows_from(a.x_scales, first, 1);
  p.out = rows_from(a.out, first, type_bytes(a.out_type));
  p.tokens = tokens;
  return p;
}

// Workgroups of TR rows and TT tokens (X bytes an element) each, rows first, in as few launches as hold them.
template <uint32_t X, uint32_t TR, uint32_t TT>
hipError_t launch_tiles(void (*kernel)(MxLinearArgs), uint32_t threads, const MxLinearArgs& a, hipStream_t stream,
                        uint32_t shared = 0) {
  const uint64_t most = kMaxThreads / threads;
  return in_parts(a.rows, most * TR, [&](uint64_t row, uint64_t rows) {
    const uint64_t row_tiles = (rows + TR - 1) / TR;
    return in_parts(a.tokens, most / row_tiles * TT, [&](uint64_t token, uint64_t tokens) {
      return launch(kernel, row_tiles * ((tokens + TT - 1) / TT), threads,
                    some_tokens(some_rows(a, row, rows), X, token, tokens), stream, shared);
    });
  });
}

}  // namespace ptwm
