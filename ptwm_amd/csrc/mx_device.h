// mx_device.h -- device helpers of the MX operators: loads and stores of
// eight values, and the quantisation of a block to e4m3 codes.
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
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
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

}  // namespace ptwm
