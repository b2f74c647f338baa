// The codes of a cache held in 8 bits: e4m3 (4 exponent and 3 mantissa bits, no infinities, greatest 448) or int8, times a power
// of two for each block of tokens and head, kept as its exponent with bias 127 (255: not a number). A power of two costs e4m3
// nothing (a floating code is as exact at any scale) and int8 half a bit in the mean; in return x / scale and code x scale are
// exact, so a code is the correct rounding of its definition and code x scale, of 8 significant bits at most, is exact in bf16
// (in fp16 from its least subnormal to its greatest value; saturate_f16 has those past it become the greatest: an infinity
// would turn the probabilities 0 of the keys beside it into NaN, and 65504 rounded to e4m3 is 65536).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"

namespace bp {
namespace cache8 {

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int kE4m3 = 0;
constexpr int kInt8 = 1;

// From here on this wave's fp16 results that overflow are the greatest finite value (bit 23 of the mode register, FP16_OVFL).
__device__ __forceinline__ void saturate_f16() { __builtin_amdgcn_s_setreg(1 | 23 << 6, 1); }

// 2^(byte - 127) as the instructions that scale by a power of two take it: they read the exponent alone (0: 2^-127).
__device__ __forceinline__ float scale_field(uint32_t byte) { return __uint_as_float(byte << 23); }
// The same as a number: 255 is NaN, and 2^-127 lies below the normal ones.
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return __uint_as_float(byte == 255 ? 0x7fc00000u : byte == 0 ? 0x00400000u : byte << 23);
}

// Four codes times a scale as four values of T (two registers), exact but for values that T cannot hold; plain(): without the scale,
// which a sum over keys then takes outside: that of a score's key (kPlainK), that of a probability's (kPlainV, where T has the
// range). e4m3's conversion has it for nothing.
template <int KIND, bool BF16>
struct Codes;

template <>
struct Codes<kE4m3, true> {
  static constexpr bool kPlainK = false, kPlainV = false;
  typedef float Scale;
  static __device__ __forceinline__ Scale scale(uint32_t byte) { return scale_field(byte); }
  static __device__ __forceinline__ u32x2 four(uint32_t w, Scale s) {
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, true))};
  }
};

template <>
struct Codes<kE4m3, false> {
  static constexpr bool kPlainK = false, kPlainV = false;
  // The conversion's own overflow does not saturate: it takes scales up to 2^7, which 448 stands, and a product the rest (scales
  // past 2^22 count as 2^22).
  struct Scale {
    float field;
    f16x2 rest;
  };
  static __device__ __forceinline__ Scale scale(uint32_t byte) {
    const uint32_t n = (15 + min(max(static_cast<int>(byte) - 134, 0), 15)) << 10;
    return Scale{scale_field(byte == 255 ? 255 : min(byte, 134u)), __builtin_bit_cast(f16x2, n | n << 16)};
  }
  static __device__ __forceinline__ u32x2 four(uint32_t w, Scale s) {
    const f16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s.field, false) * s.rest;
    const f16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s.field, true) * s.rest;
    return u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
  }
};

template <>
struct Codes<kInt8, true> {
  static constexpr bool kPlainK = true, kPlainV = true;
  typedef float Scale;
  static __device__ __forceinline__ Scale scale(uint32_t byte) { return scale_value(byte); }
  static __device__ __forceinline__ u32x2 four(uint32_t w, Scale s) {
    float f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = static_cast<float>(static_cast<int8_t>(w >> (8 * i))) * s;
    // the products have 8 significant bits: their upper halves are the bf16 values
    return u32x2{__builtin_amdgcn_perm(__float_as_uint(f[1]), __float_as_uint(f[0]), 0x07060302u),
                 __builtin_amdgcn_perm(__float_as_uint(f[3]), __float_as_uint(f[2]), 0x07060302u)};
  }
  static __device__ __forceinline__ u32x2 plain(uint32_t w) { return u32x2{i8pair_to_bf16x2(w, 0), i8pair_to_bf16x2(w, 16)}; }
};

template <>
struct Codes<kInt8, false> {
  static constexpr bool kPlainK = true, kPlainV = false;
  typedef f16x2 Scale;
  static __device__ __forceinline__ Scale scale(uint32_t byte) {
    const _Float16 h = static_cast<_Float16>(scale_value(byte));
    return f16x2{h, h};
  }
  static __device__ __forceinline__ u32x2 plain(uint32_t w) {
    // a byte u under the exponent of 1024 is 1024 + u; u = code + 128
    const uint32_t u = w ^ 0x80808080u;
    const f16x2 bias = {static_cast<_Float16>(-1152.f), static_cast<_Float16>(-1152.f)};
    const f16x2 lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + bias;
    const f16x2 hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + bias;
    return u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
  }
  static __device__ __forceinline__ u32x2 four(uint32_t w, Scale s) {
    const u32x2 x = plain(w);
    const uint32_t lo = x[0], hi = x[1];  // (a bit cast of a vector's element takes the vector's first)
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, lo) * s),
                 __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, hi) * s)};
  }
};

// What a factor outside the sum is, and four codes as the sum's operand with it (PLAIN) or without.
template <class C, bool PLAIN>
struct Outside {
  typedef typename C::Scale Scale;
  static __device__ __forceinline__ Scale scale(uint32_t byte) { return C::scale(byte); }
  static __device__ __forceinline__ float times(float x, Scale) { return x; }
  static __device__ __forceinline__ u32x2 four(uint32_t w, Scale s) { return C::four(w, s); }
};
template <class C>
struct Outside<C, true> {
  typedef float Scale;
  static __device__ __forceinline__ Scale scale(uint32_t byte) { return scale_value(byte); }
  static __device__ __forceinline__ float times(float x, Scale s) { return x * s; }
  static __device__ __forceinline__ u32x2 four(uint32_t w, Scale) { return C::plain(w); }
};

// Eight codes as eight values.
template <class C>
__device__ __forceinline__ u32x4 eight(uint32_t lo, uint32_t hi, typename C::Scale s) {
  const u32x2 a = C::four(lo, s), b = C::four(hi, s);
  return u32x4{a[0], a[1], b[0], b[1]};
}

}  // namespace cache8
}  // namespace bp
