// The codes of a cache held in 8 bits: e4m3 (4 exponent and 3 mantissa bits, no infinities, greatest 448) or int8, times a power
// of two for each block of tokens and head, kept as its exponent with bias 127 (255: not a number). A power of two costs e4m3
// nothing (a floating code is as exact at any scale) and int8 half a bit in the mean; in return x / scale and code x scale are
// exact, so a code is the correct rounding of its definition and code x scale, of 8 significant bits at most, is exact in bf16
// (in fp16 rounded once below its normal values; saturate_f16 has those past its range become its greatest: an infinity would turn
// the probabilities 0 of the keys beside it into NaN, and 65504 rounded to e4m3 is 65536).
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
  // The conversion's own overflow does not saturate: it takes scales up to 2^7, which 448 stands, and a product the rest, up to 2^15
  // (Ends has no scale be greater than that).
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
  static __device__ __forceinline__ float outside(uint32_t byte) { return scale_value(byte); }
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
  // (below 2^-31 every code rounds to 0 in fp16)
  static __device__ __forceinline__ float outside(uint32_t byte) { return byte < 96 ? 0.f : scale_value(byte); }
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

// The ends of fp16: one factor, rounded to fp16 itself, is right for a scale in the middle only. Codes at a scale that beyond() names are
// replaced by codes() at the scale byte(), which stand for the same fp16 values. (That happens for blocks of values below 2^-18 or past
// 2^15. A second factor in every product instead costs a verify round over int8 33.1 us to 34.4, a decode batch of int8 heads of 200
// columns, whose registers do not suffice then, 374 to 451; the look at the scales costs them 33.7 and 384.)
template <int KIND>
struct Ends;

// Past 2^22 all normal codes are past fp16's range, there as at 2^22, and a code m below them, m 2^-9, times 2^n is m << n.
template <>
struct Ends<kE4m3> {
  static __device__ __forceinline__ uint32_t beyond(uint32_t byte) { return byte > 149 && byte < 255; }
  static __device__ __forceinline__ uint32_t byte(uint32_t byte) { return beyond(byte) ? 149 : byte; }
  static __device__ __forceinline__ uint32_t codes(uint32_t w, uint32_t byte) {
    const uint32_t n = beyond(byte) ? min(byte - 149, 3u) : 0;
    const uint32_t normal = (((w & 0x78787878u) + 0x78787878u) >> 7 & 0x01010101u) * 0xff;
    return (w & (normal | 0x80808080u)) | (w & 0x07070707u & ~normal) << n;
  }
};

// From 2^-31 to 2^-25 a value is a whole multiple of fp16's least, 2^-24, to the nearest: that multiple is its code at 2^-24. Past 2^9, a
// code whose value is past fp16's range becomes that of 2^16 (as a factor outside of a sum takes it; inside, it is the greatest).
template <>
struct Ends<kInt8> {
  static __device__ __forceinline__ uint32_t beyond(uint32_t byte) { return (byte > 136 && byte < 255) || byte - 96u <= 102u - 96u; }
  static __device__ __forceinline__ uint32_t byte(uint32_t byte) { return beyond(byte) ? byte > 136 ? min(byte, 143u) : 103 : byte; }
  static __device__ __forceinline__ uint32_t codes(uint32_t w, uint32_t byte) {
    const float f = beyond(byte) && byte < 103 ? scale_field(byte + 24) : 1.f;
    const float most = beyond(byte) && byte > 136 ? scale_field(127 + 143 - min(byte, 143u)) : 128.f;
    uint32_t y = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = rintf(static_cast<float>(static_cast<int8_t>(w >> (8 * i))) * f);
      y |= (static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(x, -most), most))) & 0xffu) << (8 * i);
    }
    return y;
  }
};

// int8 codes as fp16 by two factors, 2^e = first x rest, first from 2^-14 to 2^5: a code times first is exact, so that the last product
// alone rounds or saturates. As many products as with one factor (the code's bias goes into the first), and right for every scale: the
// large tiles' form (chunks of 128 columns 169 us to 172, of 64 102 to 105).
struct TwoFactors {
  struct Scale {
    f16x2 factors, bias;  // first and rest; -1152 x first
  };
  static __device__ __forceinline__ Scale scale(uint32_t byte) {
    const int e = static_cast<int>(byte) - 127, n = min(max(e, -14), 5);
    const _Float16 first = __builtin_bit_cast(f16x2, (15 + n) << 10)[0], bias = first * static_cast<_Float16>(-1152.f);
    // (of the rest, below 2^-24 and past 2^15 nothing changes: 127 x 2^-38 rounds to 0, 2^20 is past the greatest)
    const _Float16 rest = byte == 255 ? static_cast<_Float16>(NAN) : static_cast<_Float16>(scale_field(min(max(e - n, -24), 15) + 127));
    return Scale{{first, rest}, {bias, bias}};
  }
  static __device__ __forceinline__ u32x2 four(uint32_t w, Scale s) {
    const uint32_t u = w ^ 0x80808080u;  // as in Codes
    const f16x2 lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u));
    const f16x2 hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u));
    const f16x2 first = s.factors.xx, rest = s.factors.yy;
    const f16x2 x = __builtin_elementwise_fma(lo, first, s.bias) * rest, y = __builtin_elementwise_fma(hi, first, s.bias) * rest;
    return u32x2{__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, y)};
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
  static __device__ __forceinline__ Scale scale(uint32_t byte) { return C::outside(byte); }
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
