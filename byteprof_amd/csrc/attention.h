// Attention of several sequences at once: the pieces of the kernels that do not depend on where a key lies (attention_plan.h: the
// plan of a launch, which every workgroup makes for itself from the device's offsets and lengths).
//
//   out[i, h] = sum_j p_ij v[j, h / group],  p_i = softmax_j(scale q[i, h] . k[j, h / group]),  j <= limit(i)
//
// The rows of a product are (token, query head of the group) pairs of one key head, token-major: row r of a sequence is
// token r / group, head r % group of the group, so the heads that share keys share the loads of them. The scores are
// computed transposed, S^T = K Q^T (32 keys x 32 rows a matrix instruction): a lane then holds scores of one row only, its
// maximum, sum and rescaling are scalars of the lane, and the probabilities, rounded to the tensors' type (the matrix instruction
// takes both operands in one type, and fp32 operands at a fraction of its rate), are the second product's operand where they lie
// (O^T = V^T P^T; its key order is the order in which the first product leaves them). Their sum is that of the unrounded ones.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"

#include "attention_plan.h"

namespace bp {
namespace attn {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

struct Bf16 {
  static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){x, y}, bf16x2));
  }
  static __device__ __forceinline__ uint32_t result(float x, float y) { return pack(x, y); }
};
struct F16 {
  static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, (h2){static_cast<_Float16>(x), static_cast<_Float16>(y)});
  }
  // The mean of values near fp16's greatest is no more than that, but rounded probabilities may add up to 1 + 2^-11, and from
  // 65504 (1 + 2^-12) on a result would be infinite. Infinities (of infinite values) stay.
  static __device__ __forceinline__ float finite(float x) { return fabsf(x) < INFINITY ? fminf(fmaxf(x, -65504.f), 65504.f) : x; }
  static __device__ __forceinline__ uint32_t result(float x, float y) { return pack(finite(x), finite(y)); }
};

// LDS images of key and value rows: [row][DP / 8] chunks of 16 bytes, the chunk of a row at a place that the row turns, so
// that 16 rows' equal chunks (the first product's operand) or 4 rows' 64 bytes (the second's) lie in different banks.
// Chunks past the head's own d / 8 are never loaded; they are zeroed once.
template <int DP>
__device__ __forceinline__ int k_place(int row, int chunk) {
  constexpr int CH = DP / 8;
  if constexpr (CH == 8) return row * CH + (chunk ^ ((row >> 1) & 7));
  else if constexpr (CH == 12) return row * CH + (chunk ^ ((row >> 2) & 3));
  else return row * CH + (chunk ^ (row & 15));
}
template <int DP>
__device__ __forceinline__ int v_place(int row, int chunk) {
  constexpr int CH = DP / 8;
  if constexpr (CH == 8) return row * CH + (chunk ^ (4 * ((row >> 1) & 1)));
  else if constexpr (CH == 12) return row * CH + chunk;
  else return row * CH + (chunk ^ (4 * (row & 3)));
}
// Chunk that lies at `place` of a row (the turns are their own inverses).
template <int DP, bool V>
__device__ __forceinline__ int chunk_at(int row, int place) {
  constexpr int CH = DP / 8;
  return (V ? v_place<DP>(row, place) : k_place<DP>(row, place)) - row * CH;
}

// 16 bytes per active lane from `src` to LDS at base + 16 x lane (base: wave-uniform byte address), without a register.
// (m0 is the compiler's only between instructions that it emits together.) Counted by vmcnt: the wave waits with wait_vm before
// it, or after a barrier another wave, reads them.
__device__ __forceinline__ void load_lds16(const void* src, uint32_t base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(__builtin_amdgcn_readfirstlane(base)), "v"(src)
               : "memory");
}
// The same from a wave-uniform address plus a lane's own unsigned byte offset (a scalar that a vector instruction wrote, such
// as a lane's value, may be an address five states later at the earliest).
__device__ __forceinline__ void load_lds16(const void* src, uint32_t offset, uint32_t base) {
  const uint64_t p = reinterpret_cast<uint64_t>(src);
  const uint64_t lo = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(p)));
  const uint64_t hi = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(p >> 32)));
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(base)),
               "v"(offset), "s"(hi << 32 | lo)
               : "memory");
}
// 4 bytes per active lane, to base + 4 x lane.
__device__ __forceinline__ void load_lds4(const void* src, uint32_t base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(__builtin_amdgcn_readfirstlane(base)), "v"(src)
               : "memory");
}
// Waits until at most N of the wave's vector-memory loads are outstanding; wait_lds until no LDS access is. As builtins and not
// as asm: the compiler then knows that its own earlier loads have arrived too. Not knowing, it waited in every step for the
// query's registers, and with them for the next tile's loads.
__device__ constexpr int vm_count(int n) { return (n & 0xF) | ((n >> 4) << 14) | (0x7 << 4) | (0xF << 8); }
template <int N>
__device__ __forceinline__ void wait_vm() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(vm_count(N));
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ void wait_lds() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xF | (3 << 14) | (0x7 << 4));
  asm volatile("" ::: "memory");
}

__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
      (__attribute__((address_space(3))) const void*)(p)));
}

// S^T of 32 keys x 32 rows over DP / 16 steps: K rows from an LDS image, Q from registers.
template <class T, int DP>
__device__ __forceinline__ f32x16 scores(const u32x4* kimg, int row0, const u32x4 (&q)[DP / 16], int lane) {
  f32x16 s = {};
  const int row = row0 + (lane & 31), half = lane >> 5;
#pragma unroll
  for (int i = 0; i < DP / 16; ++i) s = T::mfma(kimg[k_place<DP>(row, 2 * i + half)], q[i], s);
  return s;
}

// O^T += V^T P^T over 32 keys whose probabilities are p (16 per lane, in the order of the scores).
template <class T, int DP>
__device__ __forceinline__ void weighted(const u32x4* vimg, int row0, const u32x4 (&p)[2], f32x16 (&o)[DP / 32], int lane) {
  typedef __attribute__((address_space(3))) s16x4* lds4;
  const int half = lane >> 5, sub = (lane >> 4) & 1, j = (lane & 15) >> 2, e = lane & 3;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) {
      u32x4 a;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        // a 16-lane group reads 4 keys x 16 columns, 4 columns a lane, and gets them transposed: its column's 4 keys
        const int key = row0 + 16 * t + 8 * u + 4 * half + j;
        const int place = v_place<DP>(key, 4 * db + 2 * sub + (e >> 1));
        const char* at = reinterpret_cast<const char*>(vimg + place) + 8 * (e & 1);
        const s16x4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(__attribute__((address_space(3))) void*)at);
        const u32x2 w = __builtin_bit_cast(u32x2, r);
        a[2 * u] = w[0];
        a[2 * u + 1] = w[1];
      }
      o[db] = T::mfma(a, p[t], o[db]);
    }
  }
}

__device__ __forceinline__ float max_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float add_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Exponents are fma(score, c, -M) with M = m c rounded once, m the row's greatest score and c = scale log2(e); the sums are
// relative to M. From kFar on a step of M is more than 1: what its rounding leaves goes into the exponents, past fp16's range from
// 2^28 on and past exp2's from 2^31. There the difference of the scores is taken first, and the sums are relative to m itself.
// (Looking for such rows in every step costs 0 to 1.5% up to 128 columns, and packed prompts of 256 columns, one wave a SIMD, 3 to
// 4%: 2 x 4096 tokens 313 us against 301. With the test kept from step to step in a scalar or a register they took 312 to 322 us, and
// paged chunks of 128 columns 173 us in place of 167: the scalars no longer fit.)
constexpr float kFar = 16777216.f;

// What sums relative to the maximum `from` are multiplied by when `to`, no less, takes its place.
__device__ __forceinline__ float rescaled(float from, float to, float c) {
#pragma clang fp contract(off)
  const float a = from * c, b = to * c;
  return from == to ? 1.f : __builtin_amdgcn_exp2f(fabsf(b) < kFar ? a - b : (from - to) * c);
}

// The running softmax of one row (both halves of a wave hold the row's maximum, unscaled; each its own part of the sum).
template <int DP>
struct Running {
  f32x16 o[DP / 32];
  float m, l;
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) o[i] = f32x16{};
    m = -INFINITY;
    l = 0.f;
  }
};

// One step over NB x 32 keys from position key0: masks past the row's limit, the new maximum, the probabilities.
template <class T, int DP, int NB>
__device__ __forceinline__ void softmax_step(f32x16 (&s)[NB], u32x4 (&p)[NB][2], Running<DP>& r, float c, int key0, int limit,
                                             bool mask, int lane) {
  if (mask) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = key0 + 32 * b + 8 * (i / 4) + 4 * (lane >> 5) + i % 4;
        if (key > limit) s[b][i] = -INFINITY;
      }
  }
  float mx = s[0][0];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[b][i]);
  const float m = fmaxf(r.m, max_halves(mx));
  if (__any(m > r.m)) {
    // exp2(-inf - m) = 0 clears a row's empty start; a row that has seen nothing keeps m = -inf and scales by 1
    const float f = rescaled(r.m, m, c);
    r.m = m;
    r.l *= f;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) r.o[d][i] *= f;
  }
  float shift = r.m == -INFINITY ? 0.f : -(r.m * c);
  if (__any(!(fabsf(shift) < kFar))) {
    const float less = fabsf(shift) < kFar ? 0.f : r.m;
    shift = fabsf(shift) < kFar ? shift : 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[b][i] -= less;
  }
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[b][i] = __builtin_amdgcn_exp2f(fmaf(s[b][i], c, shift));
      r.l += s[b][i];
    }
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) p[b][t][i] = T::pack(s[b][8 * t + 2 * i], s[b][8 * t + 2 * i + 1]);
}

}  // namespace attn
}  // namespace bp
