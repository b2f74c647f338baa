// Rotary positions of queries and keys: pairs of columns (x1, x2) of a head turned by the angle position x frequency,
//   (x1 cos a - x2 sin a, x2 cos a + x1 sin a) x factor,
// the pairs (i, i + rot / 2) or (2 i, 2 i + 1) of the first rot columns; the others as they are.
//
// Angles: at position 10^6 a float32 product is off by up to 0.03, so position x frequency / 2 pi is formed in 64 bits, whole turns are
// taken off, and the rest goes into sine and cosine in 32 bits. That is done once for a token and frequency, through LDS, and used by
// all heads. Bound by memory: 8192 tokens of 32 + 8 heads of 128 columns in bf16, 168 MB in 34.5 us (4.9 TB/s; 29 us where a part is
// still in the last level's cache); one token 2.2 us, as long as any launch. Vectors are as wide as the halves and the alignment allow,
// 16 bytes down to an element: 5000 such tokens of 128 turned columns 17 us, of 90 (an odd half, elements) 49.

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "common.h"

#include "attention_plan.h"

namespace bp {
namespace rotary {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxDim = 1024;
constexpr int kPairs = 512;  // of the tokens of a workgroup; one token has kMaxDim / 2 at most

struct Bf16 {
  typedef uint16_t Bits;
  static __device__ __forceinline__ float value(uint32_t b) { return bf16_bits_to_float(b); }
  static __device__ __forceinline__ uint32_t bits(float f) { return float_to_bf16_bits(f); }
};
struct F16 {
  typedef uint16_t Bits;
  static __device__ __forceinline__ float value(uint32_t b) {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(b)));
  }
  static __device__ __forceinline__ uint32_t bits(float f) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(f)); }
};
struct F32 {
  typedef uint32_t Bits;
  static __device__ __forceinline__ float value(uint32_t b) { return __uint_as_float(b); }
  static __device__ __forceinline__ uint32_t bits(float f) { return __float_as_uint(f); }
};

struct Args {
  const void* in[2];  // q, k
  void* out[2];
  int64_t in_t[2], in_h[2], out_t[2], out_h[2];  // elements
  const void* positions;
  const float* inv_freq;
  attn::Div token, head, pairs;  // pieces of a token and of a head; pairs of a head
  int64_t tokens;
  int hq, rot, turned, wide_positions, group;  // turned: pieces of a head that turn; group: tokens of a workgroup
  float factor;
};

// V elements: 16, 8 or 4 bytes, or one element.
template <class T, int V>
struct Piece {
  static constexpr int BYTES = V * static_cast<int>(sizeof(typename T::Bits)), W = BYTES < 4 ? 1 : BYTES / 4;
  typedef uint32_t Words __attribute__((ext_vector_type(W)));
  uint32_t w[W];
  __device__ __forceinline__ void load(const typename T::Bits* p) {
    if constexpr (BYTES < 4) w[0] = *p;
    else {
      const Words x = *reinterpret_cast<const Words*>(p);
#pragma unroll
      for (int i = 0; i < W; ++i) w[i] = x[i];
    }
  }
  __device__ __forceinline__ void store(typename T::Bits* p) const {
    if constexpr (BYTES < 4) *p = static_cast<typename T::Bits>(w[0]);
    else {
      Words x;
#pragma unroll
      for (int i = 0; i < W; ++i) x[i] = w[i];
      *reinterpret_cast<Words*>(p) = x;
    }
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (V == 1 || sizeof(typename T::Bits) == 4) return T::value(w[e]);
    else return T::value(w[e / 2] >> (16 * (e % 2)) & 0xffffu);
  }
  __device__ __forceinline__ void set(int e, float f) {
    if constexpr (V == 1 || sizeof(typename T::Bits) == 4) w[e] = T::bits(f);
    else w[e / 2] = e % 2 == 0 ? T::bits(f) : w[e / 2] | T::bits(f) << 16;
  }
};

// A piece of work: V pairs of a head (two vectors, rot / 2 columns apart; interleaved: two neighbouring ones), or V columns that do
// not turn.
template <class T, int V, bool INTER>
__global__ __launch_bounds__(kThreads) void rotary_kernel(Args a) {
  __shared__ float2 turns[kPairs];  // cosine and sine, times factor
  const int64_t tok0 = static_cast<int64_t>(blockIdx.x) * a.group;
  const int toks = static_cast<int>(min(static_cast<int64_t>(a.group), a.tokens - tok0)), half = a.rot / 2;
  for (int i = threadIdx.x; i < toks * half; i += kThreads) {
    const int t = a.pairs(i), f = i - t * half;
    const int64_t pos = a.wide_positions ? static_cast<const int64_t*>(a.positions)[tok0 + t]
                                         : static_cast<const int32_t*>(a.positions)[tok0 + t];
    const double turn = static_cast<double>(pos) * (static_cast<double>(a.inv_freq[f]) * 0.15915494309189533577);
    float s, c;
    sincospif(2.f * static_cast<float>(turn - rint(turn)), &s, &c);
    turns[i] = float2{c * a.factor, s * a.factor};
  }
  __syncthreads();
  for (int i = threadIdx.x; i < toks * a.token.d; i += kThreads) {
    const int t = a.token(i), rest = i - t * a.token.d, h = a.head(rest), p = rest - h * a.head.d;
    const int w = h < a.hq ? 0 : 1, hh = w == 0 ? h : h - a.hq;
    const typename T::Bits* in = static_cast<const typename T::Bits*>(a.in[w]) + (tok0 + t) * a.in_t[w] + hh * a.in_h[w];
    typename T::Bits* out = static_cast<typename T::Bits*>(a.out[w]) + (tok0 + t) * a.out_t[w] + hh * a.out_h[w];
    Piece<T, V> x, y;
    if (p < a.turned) {
      const float2* cs = turns + t * half + p * V;
      const int c0 = INTER ? 2 * p * V : p * V, c1 = INTER ? c0 + V : c0 + half;
      x.load(in + c0);
      y.load(in + c1);
      Piece<T, V> u, v;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float2 r = cs[e];
        // interleaved: pair e lies in elements 2 e, 2 e + 1 of the two vectors one after another
        float x1, x2;
        if constexpr (!INTER || V == 1) x1 = x.get(e), x2 = y.get(e);
        else x1 = 2 * e < V ? x.get(2 * e) : y.get(2 * e - V), x2 = 2 * e < V ? x.get(2 * e + 1) : y.get(2 * e + 1 - V);
        const float y1 = x1 * r.x - x2 * r.y, y2 = x2 * r.x + x1 * r.y;
        if constexpr (!INTER || V == 1) u.set(e, y1), v.set(e, y2);
        else if (2 * e < V) u.set(2 * e, y1), u.set(2 * e + 1, y2);
        else v.set(2 * e - V, y1), v.set(2 * e + 1 - V, y2);
      }
      u.store(out + c0);
      v.store(out + c1);
    } else {
      const int c = a.rot + (p - a.turned) * V;
      x.load(in + c);
      x.store(out + c);
    }
  }
}

template <class T, int V>
void launch_of(const Args& a, bool inter, unsigned grid, hipStream_t st) {
  if (inter) rotary_kernel<T, V, true><<<grid, kThreads, 0, st>>>(a);
  else rotary_kernel<T, V, false><<<grid, kThreads, 0, st>>>(a);
}

template <class T>
void launch(const Args& a, int v, bool inter, unsigned grid, hipStream_t st) {
  constexpr int V = 16 / sizeof(typename T::Bits);
  if (v == V) launch_of<T, V>(a, inter, grid, st);
  else if (v == V / 2) launch_of<T, V / 2>(a, inter, grid, st);
  else if (V / 4 > 1 && v == V / 4) launch_of<T, V / 4>(a, inter, grid, st);
  else launch_of<T, 1>(a, inter, grid, st);
}

// Whether the elements of two tensors [tokens, heads, d] are apart: their ranges are, or they have one token stride and lie in
// different columns of it (slices of one projection).
bool apart(const void* p, int64_t p_t, int64_t p_row, const void* q, int64_t q_t, int64_t q_row, int64_t tokens) {
  if (!ranges_overlap(p, (tokens - 1) * p_t + p_row, q, (tokens - 1) * q_t + q_row)) return true;
  if (p_t != q_t || p_row > p_t || q_row > p_t) return false;
  const int64_t off = static_cast<int64_t>(reinterpret_cast<uintptr_t>(q) - reinterpret_cast<uintptr_t>(p));
  const int64_t m = ((off % p_t) + p_t) % p_t;
  return m >= p_row && m + q_row <= p_t;
}

}  // namespace
}  // namespace rotary
}  // namespace bp

extern "C" int bp_rotary(const BpRotary* rotary, void* stream) {
  using namespace bp::rotary;
  if (rotary == nullptr) return BP_E_INVALID_ARG;
  const auto [q, k, q_out, k_out, positions, inv_freq, tokens, q_st, k_st, qo_st, ko_st, dtype, position_bytes, hq, hk, head_dim, rot,
              interleaved, factor] = *rotary;
  if (dtype != BP_DT_BF16 && dtype != BP_DT_F16 && dtype != BP_DT_F32) return BP_E_UNSUPPORTED;
  if (tokens < 0 || hq < 0 || hk < 0 || head_dim < 0 || rot < 0 || rot % 2 != 0 || rot > head_dim ||
      (position_bytes != 4 && position_bytes != 8) || !(fabsf(factor) <= 3.0e38f) || (q_st[0] | q_st[1] | k_st[0] | k_st[1]) < 0)
    return BP_E_INVALID_ARG;
  if (head_dim > kMaxDim) return BP_E_UNSUPPORTED;
  const int64_t all = static_cast<int64_t>(hq) + hk;
  if (tokens == 0 || all == 0 || head_dim == 0) return BP_OK;
  if ((hq > 0 && (q == nullptr || q_out == nullptr)) || (hk > 0 && (k == nullptr || k_out == nullptr)) ||
      (rot > 0 && (positions == nullptr || inv_freq == nullptr)))
    return BP_E_INVALID_ARG;
  Args a = {};
  const int heads[2] = {hq, hk};
  a.in[0] = q, a.in[1] = k, a.out[0] = q_out, a.out[1] = k_out;
  a.in_t[0] = q_st[0], a.in_t[1] = k_st[0], a.in_h[0] = q_st[1], a.in_h[1] = k_st[1];
  a.out_t[0] = qo_st[0], a.out_t[1] = ko_st[0], a.out_h[0] = qo_st[1], a.out_h[1] = ko_st[1];
  const int size = dtype == BP_DT_F32 ? 4 : 2, V = 16 / size;
  int64_t odd = 0;
  uintptr_t at = 0;
  bool in_place = true;
  for (int w = 0; w < 2; ++w) {
    if (heads[w] == 0) continue;
    // a stride that nothing is multiplied with may be anything
    if (tokens == 1) a.in_t[w] = a.out_t[w] = static_cast<int64_t>(heads[w]) * head_dim;
    if (heads[w] == 1) a.in_h[w] = a.out_h[w] = head_dim;
    // an output's own rows are apart: a head after another within a token, or a token after another within a head
    const int64_t t = a.out_t[w], h = a.out_h[w];
    const bool by_token = h >= head_dim && t >= (heads[w] - 1) * h + head_dim;
    const bool by_head = t >= head_dim && h >= (tokens - 1) * t + head_dim;
    if (!by_token && !by_head) return BP_E_INVALID_ARG;
    odd |= a.in_t[w] | a.in_h[w] | t | h;
    at |= reinterpret_cast<uintptr_t>(a.in[w]) | reinterpret_cast<uintptr_t>(a.out[w]);
    in_place = in_place && a.in[w] == a.out[w] && a.in_t[w] == t && a.in_h[w] == h;
  }
  const int64_t dim = head_dim;
  const auto row = [&](int w, int64_t h) { return size * ((heads[w] - 1) * h + dim); };
  for (int o = 0; o < 2; ++o) {
    if (heads[o] == 0) continue;
    for (int i = 0; i < 4; ++i) {
      const int w = i & 1;
      if (heads[w] == 0 || (i == 2 + o)) continue;  // i < 2: an input; else the other output
      const void* p = i < 2 ? a.in[w] : a.out[w];
      const int64_t t = i < 2 ? a.in_t[w] : a.out_t[w], h = i < 2 ? a.in_h[w] : a.out_h[w];
      if (i == o && p == a.out[o] && t == a.out_t[o] && h == a.out_h[o]) continue;  // in place
      if (!apart(a.out[o], size * a.out_t[o], row(o, a.out_h[o]), p, size * t, row(w, h), tokens)) return BP_E_INVALID_ARG;
    }
    const int64_t reach = size * (tokens - 1) * a.out_t[o] + row(o, a.out_h[o]);
    if (rot > 0 && (bp::ranges_overlap(a.out[o], reach, positions, tokens * position_bytes) ||
                    bp::ranges_overlap(a.out[o], reach, inv_freq, rot / 2 * 4)))
      return BP_E_INVALID_ARG;
  }
  a.positions = positions, a.wide_positions = position_bytes == 8, a.inv_freq = inv_freq;
  a.tokens = tokens, a.hq = hq, a.rot = rot, a.factor = factor;
  const bool inter = interleaved != 0;
  // The widest vectors that rows, halves and heads are made of. (5000 tokens of 40 heads of 128: halves of 64 or 32 17 to 19 us, of 36
  // 21, of 45, an element at a time, 49.)
  int v = V;
  while (v > 1 && !(at % (v * size) == 0 && odd % v == 0 && head_dim % v == 0 && rot % (2 * v) == 0)) v /= 2;
  a.turned = rot / 2 / v;
  const int of_head = a.turned + (in_place ? 0 : (head_dim - rot) / v);
  if (of_head == 0) return BP_OK;
  a.head = bp::attn::Div::of(of_head);
  const int64_t pieces = of_head * all;
  if (pieces >= (1 << 24)) return BP_E_UNSUPPORTED;
  a.token = bp::attn::Div::of(static_cast<int>(pieces));
  a.pairs = bp::attn::Div::of(rot > 0 ? rot / 2 : 1);
  // tokens of a workgroup: a sine and cosine a thread, but fewer where that leaves CUs idle
  int group = rot > 0 ? kThreads / (rot / 2) : kThreads / 16;
  if (group > 16) group = 16;
  while (group > 1 && tokens / group < 1024) group /= 2;
  a.group = group < 1 ? 1 : group;
  const int64_t grid = (tokens + a.group - 1) / a.group;
  if (grid >= (1ll << 24)) return BP_E_UNSUPPORTED;  // threads in 32 bits
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == BP_DT_BF16) launch<Bf16>(a, v, inter, static_cast<unsigned>(grid), st);
  else if (dtype == BP_DT_F16) launch<F16>(a, v, inter, static_cast<unsigned>(grid), st);
  else launch<F32>(a, v, inter, static_cast<unsigned>(grid), st);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? BP_OK : static_cast<int>(e);
}
