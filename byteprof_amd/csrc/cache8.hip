// The append to a paged cache held in 8 bits, and the way back: positions of a cache of either kind as values.

#include "cache8.h"

#include <type_traits>

#include "attention_plan.h"

namespace bp {
namespace cache8 {
namespace {

constexpr int kThreads = 256;

// Types of the values.
struct Bf16 {
  typedef uint16_t Bits;
  static constexpr uint32_t kAbs = 0x7fff, kInf = 0x7f80;
  static __device__ __forceinline__ float value(uint32_t b) { return bf16_bits_to_float(b); }
  static __device__ __forceinline__ uint32_t bits(float f) { return float_to_bf16_bits(f); }
};
struct F16 {
  typedef uint16_t Bits;
  static constexpr uint32_t kAbs = 0x7fff, kInf = 0x7c00;
  static __device__ __forceinline__ float value(uint32_t b) {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(b)));
  }
  static __device__ __forceinline__ uint32_t bits(float f) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(f)); }
};
struct F32 {
  typedef uint32_t Bits;
  static constexpr uint32_t kAbs = 0x7fffffff, kInf = 0x7f800000;
  static __device__ __forceinline__ float value(uint32_t b) { return __uint_as_float(b); }
  static __device__ __forceinline__ uint32_t bits(float f) { return __float_as_uint(f); }
};

// The exponent byte of the least power of two s with amax <= Q s, Q = 1.75 2^8 (e4m3) or 1.984375 2^6 (int8): amax's own exponent
// less Q's, one more where its significand is the greater (the addition then carries into the exponent).
template <int KIND>
__device__ __forceinline__ uint32_t scale_byte(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = KIND == kE4m3 ? static_cast<int>((b + 0x1fffffu) >> 23) - 8 : static_cast<int>((b + 0x01ffffu) >> 23) - 6;
  return max(e, 0);
}

// x / s to the nearest code, ties to even; infinities to the greatest, NaN to NaN (e4m3) or 0 (int8). Two of them.
template <int KIND>
__device__ __forceinline__ uint32_t encode2(float x, float y) {
  if constexpr (KIND == kE4m3) {
    x = fabsf(x) > 448.f ? copysignf(448.f, x) : x;
    y = fabsf(y) > 448.f ? copysignf(448.f, y) : y;
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(x, y, 0, false)) & 0xffffu;
  } else {
    const auto one = [](float v) {
      v = fabsf(v) > 127.f ? copysignf(127.f, v) : v;
      return static_cast<uint32_t>(static_cast<int>(rintf(v != v ? 0.f : v))) & 0xffu;
    };
    return one(x) | one(y) << 8;
  }
}

template <int KIND>
__device__ __forceinline__ float decode(uint32_t code) {
  if constexpr (KIND == kE4m3) return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(code), 0);
  else return static_cast<float>(static_cast<int8_t>(code));
}

struct Append {
  const void* in[2];  // keys, values [tokens, hk, d]
  uint8_t* pages[2];
  uint8_t* scales[2];
  const int* cu;
  const int* lengths;
  const int* table;
  int64_t in_t[2], in_h[2], p_p[2], p_t[2], p_h[2], s_p[2], s_b[2], s_h[2], table_stride;  // elements
  attn::Div page, block, heads, row;  // row: pieces of a row
  int tokens, seqs, pool, max_keys, hk, d, units;
};

// Units of a launch are numbered ahead of what the offsets hold: sequence b's begin at cu[b] / block + 2 b, which leaves every
// sequence as many as its tokens can touch (tokens / block, rounded down, and 2).
__device__ __forceinline__ int first_unit(const Append& a, int b) { return a.block(min(max(a.cu[b], 0), a.tokens)) + 2 * b; }

// The last sequence whose units begin at or before u: a wave asks 64 sequences at a time.
__device__ __forceinline__ int sequence_of(const Append& a, int u, int lane) {
  int lo = 0, n = a.seqs;
  while (true) {
    const int step = (n + kWave - 1) / kWave, at = lane * step;
    const uint64_t below = __ballot(at < n && first_unit(a, lo + min(at, n - 1)) <= u);
    const int l = below ? 63 - __builtin_clzll(below) : 0;
    lo += l * step;
    n = min(step, n - l * step);
    if (step == 1) return lo;
  }
}

// A unit: the new tokens of one sequence in one block of one head, of keys or of values. G threads (a wave, or the workgroup where
// a block has more pieces than a wave holds) take the greatest magnitude, then write the codes; what of the tokens they can hold
// (8 pieces of V elements a thread) is read once. Where the block holds tokens from before the chunk and the scale grows, their
// codes are rounded to it. Bound by memory where there are many (7889 tokens of 16 heads of 128 columns from bf16 to e4m3, 97 MB in
// 22 us, 4.4 TB/s), by the chain of reads of offsets, length, page and row where there are few (one token 5 us).
template <class T, int KIND, int V, int G>
__global__ __launch_bounds__(kThreads) void append8_kernel(Append a) {
  constexpr int HELD = 8, BYTES = V * static_cast<int>(sizeof(typename T::Bits)), WORDS = BYTES > 4 ? BYTES / 4 : 1;
  __shared__ float red[kThreads / kWave];
  const int lane = static_cast<int>(threadIdx.x) & 63, tid = static_cast<int>(threadIdx.x) % G;
  const int index = blockIdx.x * (kThreads / G) + __builtin_amdgcn_readfirstlane(threadIdx.x / G);
  const int kv = index & 1, hu = index >> 1, u = a.heads(hu), h = hu - u * a.hk;
  if (u >= a.units) return;
  const int b = sequence_of(a, u, lane);
  const int begin = min(max(a.cu[b], 0), a.tokens), end = min(max(a.cu[b + 1], begin), a.tokens);
  const int length = max(a.lengths[b], 0), start = length - (end - begin);
  if (u < first_unit(a, b) || end == begin || start >= a.max_keys) return;
  // the block's first position, and the rows of it that are new
  const int64_t at0 = (a.block(max(start, 0)) + static_cast<int64_t>(u - first_unit(a, b))) * a.block.d;
  if (at0 >= min(length, a.max_keys)) return;
  const int at = static_cast<int>(at0);
  const int lo = max(start - at, 0), hi = min(length - at, a.block.d);
  const int n = a.page(at), slot = at - n * a.page.d;
  const int id = a.table[b * a.table_stride + n];
  if (lo >= hi || static_cast<unsigned>(id) >= static_cast<unsigned>(a.pool)) return;
  const typename T::Bits* in = static_cast<const typename T::Bits*>(a.in[kv]) + (end - length + at) * a.in_t[kv] + h * a.in_h[kv];
  uint8_t* out = a.pages[kv] + id * a.p_p[kv] + slot * a.p_t[kv] + h * a.p_h[kv];
  uint8_t* scale = a.scales[kv] + id * a.s_p[kv] + a.block(slot) * a.s_b[kv] + h * a.s_h[kv];
  const bool held = start > at;  // tokens from before the chunk
  const uint32_t had = held ? *scale : 0;

  uint32_t x[HELD][WORDS];
  const int pieces = (hi - lo) * a.row.d;
  const auto load = [&](int i, uint32_t (&w)[WORDS]) {
    const int r = a.row(i), c = i - r * a.row.d;
    const typename T::Bits* p = in + (lo + r) * a.in_t[kv] + c * V;
    if constexpr (V == 1) w[0] = *p;
    else {
#pragma unroll
      for (int j = 0; j < WORDS / 4; ++j) {
        const u32x4 q = reinterpret_cast<const u32x4*>(p)[j];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[4 * j + e] = q[e];
      }
    }
  };
  const auto element = [](const uint32_t (&w)[WORDS], int e) -> uint32_t {
    if constexpr (sizeof(typename T::Bits) == 4) return w[e];
    else return V == 1 ? w[0] : (w[e / 2] >> (16 * (e % 2))) & 0xffffu;
  };
  uint32_t top = 0;
  const auto widen = [&](const uint32_t (&w)[WORDS]) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const uint32_t m = element(w, e) & T::kAbs;
      top = max(top, m < T::kInf ? m : 0u);
    }
  };
#pragma unroll
  for (int j = 0; j < HELD; ++j)
    if (tid + j * G < pieces) load(tid + j * G, x[j]);
#pragma unroll
  for (int j = 0; j < HELD; ++j)
    if (tid + j * G < pieces) widen(x[j]);
  for (int i = tid + HELD * G; i < pieces; i += G) {
    uint32_t w[WORDS];
    load(i, w);
    widen(w);
  }
  float amax = xor_butterfly<true>(T::value(top), MaxOp());
  if constexpr (G > kWave) {
    if (lane == 0) red[threadIdx.x / kWave] = amax;
    __syncthreads();
    amax = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  }
  const uint32_t byte = max(had, scale_byte<KIND>(amax));
  const int inv_byte = 254 - static_cast<int>(byte);
  const float inv = inv_byte < 0 ? 0.f : scale_value(inv_byte);
  const auto store = [&](int i, const uint32_t (&w)[WORDS]) {
    const int r = a.row(i), c = i - r * a.row.d;
    uint8_t* p = out + (lo + r) * a.p_t[kv] + c * V;
    if constexpr (V == 1) {
      *p = static_cast<uint8_t>(encode2<KIND>(T::value(w[0]) * inv, 0.f));
    } else {
      u32x2 y;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        uint32_t half[2];
#pragma unroll
        for (int g = 0; g < 2; ++g)
          half[g] = encode2<KIND>(T::value(element(w, 4 * e + 2 * g)) * inv, T::value(element(w, 4 * e + 2 * g + 1)) * inv);
        y[e] = half[0] | half[1] << 16;
      }
      *reinterpret_cast<u32x2*>(p) = y;
    }
  };
#pragma unroll
  for (int j = 0; j < HELD; ++j)
    if (tid + j * G < pieces) store(tid + j * G, x[j]);
  for (int i = tid + HELD * G; i < pieces; i += G) {
    uint32_t w[WORDS];
    load(i, w);
    store(i, w);
  }
  if (held && byte > had) {
    const int less = static_cast<int>(byte - had);  // a code times 2^-less; from 126 on nothing is left of it
    const float f = less < 126 ? scale_value(127 - less) : 0.f;
    for (int i = tid; i < lo * a.row.d; i += G) {
      const int r = a.row(i), c = i - r * a.row.d;
      uint8_t* p = out + r * a.p_t[kv] + c * V;
      if constexpr (V == 1) {
        *p = static_cast<uint8_t>(encode2<KIND>(decode<KIND>(*p) * f, 0.f));
      } else {
        u32x2 y = *reinterpret_cast<const u32x2*>(p);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t w = 0;
#pragma unroll
          for (int g = 0; g < 2; ++g)
            w |= encode2<KIND>(decode<KIND>(y[e] >> (16 * g) & 0xff) * f, decode<KIND>(y[e] >> (16 * g + 8) & 0xff) * f) << (16 * g);
          y[e] = w;
        }
        *reinterpret_cast<u32x2*>(p) = y;
      }
    }
  }
  if (tid == 0) *scale = static_cast<uint8_t>(byte);
}

constexpr int kPieces = 2;  // of a thread

struct Read {
  const uint8_t* pages[2];
  const uint8_t* scales[2];  // null: the cache holds values
  void* out[2];              // [tokens, hk, d], contiguous
  const int* cu;
  const int* lengths;
  const int* table;
  int64_t p_p[2], p_t[2], p_h[2], s_p[2], s_b[2], s_h[2], table_stride;  // p: bytes
  attn::Div page, block, row, token;  // pieces of a row, of a token
  int tokens, seqs, pool, max_keys;
};

// A piece of 8 columns of a token's head, of keys and of values: codes times their scale in T (KIND e4m3, int8), or the cache's own
// 16 bits. Positions that the table does not have are zeros, a page outside the pool gives NaN. Where the workgroup's tokens lie is
// found once for a token, then all of a thread's pieces are asked for before the first is written. Bound by memory: 24 441 positions of
// 12 heads of 64 columns from int8 to fp16, 113 MB in 25.5 us (4.4 TB/s), two pieces a thread; one 29.5, four 26.5; with the bisection
// and the table ahead of every piece 34.6. 161 positions 4 us.
template <class T, int KIND>
__global__ __launch_bounds__(kThreads) void read_kernel(Read a) {
  constexpr int kCopy = 2, CHUNKS = std::is_same<T, F32>::value ? 2 : 1, SPAN = kThreads * kPieces;
  constexpr int kUnseen = -1, kOutside = -2;
  __shared__ int2 places[SPAN + 1];  // of the workgroup's tokens: the page and the slot in it
  if constexpr (std::is_same<T, F16>::value) saturate_f16();
  const int total = a.tokens * a.token.d;
  for (int base = blockIdx.x * SPAN; base < total; base += gridDim.x * SPAN) {
    const int tok0 = a.token(base), count = a.token(min(base + SPAN, total) - 1) - tok0 + 1;
    if (base != static_cast<int>(blockIdx.x) * SPAN) __syncthreads();  // the last places are read
    for (int t = threadIdx.x; t < count; t += kThreads) {
      const int tok = tok0 + t;
      int lo = 0, hi = a.seqs;  // the last sequence that begins at or before tok
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (a.cu[mid] <= tok) lo = mid;
        else hi = mid;
      }
      int2 at = {kUnseen, 0};
      if (a.seqs > 0) {
        const int begin = a.cu[lo], end = a.cu[lo + 1], pos = max(a.lengths[lo], 0) - (min(end, a.tokens) - tok);
        if (tok >= begin && tok < end && static_cast<unsigned>(pos) < static_cast<unsigned>(a.max_keys)) {
          const int n = a.page(pos), id = a.table[lo * a.table_stride + n];
          at = int2{static_cast<unsigned>(id) < static_cast<unsigned>(a.pool) ? id : kOutside, pos - n * a.page.d};
        }
      }
      places[t] = at;
    }
    __syncthreads();
    u32x4 x[kPieces][2];
    uint32_t byte[kPieces][2];
    int id[kPieces];
#pragma unroll
    for (int u = 0; u < kPieces; ++u) {
      const int i = min(base + u * kThreads + static_cast<int>(threadIdx.x), total - 1);
      const int tok = a.token(i), rest = i - tok * a.token.d, h = a.row(rest), c = rest - h * a.row.d;
      const int2 at = places[tok - tok0];
      id[u] = at.x;
      if (at.x < 0) continue;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const uint8_t* p = a.pages[kv] + at.x * a.p_p[kv] + at.y * a.p_t[kv] + h * a.p_h[kv];
        if constexpr (KIND == kCopy) {
          x[u][kv] = reinterpret_cast<const u32x4*>(p)[c];
        } else {
          byte[u][kv] = a.scales[kv][at.x * a.s_p[kv] + a.block(at.y) * a.s_b[kv] + h * a.s_h[kv]];
          const u32x2 w = reinterpret_cast<const u32x2*>(p)[c];
          x[u][kv][0] = w[0], x[u][kv][1] = w[1];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kPieces; ++u) {
      const int i = base + u * kThreads + static_cast<int>(threadIdx.x);
      if (i >= total) break;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        u32x4 y[CHUNKS] = {};
        if (id[u] >= 0) {
          const u32x4 w = x[u][kv];
          if constexpr (KIND == kCopy) {
            y[0] = w;
          } else if constexpr (CHUNKS == 2) {
            const float s = scale_value(byte[u][kv]);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e / 4][e % 4] = T::bits(decode<KIND>(w[e / 4] >> (8 * (e % 4)) & 0xff) * s);
          } else {
            using C = Codes<KIND, std::is_same<T, Bf16>::value>;
            if constexpr (std::is_same<T, F16>::value) {
              using E = Ends<KIND>;
              const uint32_t b = byte[u][kv];
              if (E::beyond(b)) y[0] = eight<C>(E::codes(w[0], b), E::codes(w[1], b), C::scale(E::byte(b)));
              else y[0] = eight<C>(w[0], w[1], C::scale(b));
            } else {
              y[0] = eight<C>(w[0], w[1], C::scale(byte[u][kv]));
            }
          }
        } else if (id[u] == kOutside) {
          const uint32_t nan = T::bits(NAN), two = CHUNKS == 2 ? nan : nan | nan << 16;
#pragma unroll
          for (int j = 0; j < CHUNKS; ++j) y[j] = u32x4{two, two, two, two};
        }
        u32x4* out = reinterpret_cast<u32x4*>(static_cast<typename T::Bits*>(a.out[kv]) + static_cast<int64_t>(i) * 8);
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j) out[j] = y[j];
      }
    }
  }
}

bool aligned(const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

constexpr int64_t kHeld = 8 * kWave;

template <class T, int KIND, int V>
void append_launch(const Append& a, hipStream_t st) {
  const int64_t pieces = static_cast<int64_t>(a.block.d) * a.row.d, waves = 2ll * a.units * a.hk;
  // a wave holds 512 pieces; past those a workgroup takes the unit, and what is held is still read once
  if (pieces <= kHeld)
    append8_kernel<T, KIND, V, kWave><<<static_cast<unsigned>((waves + 3) / 4), kThreads, 0, st>>>(a);
  else append8_kernel<T, KIND, V, kThreads><<<static_cast<unsigned>(waves), kThreads, 0, st>>>(a);
}

template <class T, int KIND>
void append_vector(const Append& a, bool wide, hipStream_t st) {
  if (wide) append_launch<T, KIND, 8>(a, st);
  else append_launch<T, KIND, 1>(a, st);
}

template <class T>
void append_kind(const Append& a, int kind, bool wide, hipStream_t st) {
  if (kind == BP_DT_E4M3) append_vector<T, kE4m3>(a, wide, st);
  else append_vector<T, kInt8>(a, wide, st);
}

template <class T>
void read_kind(const Read& a, int kind, unsigned grid, hipStream_t st) {
  if (kind == BP_DT_E4M3) read_kernel<T, kE4m3><<<grid, kThreads, 0, st>>>(a);
  else if (kind == BP_DT_I8) read_kernel<T, kInt8><<<grid, kThreads, 0, st>>>(a);
  else read_kernel<T, 2><<<grid, kThreads, 0, st>>>(a);
}

bool sizes_fit(const BpPagedCache* c, int tokens) {
  return c != nullptr && tokens >= 0 && c->seqs >= 0 && c->pool >= 0 && c->page > 0 && c->max_pages >= 0 &&
         static_cast<int64_t>(c->page) * c->max_pages < (1ll << 29) && c->hk >= 0 && c->head_dim >= 0;
}

bool has_codes(const BpPagedCache& c) { return c.dtype == BP_DT_E4M3 || c.dtype == BP_DT_I8; }

}  // namespace
}  // namespace cache8
}  // namespace bp

extern "C" {

int bp_paged_append8(const BpPagedCache* cache, int dtype, const void* k, const void* v, const int32_t* cu, int tokens, int64_t k_t,
                     int64_t k_h, int64_t v_t, int64_t v_h, void* stream) {
  using namespace bp::cache8;
  if (!sizes_fit(cache, tokens)) return BP_E_INVALID_ARG;
  const BpPagedCache& c = *cache;
  if ((dtype != BP_DT_BF16 && dtype != BP_DT_F16 && dtype != BP_DT_F32) || !has_codes(c)) return BP_E_UNSUPPORTED;
  if (c.block <= 0 || c.page % c.block != 0) return BP_E_INVALID_ARG;
  if (tokens == 0 || c.seqs == 0 || c.pool == 0 || c.max_pages == 0 || c.hk == 0 || c.head_dim == 0) return BP_OK;
  if (k == nullptr || v == nullptr || c.k_pages == nullptr || c.v_pages == nullptr || c.k_scales == nullptr ||
      c.v_scales == nullptr || c.table == nullptr || c.lengths == nullptr || cu == nullptr)
    return BP_E_INVALID_ARG;
  Append a = {};
  const void *pages[2] = {c.k_pages, c.v_pages}, *scales[2] = {c.k_scales, c.v_scales};
  const int64_t *page_strides[2] = {c.kp, c.vp}, *scale_strides[2] = {c.ks, c.vs};
  a.in[0] = k, a.in[1] = v;
  a.in_t[0] = k_t, a.in_t[1] = v_t, a.in_h[0] = k_h, a.in_h[1] = v_h;
  const int size = dtype == BP_DT_F32 ? 4 : 2;
  bool wide = c.head_dim % 8 == 0 && aligned(k, 16) && aligned(v, 16) && ((k_t | k_h | v_t | v_h) * size & 15) == 0;
  for (int w = 0; w < 2; ++w) {
    a.pages[w] = static_cast<uint8_t*>(const_cast<void*>(pages[w]));
    a.scales[w] = static_cast<uint8_t*>(const_cast<void*>(scales[w]));
    a.p_p[w] = page_strides[w][0], a.p_t[w] = page_strides[w][1], a.p_h[w] = page_strides[w][2];
    a.s_p[w] = scale_strides[w][0], a.s_b[w] = scale_strides[w][1], a.s_h[w] = scale_strides[w][2];
    wide = wide && aligned(pages[w], 8) && ((a.p_p[w] | a.p_t[w] | a.p_h[w]) & 7) == 0;
  }
  a.cu = cu, a.lengths = c.lengths, a.table = c.table, a.table_stride = c.table_stride;
  a.page = bp::attn::Div::of(c.page), a.block = bp::attn::Div::of(c.block), a.heads = bp::attn::Div::of(c.hk);
  a.row = bp::attn::Div::of(wide ? c.head_dim / 8 : c.head_dim);
  a.tokens = tokens, a.seqs = c.seqs, a.pool = c.pool, a.max_keys = c.page * c.max_pages, a.hk = c.hk, a.d = c.head_dim;
  const int64_t units = tokens / c.block + 2ll * c.seqs;
  const int64_t threads = static_cast<int64_t>(c.block) * a.row.d <= kHeld ? bp::kWave : kThreads;
  // a unit's pieces, positions, and a launch's threads in 32 bits
  if (static_cast<int64_t>(c.block) * c.head_dim >= (1ll << 30) || 2 * units * c.hk >= (1ll << 32) / threads || tokens >= (1 << 30))
    return BP_E_UNSUPPORTED;
  if (c.k_pages == c.v_pages || c.k_scales == c.v_scales) return BP_E_INVALID_ARG;
  a.units = static_cast<int>(units);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == BP_DT_BF16) append_kind<Bf16>(a, c.dtype, wide, st);
  else if (dtype == BP_DT_F16) append_kind<F16>(a, c.dtype, wide, st);
  else append_kind<F32>(a, c.dtype, wide, st);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? BP_OK : static_cast<int>(e);
}

int bp_paged_read(const BpPagedCache* cache, int dtype, void* k, void* v, const int32_t* cu, int tokens, void* stream) {
  using namespace bp::cache8;
  if (!sizes_fit(cache, tokens)) return BP_E_INVALID_ARG;
  const BpPagedCache& c = *cache;
  const bool codes = has_codes(c);
  if (dtype != BP_DT_BF16 && dtype != BP_DT_F16 && dtype != BP_DT_F32) return BP_E_UNSUPPORTED;
  if (!codes && (c.dtype != dtype || dtype == BP_DT_F32)) return BP_E_UNSUPPORTED;
  if (codes && (c.block <= 0 || c.page % c.block != 0)) return BP_E_INVALID_ARG;
  if (c.head_dim % 8 != 0) return BP_E_UNSUPPORTED;
  if (tokens == 0 || c.hk == 0 || c.head_dim == 0) return BP_OK;
  const bool empty = c.seqs == 0 || c.pool == 0 || c.max_pages == 0;
  // (a pool without pages still has its table read)
  if (k == nullptr || v == nullptr || (c.seqs > 0 && (c.lengths == nullptr || cu == nullptr || (c.max_pages > 0 && c.table == nullptr))) ||
      (!empty && (c.k_pages == nullptr || c.v_pages == nullptr || (codes && (c.k_scales == nullptr || c.v_scales == nullptr)))))
    return BP_E_INVALID_ARG;
  const int size = codes ? 1 : 2;
  Read a = {};
  a.out[0] = k, a.out[1] = v;
  const void *pages[2] = {c.k_pages, c.v_pages}, *scales[2] = {c.k_scales, c.v_scales};
  const int64_t *page_strides[2] = {c.kp, c.vp}, *scale_strides[2] = {c.ks, c.vs};
  for (int w = 0; w < 2; ++w) {
    // a stride that nothing is multiplied with may be anything
    const int64_t p = c.pool == 1 ? 0 : page_strides[w][0], t = c.page == 1 ? 0 : page_strides[w][1],
                  h = c.hk == 1 ? 0 : page_strides[w][2];
    if (!aligned(a.out[w], 16) || !aligned(pages[w], 8 * size) || ((p | t | h) & 7) != 0) return BP_E_INVALID_ARG;
    a.pages[w] = static_cast<const uint8_t*>(pages[w]);
    a.scales[w] = static_cast<const uint8_t*>(scales[w]);
    a.p_p[w] = p * size, a.p_t[w] = t * size, a.p_h[w] = h * size;
    a.s_p[w] = scale_strides[w][0], a.s_b[w] = scale_strides[w][1], a.s_h[w] = scale_strides[w][2];
  }
  if (static_cast<int64_t>(tokens) * c.hk * (c.head_dim / 8) >= (1ll << 30)) return BP_E_UNSUPPORTED;
  const int64_t out = static_cast<int64_t>(tokens) * c.hk * c.head_dim * (dtype == BP_DT_F32 ? 4 : 2);
  const auto reach = [&](const int64_t* st, int rows, int last, int bytes) {
    return bytes * ((c.pool - 1) * st[0] + (rows - 1) * st[1] + (c.hk - 1) * st[2] + last);
  };
  if (bp::ranges_overlap(k, out, v, out)) return BP_E_INVALID_ARG;
  for (int w = 0; w < 2 && !empty; ++w)
    for (int o = 0; o < 2; ++o)
      if (bp::ranges_overlap(a.out[o], out, pages[w], reach(page_strides[w], c.page, c.head_dim, size)) ||
          (codes && bp::ranges_overlap(a.out[o], out, scales[w], reach(scale_strides[w], c.page / c.block, 1, 1))))
        return BP_E_INVALID_ARG;
  a.cu = cu, a.lengths = c.lengths, a.table = c.table, a.table_stride = c.table_stride;
  a.page = bp::attn::Div::of(c.page), a.block = bp::attn::Div::of(codes ? c.block : c.page);
  a.row = bp::attn::Div::of(c.head_dim / 8), a.token = bp::attn::Div::of(c.hk * (c.head_dim / 8));
  a.tokens = tokens, a.seqs = c.seqs, a.pool = c.pool, a.max_keys = c.page * c.max_pages;
  const int64_t total = static_cast<int64_t>(tokens) * a.token.d, blocks = (total + kThreads * kPieces - 1) / (kThreads * kPieces);
  const unsigned grid = static_cast<unsigned>(blocks < 16384 ? blocks : 16384);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == BP_DT_BF16) read_kind<Bf16>(a, c.dtype, grid, st);
  else if (dtype == BP_DT_F16) read_kind<F16>(a, c.dtype, grid, st);
  else if (c.dtype == BP_DT_E4M3) read_kernel<F32, kE4m3><<<grid, kThreads, 0, st>>>(a);
  else read_kernel<F32, kInt8><<<grid, kThreads, 0, st>>>(a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? BP_OK : static_cast<int>(e);
}

}  // extern "C"
