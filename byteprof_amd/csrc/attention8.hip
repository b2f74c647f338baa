// Attention of chunks of new tokens over a paged cache held in 8 bits (cache8.h: the codes; attention.h: the mathematics of the
// tiles; attention_plan.h: the plan). A position's codes become values of the queries' type, exactly, on their way to the matrix
// instructions; from there on everything is as over a cache in 16 bits.

#include "attention_rows.h"
#include "cache8.h"

#include <float.h>

#include <type_traits>

#include "byteprof_amd.h"

namespace bp {
namespace attn {

// The launch's arguments: those of the 16-bit kernels (k, v: the codes) and the scales' places.
struct Args8 : Args {
  const uint8_t* ks;  // [pool, blocks of a page, hk]
  const uint8_t* vs;
  int64_t ks_p, ks_b, ks_h, vs_p, vs_b, vs_h;
  Div block;
  int wide;  // 16 codes at a time: all rows lie on 16 bytes and are made of them
  int even;  // pages of whole 16 positions, blocks that are whole 16s or parts of one, and keys and values laid out alike
};

namespace {

// The cache as an item sees it. Ids of pages are looked up ahead of the loads that need them.
struct Cache {
  const uint8_t* k;
  const uint8_t* v;
  const uint8_t* ks;
  const uint8_t* vs;
  const int* pages;
  int last;  // the item's last key
  bool bad;  // a page outside the pool: the item's rows become NaN

  __device__ __forceinline__ Cache(const Args8& a, const Item& it, int kvh) {
    k = static_cast<const uint8_t*>(a.k) + kvh * a.k_h;
    v = static_cast<const uint8_t*>(a.v) + kvh * a.v_h;
    ks = a.ks + kvh * a.ks_h;
    vs = a.vs + kvh * a.vs_h;
    pages = a.table + static_cast<int64_t>(it.b) * a.table_stride;
    last = it.key1 - 1;
    bad = false;
  }
  __device__ __forceinline__ int id(const Args8& a, int key) const { return pages[a.page(min(key, last))]; }
  // Where a key's row of codes and its scales lie; n: what id() gave for it.
  __device__ __forceinline__ void at(const Args8& a, int key, int n, int64_t& ko, int64_t& vo, int64_t& kso, int64_t& vso) {
    key = min(key, last);
    const int slot = key - a.page(key) * a.page.d, blk = a.block(slot);
    if (static_cast<unsigned>(n) >= static_cast<unsigned>(a.pool)) {
      bad = true;
      n = 0;
    }
    ko = n * a.k_p + slot * a.k_t;
    vo = n * a.v_p + slot * a.v_t;
    kso = n * a.ks_p + blk * a.ks_b;
    vso = n * a.vs_p + blk * a.vs_b;
  }
};

// 16 keys from a multiple of 16 on, where the cache is even (Args8::even): they lie in one page, and in one block or in whole blocks,
// so that their addresses are a wave's, with offsets of the lanes that do not change. Of the item's last keys, those that there are:
// `rest` of them after the first.
struct Sixteen {
  const uint8_t* k;
  const uint8_t* v;
  const uint8_t* ks;
  const uint8_t* vs;
  int rest;

  __device__ __forceinline__ Sixteen(const Args8& a, Cache& c, int key, int id) {
    key = min(key, c.last & ~15);
    rest = c.last - key;
    const uint32_t slot = key - a.page(key) * a.page.d, blk = a.block(slot);
    uint32_t n = __builtin_amdgcn_readfirstlane(id);
    if (n >= static_cast<uint32_t>(a.pool)) {
      c.bad = true;
      n = 0;
    }
    const uint64_t at = static_cast<uint64_t>(n) * static_cast<uint32_t>(a.k_p) + slot * static_cast<uint32_t>(a.k_t);
    const uint64_t sat = static_cast<uint64_t>(n) * static_cast<uint32_t>(a.ks_p) + blk * static_cast<uint32_t>(a.ks_b);
    k = c.k + at;
    v = c.v + at;
    ks = c.ks + sat;
    vs = c.vs + sat;
  }
};

// 16 codes from column 16 c of a row; of heads that are not whole tiles, zeros past the head's own columns.
template <bool FULL>
__device__ __forceinline__ u32x4 codes16(const Args8& a, const uint8_t* row, int c) {
  if (FULL || (a.wide && 16 * c < a.d)) return *reinterpret_cast<const u32x4*>(row + 16 * c);
  u32x4 r = {};
  if (!a.wide) {
    if (16 * c < a.d) {
      const u32x2 x = *reinterpret_cast<const u32x2*>(row + 16 * c);
      r[0] = x[0], r[1] = x[1];
    }
    if (16 * c + 8 < a.d) {
      const u32x2 x = *reinterpret_cast<const u32x2*>(row + 16 * c + 8);
      r[2] = x[0], r[3] = x[1];
    }
  }
  return r;
}

// How few rows a tile has: 16 RB of them, for launches whose sequences have no more (RB: 1, 2 or 3), and RB = 2 for the small
// sequences beside large ones.
template <int DP, int RB>
struct Few {
  static constexpr int kImages = kWaves * 2 * 32 * DP / 16;        // a wave's keys and values of a step, 16-byte chunks
  static constexpr int kMost = RB == 1 ? 128 : RB == 2 ? 64 : 32;  // columns of a round of the waves' join: 32 KB at most
  static constexpr int G = DP < kMost ? DP : kMost;
  static constexpr int kJoin = kWaves * 16 * RB * G / 4;
  // The queries of 48 rows are operands in LDS, 64 lanes' 16 bytes each, behind the images: beside the sums there are no registers
  // for them, and what the compiler then puts aside is fetched behind the loads that are out (a verify round of six sequences, fp16
  // over int8, 38.6 us without, 32.7 with).
  static constexpr bool kQueries = RB > 2;
  static constexpr int kAhead = kImages + (kQueries ? RB * DP / 32 * kWave : 0);
  static constexpr int kChunks = kAhead > kJoin ? kAhead : kJoin;
  static constexpr int kStats = 16 * RB * (2 * kWaves + 1);
};

__device__ __forceinline__ f32x4 mfma16(Bf16, u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(F16, u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Place of 16-code chunk `chunk` of a row in a wave's image of 32 rows: 8 rows written, and the 16 rows that two 16-lane groups
// read transposed (4 and 4, 16 apart, of either), lie in different banks.
template <int DP>
__device__ __forceinline__ int place16(int row, int chunk) {
  constexpr int CH = DP / 16;
  const int high = row >> 4 & 1;
  if constexpr (CH == 4) return row * CH + (chunk ^ ((row >> 2 & 1) | high << 1));
  else if constexpr (CH == 8) return row * CH + (chunk ^ ((row >> 1 & 3) | high << 2));
  else return row * CH + (chunk ^ ((row & 7) | high << 3));
}

// 16 RB rows; every wave has all of them and takes every fourth block of 32 keys, then the waves' parts are joined. A lane has rows
// lane % 16 of each 16: of 16 keys' scores (S^T = K Q^T, 16 x 16) four, keys 4 (lane / 16) + 0..3; those of 32 keys are the operand
// of O^T = V^T P^T where they lie, whose values come transposed from LDS in the same order of the keys. Codes become operands
// once for all rows.
template <class T, int KIND, int DP, bool FULL, int RB>
__device__ __forceinline__ void few_rows(const Args8& a, const Item& it, int kvh, u32x4* smem, float* stats) {
  using S = Few<DP, RB>;
  using C = cache8::Codes<KIND, std::is_same<T, Bf16>::value>;
  using E = cache8::Ends<KIND>;
  using K = cache8::Outside<C, C::kPlainK>;
  using V = cache8::Outside<C, C::kPlainV>;
  constexpr int NC = DP / 64, STEP = 32 * kWaves;
  // Rows of codes go from memory to registers as they lie, a row's 16-byte chunks on neighbouring lanes, a step ahead; through LDS
  // they become operands. (Keys straight in their operand's layout, a row to a lane: every lane then asks for a line of its own, and
  // the address unit is busy half of the time.)
  constexpr int CH = DP / 16, RPI = kWave / CH, N = 32 / RPI, M = 16 / RPI;  // rows of a load, loads of a step and of 16 keys
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), row = lane & 15, g = lane >> 4;
  const int top = it.row0 + it.rows - 1;
  u32x4 q[S::kQueries ? 1 : RB][2 * NC];
  u32x4* queries = smem + S::kImages;
  int limit[RB];
#pragma unroll
  for (int x = 0; x < RB; ++x) {
    const int mine = min(it.row0 + 16 * x + row, top), n = a.group(mine);
    limit[x] = min(it.first + n, it.keys - 1);
    if (S::kQueries && wave != x) continue;
    const uint16_t* p = static_cast<const uint16_t*>(a.q) + static_cast<int64_t>(it.begin + n) * a.q_t +
                        static_cast<int64_t>(kvh * a.group.d + mine - n * a.group.d) * a.q_h;
#pragma unroll
    for (int i = 0; i < 2 * NC; ++i) {
      const int col = 64 * (i / 2) + 16 * g + 8 * (i % 2);
      const u32x4 y = FULL || col < a.d ? *reinterpret_cast<const u32x4*>(p + col) : u32x4{};
      if constexpr (S::kQueries) queries[(x * 2 * NC + i) * kWave + lane] = y;
      else q[x][i] = y;
    }
  }
  const auto query = [&](int x, int i) {
    if constexpr (S::kQueries) return queries[(x * 2 * NC + i) * kWave + lane];
    else return q[x][i];
  };
  const int least = __builtin_amdgcn_readfirstlane(limit[0]);
  const float c = a.scale_log2;
  f32x4 o[RB][DP / 16];
  float m[RB], l[RB];
#pragma unroll
  for (int x = 0; x < RB; ++x) {
    m[x] = -INFINITY;
    l[x] = 0.f;
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) o[x][d] = f32x4{};
  }
  Cache cache(a, it, kvh);
  u32x4* kimg = smem + wave * 2 * 32 * CH;
  u32x4* vimg = kimg + 32 * CH;
  const int lr = lane / CH, lc = lane % CH;
  u32x4 kc[N], vc[N];
  int ks[2], vs[2], id[2];
  const uint32_t k_t = static_cast<uint32_t>(a.k_t);
  const auto part_of = [&](int r) { return static_cast<uint32_t>(a.block(r)) * static_cast<uint32_t>(a.ks_b); };
  const int k_key = C::kPlainK ? 4 * g : row;  // the first product's operand is of key `row` of 16, its result of 4 g + 0..3
  const uint32_t at_lane = lr * k_t + 16 * lc, ks_lane = FULL ? part_of(k_key) : 0, vs_lane = FULL ? part_of(4 * g) : 0;
  // Every load is sent, past the item's keys from its last ones over again. Scales: of key k_key of 16, and of keys 4 g + 0..3 (the
  // second product's operand); not FULL: of key lane % 32, to be fetched from there.
  const auto load = [&](int at) {
    if constexpr (FULL) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const Sixteen x(a, cache, at + 16 * b, id[b]);
        if (x.rest >= 15) {
          ks[b] = x.ks[ks_lane];
          vs[b] = x.vs[vs_lane];
#pragma unroll
          for (int j = 0; j < M; ++j) kc[b * M + j] = *reinterpret_cast<const u32x4*>(x.k + j * RPI * k_t + at_lane);
#pragma unroll
          for (int j = 0; j < M; ++j) vc[b * M + j] = *reinterpret_cast<const u32x4*>(x.v + j * RPI * k_t + at_lane);
        } else {
          ks[b] = x.ks[part_of(min(k_key, x.rest))];
          vs[b] = x.vs[part_of(min(4 * g, x.rest))];
#pragma unroll
          for (int j = 0; j < M; ++j) {
            const uint32_t off = min(j * RPI + lr, x.rest) * k_t + 16 * lc;
            kc[b * M + j] = *reinterpret_cast<const u32x4*>(x.k + off);
            vc[b * M + j] = *reinterpret_cast<const u32x4*>(x.v + off);
          }
        }
        id[b] = cache.id(a, at + STEP + 16 * b);
      }
    } else {
      int64_t ko, vo, kso, vso;
      cache.at(a, at + lane % 32, id[0], ko, vo, kso, vso);
      ks[0] = cache.ks[kso];
      vs[0] = cache.vs[vso];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        kc[j] = codes16<false>(a, cache.k + __shfl(ko, j * RPI + lr), lc);
        vc[j] = codes16<false>(a, cache.v + __shfl(vo, j * RPI + lr), lc);
      }
      id[0] = cache.id(a, at + STEP + lane % 32);
    }
  };
  int key = it.key0 + 32 * wave;
  if (key < it.key1) {
    id[0] = cache.id(a, FULL ? key : key + lane % 32);
    if constexpr (FULL) id[1] = cache.id(a, key + 16);
    load(key);
  }
  if constexpr (S::kQueries) __syncthreads();
  for (; key < it.key1; key += STEP) {
#pragma unroll
    for (int j = 0; j < N; ++j) kimg[place16<DP>(j * RPI + lr, lc)] = kc[j];
#pragma unroll
    for (int j = 0; j < N; ++j) vimg[place16<DP>(j * RPI + lr, lc)] = vc[j];
    if constexpr (std::is_same<T, F16>::value) {  // codes at scales near fp16's ends become others
      if (__any(E::beyond(ks[0]) | E::beyond(vs[0]) | (FULL ? E::beyond(ks[1]) | E::beyond(vs[1]) : 0))) {
        // (a row's scales lie in the lanes that load() says)
#pragma unroll 1
        for (int i = lane; i < 32 * CH; i += kWave) {
          const int r = i / CH, at = place16<DP>(r, i % CH), four = FULL ? (r & 15) / 4 * 16 : r, k_lane = FULL && !C::kPlainK ? r & 15 : four;
          int kb = __shfl(ks[0], k_lane), vb = __shfl(vs[0], four);
          if constexpr (FULL) {
            const int k_high = __shfl(ks[1], k_lane), v_high = __shfl(vs[1], four);
            kb = r < 16 ? kb : k_high, vb = r < 16 ? vb : v_high;
          }
          u32x4 k = kimg[at], v = vimg[at];
#pragma unroll
          for (int e = 0; e < 4; ++e) k[e] = E::codes(k[e], kb), v[e] = E::codes(v[e], vb);
          kimg[at] = k;
          vimg[at] = v;
        }
#pragma unroll
        for (int b = 0; b < (FULL ? 2 : 1); ++b) ks[b] = E::byte(ks[b]), vs[b] = E::byte(vs[b]);
      }
    }
    typename K::Scale k_scale[2];
    typename V::Scale v_scale[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      k_scale[b] = K::scale(FULL ? ks[b] : __shfl(ks[0], 16 * b + k_key));
      v_scale[b] = V::scale(FULL ? vs[b] : __shfl(vs[0], 16 * b + 4 * g));
    }
    load(key + STEP);
    f32x4 s[RB][2];
#pragma unroll
    for (int x = 0; x < RB; ++x) s[x][0] = s[x][1] = f32x4{};
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      u32x4 k[2][2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const u32x4 w = kimg[place16<DP>(16 * b + row, 4 * i + g)];
        k[b][0] = cache8::eight<K>(w[0], w[1], k_scale[b]);
        k[b][1] = cache8::eight<K>(w[2], w[3], k_scale[b]);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int x = 0; x < RB; ++x) {
          const u32x4 y = query(x, 2 * i + h);
#pragma unroll
          for (int b = 0; b < 2; ++b) s[x][b] = mfma16(T(), k[b][h], y, s[x][b]);
        }
    }
#pragma unroll
    for (int x = 0; x < RB; ++x)
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[x][b][i] = K::times(s[x][b][i], k_scale[b]);
    if (key + 31 > min(least, cache.last)) {
#pragma unroll
      for (int x = 0; x < RB; ++x)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (key + 16 * b + 4 * g + i > min(limit[x], cache.last)) s[x][b][i] = -INFINITY;
    }
    u32x4 p[RB];
#pragma unroll
    for (int x = 0; x < RB; ++x) {
      float mx = s[x][0][0];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[x][b][i]);
      mx = fmaxf(m[x], xor_stage<32>(xor_stage<16>(mx, MaxOp()), MaxOp()));
      if (__any(mx > m[x])) {
        const float f = rescaled(m[x], mx, c);
        m[x] = mx;
        l[x] *= f;
#pragma unroll
        for (int d = 0; d < DP / 16; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[x][d][i] *= f;
      }
      // as in softmax_step: far from zero the difference is taken first
      float shift = m[x] == -INFINITY ? 0.f : -(m[x] * c);
      if (__any(!(fabsf(shift) < kFar))) {
        const float less = fabsf(shift) < kFar ? 0.f : m[x];
        shift = fabsf(shift) < kFar ? shift : 0.f;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[x][b][i] -= less;
      }
#pragma unroll
      for (int b = 0; b < 2; ++b) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[x][b][i] = __builtin_amdgcn_exp2f(fmaf(s[x][b][i], c, shift));
          l[x] += s[x][b][i];
        }
        const auto weight = [&](int i) { return V::times(s[x][b][i], v_scale[b]); };
        p[x][2 * b] = T::pack(weight(0), weight(1));
        p[x][2 * b + 1] = T::pack(weight(2), weight(3));
      }
    }
    typedef int i32x2 __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) i32x2* lds2;
    const int j = row >> 1, from = 16 * (j >> 2) + 4 * g + (j & 3);
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) {
      // a 16-lane group reads 8 keys x 16 columns, 8 columns a lane, and gets them transposed: its column's 8 keys
      const char* at = reinterpret_cast<const char*>(vimg + place16<DP>(from, d)) + 8 * (row & 1);
      const i32x2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds2)(__attribute__((address_space(3))) void*)at);
      const u32x2 v0 = V::four(w[0], v_scale[0]), v1 = V::four(w[1], v_scale[1]);
#pragma unroll
      for (int x = 0; x < RB; ++x) o[x][d] = mfma16(T(), u32x4{v0[0], v0[1], v1[0], v1[1]}, p[x], o[x][d]);
    }
  }
  const bool bad = __any(cache.bad);
  // The waves' parts are joined. stats: [wave][rows] maxima, [wave][rows] sums, [rows] factors of the result.
  constexpr int R = 16 * RB;
#pragma unroll
  for (int x = 0; x < RB; ++x) {
    l[x] = bad ? NAN : xor_stage<32>(xor_stage<16>(l[x], AddOp()), AddOp());
    if (lane < 16) {
      stats[R * wave + 16 * x + lane] = m[x];
      stats[R * (kWaves + wave) + 16 * x + lane] = l[x];
    }
  }
  __syncthreads();
  const bool whole = !it.divided, keep = whole || it.slot + it.split < a.slots;
  const int wd = a.d <= 64 ? 64 : a.d <= 96 ? 96 : DP;  // columns of a slot
  float* ws = whole ? nullptr : a.ws + (static_cast<int64_t>(it.slot + it.split) * a.hk.d + kvh) * a.ws_rows * (wd + 2);
  float f[RB];
#pragma unroll
  for (int x = 0; x < RB; ++x) {
    float all_m = -INFINITY, all_l = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) all_m = fmaxf(all_m, stats[R * w + 16 * x + row]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
      all_l += stats[R * (kWaves + w) + 16 * x + row] * rescaled(stats[R * w + 16 * x + row], all_m, c);
    f[x] = rescaled(m[x], all_m, c);
    if (wave == 0 && lane < 16) {
      stats[R * 2 * kWaves + 16 * x + lane] = whole ? inverse(all_l) : 1.f;
      if (!whole && keep && 16 * x + lane < it.rows) {
        ws[a.ws_rows * wd + 16 * x + lane] = all_m;
        ws[a.ws_rows * (wd + 1) + 16 * x + lane] = all_l;
      }
    }
  }
  f32x4* parts = reinterpret_cast<f32x4*>(smem);  // [wave][4 columns][rows]
  constexpr int G = S::G;
#pragma unroll
  for (int r = 0; r < DP / G; ++r) {
#pragma unroll
    for (int x = 0; x < RB; ++x) {
      if (16 * x + row < it.rows) {
#pragma unroll
        for (int d = 0; d < G / 16; ++d) {
          const f32x4 y = o[x][r * (G / 16) + d];
          parts[(wave * (G / 4) + 4 * d + g) * R + 16 * x + row] = f32x4{y[0] * f[x], y[1] * f[x], y[2] * f[x], y[3] * f[x]};
        }
      }
    }
    __syncthreads();
    for (int i = tid; i < it.rows * (G / 4); i += kThreads) {
      const int rw = i / (G / 4), piece = i % (G / 4), col = 4 * piece + r * G;
      f32x4 y = parts[piece * R + rw];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) y += parts[(w * (G / 4) + piece) * R + rw];
      if (whole) {
        const float inv = stats[R * 2 * kWaves + rw];
        if (col < a.d)
          *reinterpret_cast<u32x2*>(out_row(a, it, kvh, it.row0 + rw) + col) =
              u32x2{T::pack(y[0] * inv, y[1] * inv), T::pack(y[2] * inv, y[3] * inv)};
      } else if (keep && col < wd) {
        *reinterpret_cast<f32x4*>(ws + rw * wd + col) = y;
      }
    }
    if (r + 1 < DP / G) __syncthreads();
  }
}

// Launches of few rows a sequence. Bound by the codes' way from memory: 64 contexts of 64 to 8100 keys, 8 key heads of 128 columns,
// 540 MB in 119 us with the merge of their parts (4.5 TB/s; the kernel alone 112 us, 4.8 TB/s), against 201 us over the same positions
// in 16 bits; three contexts of 9000 to 65537 keys, 16 heads of 64 columns in int8, 235 MB in 65 us (the kernel alone 57, the merge
// 7). A launch of one token is 6 us, finding the item, the first load and the join of the waves one behind the other.
template <class T, int KIND, int DP, bool FULL, int RB>
__global__ __launch_bounds__(kThreads, FewTiles<RB>::workgroups_a_cu(DP)) void attention8_few_kernel(Args8 a) {
  __shared__ __align__(16) u32x4 smem[Few<DP, RB>::kChunks];
  __shared__ float stats[Few<DP, RB>::kStats];
  if constexpr (std::is_same<T, F16>::value) cache8::saturate_f16();
  // Workgroup b runs on XCD b % 8: a part's key heads, whose rows lie side by side, go to one XCD. (With a head to an XCD, as
  // b % hk deals them where hk is 8 or 16, an XCD asks for every eighth 128 bytes only, and those are in 2 of the 16 channels of
  // its L2: a decode batch of 64 sequences took 149 us in place of 137.)
  const int place = blockIdx.x / kXcds, part = a.hk(place), kvh = place - part * a.hk.d;
  const int index = part * kXcds + blockIdx.x % kXcds;
  const Item it = find_item<false, FewTiles<RB>>(a, index);
  if (it.b < 0) {
    fill_rest(a, kvh, it.extra, a.hk(gridDim.x) - (index - it.extra));
    return;
  }
  if (it.key0 >= it.key1 && it.split > 0) return;
  few_rows<T, KIND, DP, FULL, RB>(a, it, kvh, smem, stats);
}

// A large tile's steps: BN keys, whose codes the workgroup turns into values once, in registers, and writes to the images that the
// 16-bit kernel's tiles have (two of keys and two of values in turn).
template <int DP>
struct Large {
  static constexpr int BN = DP <= 128 ? 64 : 32;
  static constexpr int kImages = 4 * BN * DP / 8;
};

// 128 rows, 32 a wave; the keys in steps of BN that all waves share; a step's loads are sent a step before it is turned. Bound by a
// wave's own chain of products, exponentials and turned codes (of a launch's cycles vector units are busy in 46 %, the matrix units and
// LDS in 33 % each, two waves to a SIMD): chunks of 512, 512, 511 and 1 token behind contexts of up to 8192, 32 heads over 8 of 128
// columns, 106 GFLOP in 156 us (0.68 PFLOP/s), 19 of them the merge of 68 MB of parts; in 16 bits 162 us. (Of 64 rows a wave, one
// workgroup a CU, the next step's scores between the exponentials: heads of 64 columns 194 us in place of 101; steps of 32 keys for
// three workgroups a CU: 259 us in place of 162, what the registers do not hold is put aside.)
template <class T, int KIND, int DP, bool FULL>
__device__ __forceinline__ void large_tile8(const Args8& a, const Item& it, int kvh, u32x4* smem) {
  constexpr bool F = std::is_same<T, F16>::value;
  using C = typename std::conditional<F && KIND == cache8::kInt8, cache8::TwoFactors, cache8::Codes<KIND, !F>>::type;
  using E = cache8::Ends<KIND>;
  constexpr int BN = Large<DP>::BN, NB = BN / 32, CH = DP / 16, IMG = BN * DP / 8;
  constexpr int N = (BN * CH + kThreads - 1) / kThreads;  // 16-code pieces of a thread
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int top = it.row0 + it.rows - 1;
  const int row = it.row0 + 32 * wave + (lane & 31);
  const int mine = min(row, top);
  const bool active = it.row0 + 32 * wave <= top;
  u32x4 q[DP / 16];
  load_q<T, DP, FULL>(a, it, kvh, mine, q, lane);
  const int limit = min(it.first + a.group(mine), it.keys - 1);
  const int least = __builtin_amdgcn_readfirstlane(limit), most = __builtin_amdgcn_readlane(limit, 31);
  Running<DP> r;
  r.clear();
  Cache cache(a, it, kvh);
  u32x4 kc[N], vc[N];
  int ks[N], vs[N], next[N];
  const auto mine_of = [&](int n) { return BN * CH % kThreads == 0 || tid + n * kThreads < BN * CH; };
  // FULL: a wave's piece is rows of one 16-key block, its first at `first_row`.
  constexpr int RPI = kWave / CH;
  const auto first_row = [&](int n) { return RPI * (wave + kWaves * n); };
  const uint32_t k_t = static_cast<uint32_t>(a.k_t);
  const auto look = [&](int key) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if constexpr (FULL) next[n] = cache.id(a, key + (first_row(n) & ~15));
      else if (mine_of(n)) next[n] = cache.id(a, key + (tid + n * kThreads) / CH);
    }
  };
  const auto load = [&](int key) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if constexpr (FULL) {
        const Sixteen x(a, cache, key + (first_row(n) & ~15), next[n]);
        const int r = min((first_row(n) & 15) + lane / CH, x.rest);
        const uint32_t off = r * k_t + 16 * (lane % CH), part = static_cast<uint32_t>(a.block(r)) * static_cast<uint32_t>(a.ks_b);
        ks[n] = x.ks[part];
        vs[n] = x.vs[part];
        kc[n] = *reinterpret_cast<const u32x4*>(x.k + off);
        vc[n] = *reinterpret_cast<const u32x4*>(x.v + off);
      } else {
        if (!mine_of(n)) continue;
        const int i = tid + n * kThreads;
        int64_t ko, vo, kso, vso;
        cache.at(a, key + i / CH, next[n], ko, vo, kso, vso);
        ks[n] = cache.ks[kso];
        vs[n] = cache.vs[vso];
        kc[n] = codes16<false>(a, cache.k + ko, i % CH);
        vc[n] = codes16<false>(a, cache.v + vo, i % CH);
      }
    }
  };
  // e4m3 to fp16: codes at scales past 2^22 become others. A branch, behind the barrier where the step has one anyway (chunks of 128
  // columns 164 us to 166, of 64 101 to 103; inside turn() 170 and 109, and by a second factor 169 and 104).
  const auto settle = [&] {
    if constexpr (F && KIND == cache8::kE4m3) {
      uint32_t beyond = 0;
#pragma unroll
      for (int n = 0; n < N; ++n)
        if (mine_of(n)) beyond |= E::beyond(ks[n]) | E::beyond(vs[n]);
      if (!__any(beyond)) return;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (!mine_of(n)) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) kc[n][e] = E::codes(kc[n][e], ks[n]), vc[n][e] = E::codes(vc[n][e], vs[n]);
        ks[n] = E::byte(ks[n]), vs[n] = E::byte(vs[n]);
      }
    }
  };
  const auto turn = [&](int to) {
    u32x4* kimg = smem + to * IMG;
    u32x4* vimg = smem + (2 + to) * IMG;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (!mine_of(n)) continue;
      const int i = tid + n * kThreads, rw = i / CH, c = i % CH;
      const typename C::Scale sk = C::scale(ks[n]), sv = C::scale(vs[n]);
      kimg[k_place<DP>(rw, 2 * c)] = cache8::eight<C>(kc[n][0], kc[n][1], sk);
      kimg[k_place<DP>(rw, 2 * c + 1)] = cache8::eight<C>(kc[n][2], kc[n][3], sk);
      vimg[v_place<DP>(rw, 2 * c)] = cache8::eight<C>(vc[n][0], vc[n][1], sv);
      vimg[v_place<DP>(rw, 2 * c + 1)] = cache8::eight<C>(vc[n][2], vc[n][3], sv);
    }
  };
  int buf = 0;
  if (it.key0 < it.key1) {
    look(it.key0);
    load(it.key0);
    look(it.key0 + BN);
    settle();
    turn(0);
    if (it.key0 + BN < it.key1) load(it.key0 + BN);
    look(it.key0 + 2 * BN);
  }
  // Behind the barrier this step's image is written, and the next step's, whose loads were sent a step ago, may be. It is turned
  // behind the scores, whose matrix instructions the turning does not wait for, in every step: behind the last key it turns what
  // was turned before, which none reads. (Turned ahead of the scores, and only where a next step was, which is a branch: prompt
  // chunks of 128 columns 166 us in place of 162, of 64 columns 110 in place of 101.)
  const auto send = [&](int key) {
    if (key + 2 * BN < it.key1) {
      load(key + 2 * BN);
      look(key + 3 * BN);
    }
  };
  int key = it.key0;
  const int mine_end = active ? min(it.key1, most + 1) : it.key0;
  for (; key < mine_end; key += BN) {
    __syncthreads();
    settle();
    f32x16 s[NB];
    u32x4 p[NB][2];
#pragma unroll
    for (int b = 0; b < NB; ++b) s[b] = scores<T, DP>(smem + buf * IMG, 32 * b, q, lane);
    turn(buf ^ 1);
    send(key);
    softmax_step<T, DP, NB>(s, p, r, a.scale_log2, key, min(limit, cache.last), key + BN - 1 > min(least, cache.last), lane);
#pragma unroll
    for (int b = 0; b < NB; ++b) weighted<T, DP>(smem + (2 + buf) * IMG, 32 * b, p[b], r.o, lane);
    buf ^= 1;
  }
  for (; key < it.key1; key += BN) {
    __syncthreads();
    settle();
    turn(buf ^ 1);
    send(key);
    buf ^= 1;
  }
  if (__syncthreads_or(cache.bad)) r.l = NAN;
  if (active) write_rows<T, DP>(a, it, kvh, row, r, lane);
}

// The item of a workgroup of large tiles, found by one wave for all four and read back as scalars. (With every wave finding it:
// prompt chunks of 128 columns 161 us in place of 156, of 256 columns 280 in place of 252. The launches of few rows and the merge, which
// find theirs in every wave, lose 0.4 to 0.8 us this way, to the barrier.)
__device__ __forceinline__ Item found_once(const Args& a, int index, int (&words)[14]) {
  if (threadIdx.x < kWave) {
    const Item x = find_item<false, Tiles32>(a, index);
    const int all[14] = {x.b,    x.begin, x.row0,   x.rows, x.keys,  x.first, x.key0,
                         x.key1, x.split, x.splits, x.slot, x.extra, x.small, x.divided};
    if (threadIdx.x == 0) {
#pragma unroll
      for (int i = 0; i < 14; ++i) words[i] = all[i];
    }
  }
  __syncthreads();
  int w[14];
#pragma unroll
  for (int i = 0; i < 14; ++i) w[i] = __builtin_amdgcn_readfirstlane(words[i]);
  return Item{w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7], w[8], w[9], w[10], w[11], w[12] != 0, w[13] != 0};
}

// Heads of up to 96 columns: the large tiles are made for 96, the few rows' for 128.
template <class T, int KIND, int DP, bool FULL>
__global__ __launch_bounds__(kThreads, DP > 128 ? 1 : 2) void attention8_kernel(Args8 a) {
  using F = Few<DP == 96 ? 128 : DP, 2>;
  __shared__ __align__(16) u32x4 smem[F::kChunks > Large<DP>::kImages ? F::kChunks : Large<DP>::kImages];
  __shared__ float stats[F::kStats];
  if constexpr (std::is_same<T, F16>::value) cache8::saturate_f16();
  const int index = a.hk(blockIdx.x), kvh = blockIdx.x - index * a.hk.d;
  __shared__ int words[14];
  const Item it = found_once(a, index, words);
  if (it.b < 0) {
    fill_rest(a, kvh, it.extra, a.hk(gridDim.x) - (index - it.extra));
    return;
  }
  if (it.key0 >= it.key1 && it.split > 0) return;
  if (it.small) few_rows<T, KIND, DP == 96 ? 128 : DP, FULL, 2>(a, it, kvh, smem, stats);
  else large_tile8<T, KIND, DP, FULL>(a, it, kvh, smem);
}

// What a launch is made for: tiles of 16 rb rows, or (rb 0) the large ones beside small ones of 32.
template <class T, int KIND, int RB>
int launch8_few(const Args8& a, const Launch& n, hipStream_t st) {
  const unsigned grid = static_cast<unsigned>((n.index + kXcds - 1) / kXcds * kXcds * a.hk.d);
  const bool full = a.wide && a.even;
  if (a.d == 64 && full) attention8_few_kernel<T, KIND, 64, true, RB><<<grid, kThreads, 0, st>>>(a);
  else if (a.d <= 64) attention8_few_kernel<T, KIND, 64, false, RB><<<grid, kThreads, 0, st>>>(a);
  else if (a.d == 128 && full) attention8_few_kernel<T, KIND, 128, true, RB><<<grid, kThreads, 0, st>>>(a);
  else if (a.d <= 128) attention8_few_kernel<T, KIND, 128, false, RB><<<grid, kThreads, 0, st>>>(a);
  else if constexpr (RB < 3) {
    if (a.d == 256 && full) attention8_few_kernel<T, KIND, 256, true, RB><<<grid, kThreads, 0, st>>>(a);
    else attention8_few_kernel<T, KIND, 256, false, RB><<<grid, kThreads, 0, st>>>(a);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return static_cast<int>(e);
  return n.merges > 0 ? launch_merge<FewTiles<RB>>(std::is_same<T, Bf16>::value ? BP_DT_BF16 : BP_DT_F16, a, n, st) : BP_OK;
}

template <class T, int KIND>
int launch8_large(const Args8& a, const Launch& n, hipStream_t st) {
  const unsigned grid = static_cast<unsigned>(n.index * a.hk.d);
  const bool full = a.wide && a.even;
  if (a.d == 64 && full) attention8_kernel<T, KIND, 64, true><<<grid, kThreads, 0, st>>>(a);
  else if (a.d <= 64) attention8_kernel<T, KIND, 64, false><<<grid, kThreads, 0, st>>>(a);
  else if (a.d <= 96) attention8_kernel<T, KIND, 96, false><<<grid, kThreads, 0, st>>>(a);
  else if (a.d == 128 && full) attention8_kernel<T, KIND, 128, true><<<grid, kThreads, 0, st>>>(a);
  else if (a.d <= 128) attention8_kernel<T, KIND, 128, false><<<grid, kThreads, 0, st>>>(a);
  else if (a.d == 256 && full) attention8_kernel<T, KIND, 256, true><<<grid, kThreads, 0, st>>>(a);
  else attention8_kernel<T, KIND, 256, false><<<grid, kThreads, 0, st>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return static_cast<int>(e);
  return n.merges > 0 ? launch_merge<Tiles32>(std::is_same<T, Bf16>::value ? BP_DT_BF16 : BP_DT_F16, a, n, st) : BP_OK;
}

template <class T, int KIND>
int launch8(const Args8& a, const Launch& n, int rb, hipStream_t st) {
  switch (rb) {
    case 1: return launch8_few<T, KIND, 1>(a, n, st);
    case 2: return launch8_few<T, KIND, 2>(a, n, st);
    case 3: return launch8_few<T, KIND, 3>(a, n, st);
    default: return launch8_large<T, KIND>(a, n, st);
  }
}

// Few rows a sequence, as far as the host can tell (the offsets are the device's; any are right): 16-row blocks of a tile, 0: none.
// The least that hold a sequence's rows: a tile pays for its empty ones. Decode steps (one to four rows a sequence) in tiles of 16,
// 32, 48 rows and as small sequences of a launch that may have large ones, us: 64 sequences, 4 rows, 119, 120, 124, 122; three long
// contexts of 64 columns 65, 69, 79, 92; six contexts of 256 columns 34, 47, -, 40. A verify round of six sequences, 36 rows: 32.9 in
// tiles of 48, 35.4 as small sequences.
// The mean is all that the host has: beside many steps a part of a prompt, or beside many empty places a few parts, come in tiles of 16 rb
// rows too, each of which turns its sequence's codes again. 64 ragged steps and one part behind 8192 positions, by this rule and as a
// launch that may have large tiles, us: heads of 128 columns, 32 over 8, a part of 32 tokens 139 and 179, of 192 206 and 190, of 512 268
// and 241; 8 over 8, 512 tokens, 206 and 183; 16 over 1, 128 tokens, 70 and 56; heads of 64 columns, 16 over 4, 512 tokens, 89 and 109;
// of 256, 8 over 1, 128 tokens, 86 and 120. Four steps and a part of 192 tokens, 16 heads of 64, 64 and 44. Of 232 such launches (4 to 64
// steps, parts of 8 to 2048 tokens) 18 are slower by this rule by more than 5 %, that last one the most, and the others take 1.23 times
// as long in the mean without it, up to 2.7 times.
int few_of(int64_t tokens, int64_t seqs, int64_t group, int d) {
  const int most = d > 128 ? 2 : 3;
  for (int rb = 1; rb <= most; ++rb)
    if (group <= 16 * rb && tokens * group <= 16 * rb * seqs) return rb;
  return 0;
}

bool plan8(Args8& a, Launch& n, int rb) {
  switch (rb) {
    case 1: return plan_launch<FewTiles<1>>(a, n);
    case 2: return plan_launch<FewTiles<2>>(a, n);
    case 3: return plan_launch<FewTiles<3>>(a, n);
    default: return plan_launch<Tiles32>(a, n);
  }
}

bool aligned(const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int run8(int dtype, int kind, Args8& a, size_t ws_bytes, hipStream_t st) {
  const int hk = a.hk.d;
  if ((dtype != BP_DT_BF16 && dtype != BP_DT_F16) || (kind != BP_DT_E4M3 && kind != BP_DT_I8)) return BP_E_UNSUPPORTED;
  if (a.tokens < 0 || a.seqs < 0 || hk <= 0 || a.hq <= 0 || a.hq % hk != 0 || !(a.scale_log2 > 0.f && a.scale_log2 <= FLT_MAX))
    return BP_E_INVALID_ARG;
  if (a.d <= 0 || a.d % 8 != 0 || a.d > 256) return BP_E_UNSUPPORTED;
  if (a.tokens == 0) return BP_OK;
  if (a.q == nullptr || a.out == nullptr || (a.seqs > 0 && a.cu == nullptr)) return BP_E_INVALID_ARG;
  // a stride that nothing is multiplied with may be anything
  const int blocks = a.page.d / a.block.d;
  if (a.tokens == 1) a.q_t = 0;
  if (a.hq == 1) a.q_h = 0;
  if (hk == 1) a.k_h = a.v_h = a.ks_h = a.vs_h = 0;
  if (a.page.d == 1) a.k_t = a.v_t = 0;
  if (blocks == 1) a.ks_b = a.vs_b = 0;
  if (a.pool == 1) a.k_p = a.v_p = a.ks_p = a.vs_p = 0;
  const int64_t strides = a.k_p | a.k_t | a.k_h | a.v_p | a.v_t | a.v_h;
  if (!aligned(a.q, 16) || !aligned(a.out, 16) || ((a.q_t | a.q_h) & 7) != 0 || !aligned(a.k, 8) || !aligned(a.v, 8) ||
      (strides & 7) != 0)
    return BP_E_INVALID_ARG;
  a.wide = aligned(a.k, 16) && aligned(a.v, 16) && (strides & 15) == 0 && a.d % 16 == 0;
  // (and a page's strides, and offsets inside a page, in 32 bits)
  a.even = a.page.d % 16 == 0 && (a.block.d % 16 == 0 || 16 % a.block.d == 0) && a.k_p == a.v_p && a.k_t == a.v_t &&
           a.ks_p == a.vs_p && a.ks_b == a.vs_b && ((a.k_p | a.ks_p) & ~0x7fffffffll) == 0 && a.k_t >= 0 && a.ks_b >= 0 &&
           a.k_t * a.page.d < (1ll << 31) && a.ks_b * blocks < (1ll << 31);
  // rows of a sequence, and keys plus a split, in 32 bits
  if (static_cast<int64_t>(a.tokens) * a.hq >= (1ll << 30) || a.max_keys >= (1 << 29)) return BP_E_UNSUPPORTED;
  const int rb = few_of(a.tokens, a.seqs, a.hq / hk, a.d);
  Launch n;
  if (!plan8(a, n, rb)) return BP_E_UNSUPPORTED;
  if (n.workspace > 0 && (a.ws == nullptr || ws_bytes < n.workspace || !aligned(a.ws, 16))) return BP_E_WORKSPACE;
  if (n.workspace == 0) a.ws = nullptr;
  // A row of q is read by the tile that writes its result and by no other, so out may be q itself.
  const auto reach = [](int size, int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t n2, int64_t s2, int64_t last) {
    return n0 > 0 ? size * ((n0 - 1) * s0 + (n1 - 1) * s1 + (n2 - 1) * s2 + last) : 0;
  };
  const int64_t dense = static_cast<int64_t>(a.hq) * a.d, out = 2 * dense * a.tokens;
  const bool in_place = a.out == a.q && (a.tokens == 1 || a.q_t == dense) && (a.hq == 1 || a.q_h == a.d);
  if ((!in_place && ranges_overlap(a.out, out, a.q, reach(2, a.tokens, a.q_t, a.hq, a.q_h, 1, 0, a.d))) ||
      ranges_overlap(a.out, out, a.k, reach(1, a.pool, a.k_p, a.page.d, a.k_t, hk, a.k_h, a.d)) ||
      ranges_overlap(a.out, out, a.v, reach(1, a.pool, a.v_p, a.page.d, a.v_t, hk, a.v_h, a.d)) ||
      ranges_overlap(a.out, out, a.ks, reach(1, a.pool, a.ks_p, blocks, a.ks_b, hk, a.ks_h, 1)) ||
      ranges_overlap(a.out, out, a.vs, reach(1, a.pool, a.vs_p, blocks, a.vs_b, hk, a.vs_h, 1)))
    return BP_E_INVALID_ARG;
  const bool e4m3 = kind == BP_DT_E4M3;
  if (dtype == BP_DT_BF16)
    return e4m3 ? launch8<Bf16, cache8::kE4m3>(a, n, rb, st) : launch8<Bf16, cache8::kInt8>(a, n, rb, st);
  return e4m3 ? launch8<F16, cache8::kE4m3>(a, n, rb, st) : launch8<F16, cache8::kInt8>(a, n, rb, st);
}

}  // namespace
}  // namespace attn
}  // namespace bp

extern "C" size_t bp_attn_paged8_workspace_bytes(int64_t tokens, int64_t seqs, int64_t hq, int64_t hk, int64_t head_dim,
                                                 int64_t max_keys) {
  using namespace bp::attn;
  if (hk <= 0 || hq % hk != 0) return 0;
  switch (few_of(tokens, seqs, hq / hk, static_cast<int>(head_dim))) {
    case 1: return workspace_bytes<FewTiles<1>>(tokens, seqs, hq, hk, head_dim, max_keys);
    case 2: return workspace_bytes<FewTiles<2>>(tokens, seqs, hq, hk, head_dim, max_keys);
    case 3: return workspace_bytes<FewTiles<3>>(tokens, seqs, hq, hk, head_dim, max_keys);
    default: return workspace_bytes<Tiles32>(tokens, seqs, hq, hk, head_dim, max_keys);
  }
}

extern "C" int bp_attn_paged8(const BpPagedCache* cache, int dtype, const void* q, void* out, const int32_t* cu, int tokens, int hq,
                              int64_t q_t, int64_t q_h, float scale, void* workspace, size_t workspace_bytes, void* stream) {
  if (cache == nullptr) return BP_E_INVALID_ARG;
  const BpPagedCache& c = *cache;
  if (c.page <= 0 || c.pool < 0 || c.seqs < 0 || c.max_pages < 0 || static_cast<int64_t>(c.page) * c.max_pages >= (1ll << 29))
    return BP_E_INVALID_ARG;
  if (c.block <= 0 || c.block % 4 != 0 || c.page % c.block != 0) return BP_E_INVALID_ARG;
  if (tokens > 0 && c.seqs > 0 &&
      (c.lengths == nullptr || (c.max_pages > 0 && (c.table == nullptr || c.k_pages == nullptr || c.v_pages == nullptr ||
                                                    c.k_scales == nullptr || c.v_scales == nullptr || c.pool == 0))))
    return BP_E_INVALID_ARG;
  bp::attn::Args8 a = {};
  a.q = q, a.k = c.k_pages, a.v = c.v_pages, a.out = out, a.cu = cu, a.lengths = c.lengths, a.table = c.table;
  a.ks = static_cast<const uint8_t*>(c.k_scales), a.vs = static_cast<const uint8_t*>(c.v_scales);
  a.ws = static_cast<float*>(workspace);
  a.q_t = q_t, a.q_h = q_h, a.k_p = c.kp[0], a.k_t = c.kp[1], a.k_h = c.kp[2], a.v_p = c.vp[0], a.v_t = c.vp[1], a.v_h = c.vp[2];
  a.ks_p = c.ks[0], a.ks_b = c.ks[1], a.ks_h = c.ks[2], a.vs_p = c.vs[0], a.vs_b = c.vs[1], a.vs_h = c.vs[2];
  a.table_stride = c.table_stride;
  a.tokens = tokens, a.seqs = c.seqs, a.hq = hq, a.hk.d = c.hk, a.d = c.head_dim, a.causal = 1;
  a.pool = c.pool, a.page = bp::attn::Div::of(c.page), a.block = bp::attn::Div::of(c.block);
  a.max_keys = c.page * c.max_pages;
  a.scale_log2 = scale * 1.44269504088896340736f;
  return bp::attn::run8(dtype, c.dtype, a, workspace_bytes, static_cast<hipStream_t>(stream));
}
