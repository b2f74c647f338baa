// Attention of several sequences at once: the plan of a launch, which every workgroup makes for itself from the device's
// offsets and lengths, and the pieces of the kernels that do not depend on where a key lies.
//
//   out[i, h] = sum_j p_ij v[j, h / group],  p_i = softmax_j(scale q[i, h] . k[j, h / group]),  j <= limit(i)
//
// The rows of a product are (token, query head of the group) pairs of one key head, token-major: row r of a sequence is
// token r / group, head r % group of the group, so the heads that share keys share the loads of them. The scores are
// computed transposed, S^T = K Q^T (32 keys x 32 rows a matrix instruction): a lane then holds scores of one row only, its
// maximum, sum and rescaling are scalars of the lane, and the probabilities, rounded to the tensors' type, are the second
// product's operand where they lie (O^T = V^T P^T; its key order is the order in which the first product leaves them).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"

namespace bp {
namespace attn {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kSmallRows = 64;   // sequences of at most this many rows: 32-row tiles whose waves share the keys
constexpr int kTileSmall = 32;
constexpr int kTileLarge = 128;  // 32 rows a wave, all keys
constexpr int kSharedMin = 512;  // least keys of a split where the parts are more than that
constexpr int kKeyStep = 128;    // a split's keys are a multiple of this: whole steps of either kind of tile

// n / d for n below 2^30 without a division: magic = floor(2^(32 + shift) / d) + 1 with 2^shift < d <= 2^(shift + 1).
struct Div {
  uint32_t magic;
  int d, shift;
  __host__ static Div of(int d) {
    Div r = {0, d, 0};
    while ((2ll << r.shift) < d) ++r.shift;
    if (d > 1) r.magic = static_cast<uint32_t>((1ull << (32 + r.shift)) / d + 1);
    return r;
  }
  __device__ __forceinline__ int operator()(int n) const {
    return d == 1 ? n : static_cast<int>(__umulhi(static_cast<uint32_t>(n), magic) >> shift);
  }
};

struct Args {
  const void* q;
  const void* k;
  const void* v;
  void* out;           // [tokens, hq, d], contiguous
  const int* cu;       // [seqs + 1]
  const int* lengths;  // [seqs], or null: as many keys as tokens (packed)
  const int* table;    // [seqs, max_pages], or null
  float* ws;           // partials of divided tiles, or null: nothing is divided
  int64_t q_t, q_h;            // element strides
  int64_t k_p, k_t, k_h;       // page (paged), position, head
  int64_t v_p, v_t, v_h;
  int64_t table_stride;
  Div hk, group, page, tile_tokens;
  int tokens, seqs, pool, max_keys, hq, d, causal;
  int order;      // the longest tiles first, over all sequences (up to 64 of them)
  int resident;   // workgroups that the card holds at once
  int target;     // parts that splitting aims at where they are more
  int chunk_min;  // least keys of a split
  int ws_rows;    // rows of a partial's slot
  int slots;      // slots of a key head that ws holds
  float scale_log2;
};

// What a sequence asks for.
struct Seq {
  int begin, count, rows, keys, tiles;
};

__device__ __forceinline__ Seq sequence(const Args& a, int b) {
  Seq s;
  s.begin = min(max(a.cu[b], 0), a.tokens);
  const int end = min(max(a.cu[b + 1], s.begin), a.tokens);
  s.count = end - s.begin;
  s.rows = s.count * a.group.d;
  s.keys = a.lengths ? min(max(a.lengths[b], 0), a.max_keys) : s.count;
  s.tiles = s.rows <= kSmallRows ? (s.rows + kTileSmall - 1) / kTileSmall : (s.rows + kTileLarge - 1) / kTileLarge;
  return s;
}

__device__ __forceinline__ int wave_sum(int v) {
  const auto add = [](float x, float y) { return __int_as_float(__float_as_int(x) + __float_as_int(y)); };
  return __builtin_amdgcn_readfirstlane(__float_as_int(xor_butterfly<true>(__int_as_float(v), add)));
}

// Inclusive sum over the lanes: shifts within rows of 16, then the rows' last lanes into the rows behind them.
__device__ __forceinline__ int scan_add(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr:1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
  return v;
}

// Keys of a split: the whole work in keys x tiles over the workgroups that the card holds at once, where the parts are no more
// than those; else over `target`, so that ragged parts share the card evenly; never under chunk_min. (A verify round of 36 rows
// over 41k keys: 39 us in 480 parts, 53 in 660; a decode batch of 64 ragged sequences: 219 us by the first rule, 204 to 210 by
// the second.) Every workgroup adds the same numbers in the same order, so all of them find the same value.
__device__ __forceinline__ int split_keys(const Args& a, const Seq& own, int lane) {
  float units = 0.f;
  for (int b = lane; b < a.seqs; b += kWave) {
    const Seq s = b < kWave ? own : sequence(a, b);
    units += static_cast<float>(s.tiles) * static_cast<float>(s.keys);
  }
  units = xor_butterfly<true>(units, AddOp()) * static_cast<float>(a.hk.d) * 1.001f;
  const auto chunk_of = [&](int target) {
    const float want = units / static_cast<float>(target);
    const int chunk = want < 1e9f ? static_cast<int>(want) + 1 : 0x3fffff00;
    return __builtin_amdgcn_readfirstlane((max(chunk, a.chunk_min) + kKeyStep - 1) / kKeyStep * kKeyStep);
  };
  const int chunk = chunk_of(a.resident);
  int items = 0;
  for (int b = lane; b < a.seqs; b += kWave) {
    const Seq s = b < kWave ? own : sequence(a, b);
    items += s.tiles * max(1, static_cast<int>(static_cast<unsigned>(s.keys + chunk / 2) / static_cast<unsigned>(chunk)));
  }
  return wave_sum(items) <= a.resident / a.hk.d ? chunk : max(chunk_of(a.target), kSharedMin);
}

// One workgroup's part: `rows` rows from row0 of sequence b, key range [key0, key1) of split `split` of `splits`. divided: the
// tile's parts go to slots from `slot` on (a tile of fewer keys than its sequence leaves the last of them unwritten; its first
// it always writes). b < 0: beyond the last tile, `extra` tiles past it.
struct Item {
  int b, begin, row0, rows, keys, first, key0, key1, split, splits, slot, extra;
  bool small, divided;
};

constexpr int kMergeRows = 32;  // rows of a unit of the merge; of up to 64 rows with more than kMergeParts parts, one
constexpr int kMergeParts = 8;
constexpr int kLevel = 128;  // keys of a level, of which the order of the tiles is made
constexpr int kUndivided = 0x3fffffff;

// The tile of index `index` (per key head); or, of the sequences whose keys are divided, the unit of rows of index `index` with
// what its tile's parts are.
template <bool MERGE>
__device__ __forceinline__ Item find_item(const Args& a, int index) {
  const int lane = static_cast<int>(threadIdx.x) & 63;
  Seq own = {0, 0, 0, 0, 0};  // the lane's of the first 64 sequences: read once
  if (lane < a.seqs) own = sequence(a, lane);
  const bool divide = a.ws != nullptr;
  const int chunk = divide ? split_keys(a, own, lane) : 0;
  Item it;
  it.b = -1;
  int items = 0, slots = 0;
  for (int b0 = 0; b0 < a.seqs; b0 += kWave) {
    const int b = b0 + lane;
    Seq s = own;
    if (b0 > 0) s = b < a.seqs ? sequence(a, b) : Seq{0, 0, 0, 0, 0};
    int splits = 1, part = kUndivided, parts = 0, slot_upto = 0;
    if (divide) {
      splits = max(1u, static_cast<unsigned>(s.keys + chunk / 2) / static_cast<unsigned>(chunk));
      if (splits > 1) {
        // the sequence's own splits: all alike, of whole steps
        part = (static_cast<unsigned>(s.keys + splits - 1) / static_cast<unsigned>(splits) + kKeyStep - 1) / kKeyStep * kKeyStep;
        parts = s.tiles * splits;
      }
      slot_upto = scan_add(parts);
    }
    const int all = s.tiles * splits;
    int l, at, above = 0;  // the sequence's lane, the place among its items, the tiles of it that come earlier
    if (!MERGE && a.order) {
      // Tiles by level, the number of keys in steps, from the greatest down; within a level by sequence. later(x): how many
      // tiles of the lane's sequence have level x or more. A causal tile's level grows with its place, others' are alike.
      const bool ladder = a.causal && s.rows > kSmallRows && splits == 1;
      const int flat = min(s.keys, part) / kLevel, first = max(s.keys - s.count, 0), step = a.tile_tokens.d;
      const auto later = [&](int x) {
        if (!ladder) return flat >= x ? s.tiles : 0;
        const int need = x * kLevel - first;
        return s.tiles - min(s.tiles, need <= 0 ? 0 : max(a.tile_tokens(need + step - 1) - 1, 0));
      };
      if (wave_sum(all) <= index) {
        items = wave_sum(all);
        break;
      }
      int lo = 0, hi = max(a.max_keys, a.tokens) / kLevel + 2;  // more than index tiles have level lo or more; not more hi
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (wave_sum(later(mid) * splits) > index) lo = mid;
        else hi = mid;
      }
      const int before = later(hi), count = (later(lo) - before) * splits;
      const int upto = scan_add(count), from = index - wave_sum(before * splits);
      l = __builtin_ctzll(__ballot(upto > from));
      at = from - __builtin_amdgcn_readlane(upto - count, l);
      above = __builtin_amdgcn_readlane(before, l);
    } else {
      const bool single = splits > kMergeParts && s.rows <= kSmallRows;
      const int count = !MERGE ? all : splits == 1 ? 0 : single ? s.rows : (s.rows + kMergeRows - 1) / kMergeRows;
      const int upto = scan_add(count);
      const uint64_t over = __ballot(items + upto > index);
      if (over == 0) {
        items += __builtin_amdgcn_readlane(upto, 63);
        slots += __builtin_amdgcn_readlane(slot_upto, 63);
        continue;
      }
      l = __builtin_ctzll(over);
      at = index - items - __builtin_amdgcn_readlane(upto - count, l);
    }
    const int tiles = __builtin_amdgcn_readlane(s.tiles, l), count = __builtin_amdgcn_readlane(s.count, l);
    const int rows = __builtin_amdgcn_readlane(s.rows, l), keys = __builtin_amdgcn_readlane(part, l);
    it.b = b0 + l;
    it.begin = __builtin_amdgcn_readlane(s.begin, l);
    it.keys = __builtin_amdgcn_readlane(s.keys, l);
    it.splits = __builtin_amdgcn_readlane(splits, l);
    it.divided = it.splits > 1;
    it.small = rows <= kSmallRows;
    const int tile_rows = it.small ? kTileSmall : kTileLarge;
    // the last rows first: under a causal mask they have the most keys
    const int done = it.divided && !MERGE ? static_cast<unsigned>(at) / static_cast<unsigned>(it.splits) : at;
    const int unit = MERGE && (it.splits <= kMergeParts || !it.small) ? kMergeRows : 1;
    const int tile = MERGE ? at * unit / tile_rows : tiles - 1 - above - done;
    it.split = it.divided ? at - done * it.splits : 0;
    it.slot = slots + __builtin_amdgcn_readlane(slot_upto - parts, l) + tile * it.splits;
    it.row0 = tile * tile_rows;
    it.rows = min(tile_rows, rows - it.row0);
    it.first = it.keys - count;  // the key position of token 0
    const int end = a.causal ? min(it.keys, max(0, it.first + a.group(it.row0 + it.rows - 1) + 1)) : it.keys;
    it.key0 = min(end, it.split * keys);
    it.key1 = min(end, it.key0 + keys);
    if (MERGE) {
      it.split = at * unit % tile_rows;  // the first of the rows, in its tile
      it.rows = min(unit, it.rows - it.split);
      it.splits = max(1u, static_cast<unsigned>(end + keys - 1) / static_cast<unsigned>(keys));  // those that had keys
    }
    return it;
  }
  it.extra = index - items;
  return it;
}

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
};
struct F16 {
  static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, (h2){static_cast<_Float16>(x), static_cast<_Float16>(y)});
  }
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

// The running softmax of one row (both halves of a wave hold the row's maximum; each its own part of the sum).
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
  mx = max_halves(mx) * c;
  const float m = fmaxf(r.m, mx);
  if (__any(m > r.m)) {
    // exp2(-inf - m) = 0 clears a row's empty start; a row that has seen nothing keeps m = -inf and scales by 1
    const float f = m == r.m ? 1.f : __builtin_amdgcn_exp2f(r.m - m);
    r.m = m;
    r.l *= f;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) r.o[d][i] *= f;
  }
  const float shift = r.m == -INFINITY ? 0.f : -r.m;
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
