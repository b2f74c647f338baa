// The plan of a launch of attention.hip: what the host gives it, and how every workgroup finds its tile from the device's
// offsets and lengths. Needs common.h, or what it takes of it (kWave, xor_butterfly, AddOp), before it.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "byteprof_amd.h"

namespace bp {
namespace attn {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kSmallRows = 64;   // sequences of at most this many rows: 32-row tiles whose waves share the keys
constexpr int kTileSmall = 32;
constexpr int kTileLarge = 128;  // 32 rows a wave, all keys
constexpr int kSharedMin = 512;  // least keys of a split of few rows, and of others where the parts are more than the card holds
constexpr int kKeyStep = 128;    // a split's keys are a multiple of this: whole steps of either kind of tile

constexpr int kCus = 256;

// How a launch cuts sequences into tiles. Tiles32: the kernels of attention.hip, and over a cache in 8 bits wherever sequences have
// many rows. FewTiles: the kernel of attention8.hip for launches of few rows a sequence.
struct Tiles32 {
  static constexpr int kFew = kSmallRows;    // sequences of at most this many rows have the small tiles
  static constexpr int kSmall = kTileSmall;
  static constexpr bool kFit = true;         // parts that all fit the card at once, if that many do (split_keys)
  static constexpr int kMergeRows = 32;      // rows of a unit of the merge; of up to kFew rows with more than kMergeParts parts, one
  static constexpr int kTarget = 1024;       // bound of what splitting aims at (twice the workgroups that the card holds at once:
                                             // 1024, for 256 columns 512)
  static constexpr int kLeast = BP_ATTN_UNDIVIDED_KEYS;  // least keys of a split
  static constexpr int kWhole = BP_ATTN_UNDIVIDED_KEYS;  // where no sequence can have more keys, none is divided
  // By the registers of attention_kernel: 256 columns leave one wave a SIMD, 128 two (fewer columns three, but planning for three
  // made heads of 96 no faster and cached ones slower, 97 us against 90).
  static int workgroups_a_cu(int padded) { return padded > 128 ? 1 : 2; }
};
// All tiles of 16 RB rows. Parts by twice what the card holds at once, whether or not once would fit: a decode batch of 64 sequences
// took 129 us with once, 123 with one and a half times, 119 so; three long contexts 74, 65 and 65.
template <int RB>
struct FewTiles {
  static constexpr int kFew = 1 << 30;
  static constexpr int kSmall = 16 * RB;
  static constexpr bool kFit = false;
  static constexpr int kMergeRows = 16;
  static constexpr int kTarget = 2048;
  static constexpr int kLeast = kSharedMin;
  // find_item divides from one and a half least splits on. (With a launch of the merge that had no unit, from 257 on: a decode step over a
  // table of 300 or 600 positions 17 us, now 12.)
  static constexpr int kWhole = kLeast + kLeast / 2 - 1;
  // By the registers of attention8_few_kernel, a workgroup's four waves on the four SIMDs. (128 columns and 16 rows with room for
  // four: what the compiler puts aside in the loop is waited for with the loads, a decode batch 162 us in place of 119. 64 columns and 32
  // or 48 rows would have room for three: planned so, verify rounds of 6 and of 24 sequences take the same, 24.4, 27.4 and 25.4 us.)
  __host__ __device__ static constexpr int workgroups_a_cu(int padded) {
    return RB == 1 ? (padded > 128 ? 2 : padded > 64 ? 3 : 4) : padded > 128 ? 1 : 2;
  }
};

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
  Div hk, group, page;
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

template <class P>
__device__ __forceinline__ Seq sequence(const Args& a, int b) {
  Seq s;
  s.begin = min(max(a.cu[b], 0), a.tokens);
  const int end = min(max(a.cu[b + 1], s.begin), a.tokens);
  s.count = end - s.begin;
  s.rows = s.count * a.group.d;
  s.keys = a.lengths ? min(max(a.lengths[b], 0), a.max_keys) : s.count;
  s.tiles = s.rows <= P::kFew ? (s.rows + P::kSmall - 1) / P::kSmall : (s.rows + kTileLarge - 1) / kTileLarge;
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
// than those (P::kFit); else over `target`, so that ragged parts share the card evenly; never under chunk_min, by `target` with
// kFit not under kSharedMin. (A verify round of 36 rows over 41k keys: 39 us in 480 parts, 53 in 660; a decode batch of 64
// ragged sequences: 219 us by the first rule, 204 to 210 by the second.) Every workgroup adds the same numbers in the same
// order, so all of them find the same value.
template <class P>
__device__ __forceinline__ int split_keys(const Args& a, const Seq& own, int lane) {
  float units = 0.f;
  for (int b = lane; b < a.seqs; b += kWave) {
    const Seq s = b < kWave ? own : sequence<P>(a, b);
    units += static_cast<float>(s.tiles) * static_cast<float>(s.keys);
  }
  units = xor_butterfly<true>(units, AddOp()) * static_cast<float>(a.hk.d) * 1.001f;
  const auto chunk_of = [&](int target) {
    const float want = units / static_cast<float>(target);
    const int chunk = want < 1e9f ? static_cast<int>(want) + 1 : 0x3fffff00;
    return __builtin_amdgcn_readfirstlane((max(chunk, a.chunk_min) + kKeyStep - 1) / kKeyStep * kKeyStep);
  };
  if constexpr (!P::kFit) return chunk_of(a.target);
  const int chunk = chunk_of(a.resident);
  int items = 0;
  for (int b = lane; b < a.seqs; b += kWave) {
    const Seq s = b < kWave ? own : sequence<P>(a, b);
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

constexpr int kMergeParts = 8;
constexpr int kLevel = 128;  // keys of a level, of which the order of the tiles is made
constexpr int kUndivided = 0x3fffffff;

// The tile of index `index` (per key head); or, of the sequences whose keys are divided, the unit of rows of index `index` with
// what its tile's parts are.
template <bool MERGE, class P = Tiles32>
__device__ __forceinline__ Item find_item(const Args& a, int index) {
  const int lane = static_cast<int>(threadIdx.x) & 63;
  Seq own = {0, 0, 0, 0, 0};  // the lane's of the first 64 sequences: read once
  if (lane < a.seqs) own = sequence<P>(a, lane);
  const bool divide = a.ws != nullptr;
  const int chunk = divide ? split_keys<P>(a, own, lane) : 0;
  Item it;
  it.b = -1;
  int items = 0, slots = 0;
  for (int b0 = 0; b0 < a.seqs; b0 += kWave) {
    const int b = b0 + lane;
    Seq s = own;
    if (b0 > 0) s = b < a.seqs ? sequence<P>(a, b) : Seq{0, 0, 0, 0, 0};
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
      // tiles of the lane's sequence have level x or more. A causal tile's level grows with its place, others' are alike. No
      // tile has level hi: a causal one has it only if its sequence's last token is that far, whatever the rows of a token.
      const bool ladder = a.causal && s.rows > P::kFew && splits == 1;
      const int flat = min(s.keys, part) / kLevel, first = max(s.keys - s.count, 0);
      const auto later = [&](int x) {
        if (!ladder) return flat >= x ? s.tiles : 0;
        const int need = x * kLevel - first;  // tokens of the sequence up to the level's first
        if (need > s.count) return 0;
        if (need <= 0) return s.tiles;
        return s.tiles + 1 - static_cast<int>((static_cast<unsigned>(need * a.group.d) + kTileLarge - 1) / kTileLarge);
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
      const bool single = splits > kMergeParts && s.rows <= P::kFew;
      const int count = !MERGE ? all : splits == 1 ? 0 : single ? s.rows : (s.rows + P::kMergeRows - 1) / P::kMergeRows;
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
    it.small = rows <= P::kFew;
    const int tile_rows = it.small ? P::kSmall : kTileLarge;
    // the last rows first: under a causal mask they have the most keys
    const int done = it.divided && !MERGE ? static_cast<unsigned>(at) / static_cast<unsigned>(it.splits) : at;
    const int unit = MERGE && (it.splits <= kMergeParts || !it.small) ? P::kMergeRows : 1;
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

constexpr int kMergeGrid = 1024;  // workgroups of a merge launch; each takes every such unit

// Row tiles of a key head that any offsets can give: sequences of up to kFew rows (64, or all) have small tiles.
template <class P = Tiles32>
int64_t tiles_bound(int64_t tokens, int64_t seqs, int64_t group) {
  const int64_t rows = tokens * group, some = seqs < tokens ? seqs : tokens;
  const int64_t a = rows / kTileLarge + 2 * some, b = rows / P::kSmall + some;
  return P::kFew > kSmallRows || b <= a ? b : a;
}

template <class P = Tiles32>
bool may_split(int64_t max_keys) {
  return max_keys > P::kWhole;
}

inline int padded_dim(int d) { return d <= 64 ? 64 : d <= 96 ? 96 : d <= 128 ? 128 : 256; }

template <class P = Tiles32>
int slot_rows(int64_t tokens, int64_t group) {
  return tokens * group <= P::kFew ? P::kSmall : kTileLarge;
}

// Partials that any offsets can give. A split's keys are at least the whole work over the target, and a sequence is divided
// into as many parts as its keys come to, rounded to the nearest, from 1.5 on: at most a third more parts than the target. Nor
// are they more than every tile's most.
template <class P = Tiles32>
int64_t slots_bound(int64_t tokens, int64_t seqs, int64_t group, int64_t hk, int64_t max_keys) {
  const int64_t most = tiles_bound<P>(tokens, seqs, group) * hk * ((max_keys + P::kLeast - 1) / P::kLeast);
  const int64_t aim = P::kTarget + P::kTarget / 3 + 1 + hk;
  return most < aim ? most : aim;
}

template <class P = Tiles32>
size_t workspace_bytes(int64_t tokens, int64_t seqs, int64_t hq, int64_t hk, int64_t d, int64_t max_keys) {
  if (tokens <= 0 || seqs <= 0 || hk <= 0 || hq % hk != 0 || d <= 0 || d > 256 || !may_split<P>(max_keys)) return 0;
  const int64_t group = hq / hk;
  return static_cast<size_t>(slots_bound<P>(tokens, seqs, group, hk, max_keys)) * slot_rows<P>(tokens, group) *
         (padded_dim(static_cast<int>(d)) + 2) * sizeof(float);
}

// What a launch needs besides its arguments.
struct Launch {
  int64_t index;   // workgroups of a key head: every tile's, every part's, and one at least for the rows of no sequence
  int64_t merges;  // workgroups of a key head of the second launch, 0: nothing can be divided
  size_t workspace;
};

// Completes the arguments (hk.d, page and the sizes are set) and gives the launch's. False: more workgroups than a launch has.
template <class P = Tiles32>
bool plan_launch(Args& a, Launch& n) {
  const int hk = a.hk.d, group = a.hq / hk;
  a.hk = Div::of(hk);
  a.group = Div::of(group);
  a.resident = kCus * P::workgroups_a_cu(padded_dim(a.d));
  a.target = 2 * a.resident;
  a.chunk_min = P::kLeast;
  a.ws_rows = slot_rows<P>(a.tokens, group);
  const int64_t tiles = tiles_bound<P>(a.tokens, a.seqs, group);
  n.index = tiles;
  n.merges = 0;
  n.workspace = workspace_bytes<P>(a.tokens, a.seqs, a.hq, hk, a.d, a.max_keys);
  a.slots = 0;
  if (n.workspace > 0) {
    a.slots = static_cast<int>(slots_bound<P>(a.tokens, a.seqs, group, hk, a.max_keys) / hk);
    const int64_t most = tiles * ((a.max_keys + P::kLeast - 1) / P::kLeast - 1), aim = P::kTarget / hk + 1;
    n.index += most < aim ? most : aim;
    const int64_t units = static_cast<int64_t>(a.tokens) * group, wanted = kMergeGrid / hk + 1;
    n.merges = units < wanted ? units : wanted;
  }
  n.index += 1;  // rows of no sequence
  // one sequence's tiles come in this order by themselves, and with a workgroup's place for every tile none is needed
  a.order = a.seqs > 1 && a.seqs <= kWave && n.index * hk > a.resident;
  return n.index * hk < (1ll << 30);
}

}  // namespace attn
}  // namespace bp
