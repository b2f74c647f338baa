// Attention of packed prompts and of chunks over a paged cache, and the append to the cache's pages (attention.h: the
// mathematics; attention_plan.h: the plan).

#include "attention_rows.h"

#include <float.h>

#include <type_traits>

#include "byteprof_amd.h"

namespace bp {
namespace attn {
namespace {

template <int DP>
struct Shape {
  static constexpr int CH = DP / 8;
  static constexpr int NB = DP <= 128 ? 2 : 1;   // 32-key blocks of a step of a large tile
  static constexpr int BN = 32 * NB;
  static constexpr int kLarge = 4 * BN * CH;     // 16-byte chunks: two images of keys and two of values
  static constexpr bool kShare = DP > 128;       // small tiles: a wave's keys and values take turns in one image
  static constexpr int kSmall = kWaves * (kShare ? 1 : 2) * 32 * CH;
  static constexpr int G = DP / 32 < 4 ? DP / 32 : 4;  // 32-column blocks of a round of the waves' merge
  static constexpr int kMerge = kWaves * G * 8 * 32;
  static constexpr int kChunks = kLarge > kSmall ? (kLarge > kMerge ? kLarge : kMerge) : (kSmall > kMerge ? kSmall : kMerge);
};

// Rows of a load instruction: whole rows, a power of two of them, so that a page that is a multiple of it holds all of them.
template <int DP>
struct Load {
  static constexpr int CH = DP / 8;
  static constexpr int ROWS = CH == 8 ? 8 : CH == 32 ? 2 : 4;
};

// Where the keys and values of an item lie. Paged: a wave keeps two blocks of 64 entries of the item's page table in LDS, the
// one in use and the next, which it loads a tile ahead and in the order of the tiles' own loads: no address waits for the
// table. Pages of fewer than 4 positions, of which a tile may need more than a block, are looked up in memory.
constexpr int kBlock = 64;
constexpr int kRing = 2 * kBlock;

template <bool PAGED>
struct Source {
  const uint16_t* k;
  const uint16_t* v;
  int64_t k_p, k_t, v_p, v_t;
  const int* pages;
  const int* ring;
  int pool, loaded, last, last_page;
  Div page;
  bool bad;  // a page outside the pool: the item's rows become NaN

  __device__ __forceinline__ Source(const Args& a, const Item& it, int kvh, const int* wave_ring) {
    const int64_t from = PAGED ? 0 : it.begin;
    k = static_cast<const uint16_t*>(a.k) + kvh * a.k_h + from * a.k_t;
    v = static_cast<const uint16_t*>(a.v) + kvh * a.v_h + from * a.v_t;
    k_p = a.k_p;
    k_t = a.k_t;
    v_p = a.v_p;
    v_t = a.v_t;
    pool = a.pool;
    page = a.page;
    last = it.key1 - 1;
    bad = false;
    if constexpr (PAGED) {
      pages = a.table + static_cast<int64_t>(it.b) * a.table_stride;
      ring = wave_ring;
      last_page = page(last);
      loaded = -1;
    }
  }
  // Loads the blocks of the table up to the one of `key`, of a tile that begins at `first`.
  __device__ __forceinline__ void reach(int first, int key, int lane) {
    if constexpr (PAGED) {
      if (page.d < 4) return;
      const int to = min(page(key), last_page) / kBlock;
      if (loaded < 0) loaded = page(first) / kBlock - 1;
      while (loaded < to) {
        ++loaded;
        load_lds4(pages + min(loaded * kBlock + lane, last_page),
                  __builtin_amdgcn_readfirstlane(lds_address(ring)) + 4 * (loaded * kBlock % kRing));
      }
    }
  }
  // Element offsets of the row of a lane's key.
  __device__ __forceinline__ void at(int key, int64_t& ko, int64_t& vo) {
    key = min(key, last);
    if constexpr (PAGED) {
      const int n = page(key), slot = key - n * page.d;
      int id = page.d < 4 ? pages[n] : ring[n % kRing];
      if (static_cast<unsigned>(id) >= static_cast<unsigned>(pool)) {
        bad = true;
        id = 0;
      }
      ko = id * k_p + slot * k_t;
      vo = id * v_p + slot * v_t;
    } else {
      ko = key * k_t;
      vo = key * v_t;
    }
  }
};

__device__ __forceinline__ int64_t lane_value(int64_t v, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(v), lane);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane);
  return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}

// Loads ROWS rows from key0, of keys or of values, with the waves' instructions in turn; row r's element offset is lane r's
// `off`. Whole tiles whose load instructions each stay inside a page have a wave-uniform address and the lanes' offsets, which
// do not change from tile to tile; the others (a sequence's last tile, pages of odd sizes) an address a lane.
template <int DP, int ROWS, int WAVES, bool V, bool FULL, bool PAGED>
__device__ __forceinline__ void load_rows(const Source<PAGED>& src, const u32x4* img, int key0, int64_t off, int chunks, int wave,
                                          int lane) {
  constexpr int CH = DP / 8, R = Load<DP>::ROWS;
  static_assert(ROWS % (R * WAVES) == 0, "whole loads");
  const int sub = lane / CH, place = lane % CH;
  const uint16_t* from = V ? src.v : src.k;
  const int64_t stride = V ? src.v_t : src.k_t;
  const uint32_t base = __builtin_amdgcn_readfirstlane(lds_address(img));
  const bool mine = R * CH == kWave || sub < R;
  if (key0 + ROWS - 1 <= src.last && (!PAGED || src.page.d % R == 0)) {
#pragma unroll
    for (int i = 0; i < ROWS / (R * WAVES); ++i) {
      const int row0 = (i * WAVES + wave) * R, c = chunk_at<DP, V>(row0 + sub, place);
      const int64_t o = PAGED ? lane_value(off, row0) : (key0 + row0) * stride;
      const uint32_t rest = 2 * (static_cast<uint32_t>(sub) * static_cast<uint32_t>(stride) + 8u * c);
      if (mine && (FULL || c < chunks)) load_lds16(from + o, rest, base + 16 * row0 * CH);
    }
  } else {
#pragma unroll
    for (int i = 0; i < ROWS / (R * WAVES); ++i) {
      const int row0 = (i * WAVES + wave) * R, c = chunk_at<DP, V>(row0 + sub, place);
      const int64_t o = __shfl(off, row0 + sub);
      if (mine && (FULL || c < chunks)) load_lds16(from + o + 8 * c, base + 16 * row0 * CH);
    }
  }
}

// 128 rows, 32 a wave; the keys in steps of BN that all waves share in LDS, two images of each in turn. Bound by the matrix
// instructions with the softmax beside them (two workgroups a CU fill each other's gaps): a causal document of 16384 tokens, 16
// heads of 128, 1.09 to 1.14 ms or 965 to 1008 TFLOP/s, where a large library matrix product reaches 1206; heads of 64, whose
// softmax is the same for half the products, 820 (fp16) and 878 (bf16). With few tiles a step waits for its loads (about 2.5 us a
// step of one workgroup alone), which is what dividing the keys is for.
template <class T, int DP, bool PAGED, bool FULL>
__device__ __forceinline__ void large_tile(const Args& a, const Item& it, int kvh, u32x4* smem, const int* ring) {
  using S = Shape<DP>;
  constexpr int BN = S::BN, NB = S::NB, IMG = BN * S::CH;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int top = it.row0 + it.rows - 1;
  const int row = it.row0 + 32 * wave + (lane & 31);
  const int mine = min(row, top);
  const bool active = it.row0 + 32 * wave <= top;
  u32x4 q[DP / 16];
  load_q<T, DP, FULL>(a, it, kvh, mine, q, lane);
  const int limit = a.causal ? min(it.first + a.group(mine), it.keys - 1) : it.keys - 1;
  const int least = __builtin_amdgcn_readfirstlane(limit), most = __builtin_amdgcn_readlane(limit, 31);
  Running<DP> r;
  r.clear();
  Source<PAGED> src(a, it, kvh, ring);
  const int chunks = a.d / 8, last = it.key1 - 1;
  int buf = 0;
  const auto load = [&](int key, int to) {
    int64_t ko, vo;
    src.at(key + lane % BN, ko, vo);
    load_rows<DP, BN, kWaves, false, FULL>(src, smem + to * IMG, key, ko, chunks, wave, lane);
    load_rows<DP, BN, kWaves, true, FULL>(src, smem + (2 + to) * IMG, key, vo, chunks, wave, lane);
  };
  if (it.key0 < it.key1) {
    src.reach(it.key0, it.key0 + 2 * BN - 1, lane);
    if constexpr (PAGED) wait_vm<0>();
    load(it.key0, 0);
  }
  wait_vm<0>();  // the queries, too
  const auto next = [&](int key) {
    wait_vm<0>();
    __syncthreads();
    if (key + BN < it.key1) {
      src.reach(key, key + 3 * BN - 1, lane);
      load(key + BN, buf ^ 1);
    }
  };
  // The steps that hold a key for this wave, then those that only the other waves need (two loops: with one and a condition
  // the sums went to other registers and back in every step).
  int key = it.key0;
  const int mine_end = active ? min(it.key1, most + 1) : it.key0;
  for (; key < mine_end; key += BN) {
    next(key);
    f32x16 s[NB];
    u32x4 p[NB][2];
#pragma unroll
    for (int b = 0; b < NB; ++b) s[b] = scores<T, DP>(smem + buf * IMG, 32 * b, q, lane);
    softmax_step<T, DP, NB>(s, p, r, a.scale_log2, key, min(limit, last), key + BN - 1 > min(least, last), lane);
#pragma unroll
    for (int b = 0; b < NB; ++b) weighted<T, DP>(smem + (2 + buf) * IMG, 32 * b, p[b], r.o, lane);
    buf ^= 1;
  }
  for (; key < it.key1; key += BN) {
    next(key);
    buf ^= 1;
  }
  if constexpr (PAGED) {
    if (__syncthreads_or(src.bad)) r.l = NAN;
  }
  if (active) write_rows<T, DP>(a, it, kvh, row, r, lane);
}

// Up to 32 rows: every wave has all rows and takes every fourth block of 32 keys, through images of its own; then the waves'
// parts are joined. Bound by memory: a wave has keys or values in flight at any time, 128 KB a CU at most (64 sequences of 4096
// keys, 8 heads of 128, one token each: 198 us, 5.4 TB/s; 14 TB/s where the caches hold the keys, so the products do not count).
// A short call (161 keys) is 8 us: the plan 0.9, the queries and the table 0.8, its loads 2.9, the rest products and joins.
template <class T, int DP, bool PAGED, bool FULL>
__device__ __forceinline__ void small_tile(const Args& a, const Item& it, int kvh, u32x4* smem, float* stats, const int* ring) {
  using S = Shape<DP>;
  constexpr int IMG = 32 * S::CH, LOADS = 32 / Load<DP>::ROWS;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int top = it.row0 + it.rows - 1;
  const int mine = min(it.row0 + (lane & 31), top);
  u32x4 q[DP / 16];
  load_q<T, DP, FULL>(a, it, kvh, mine, q, lane);
  const int limit = a.causal ? min(it.first + a.group(mine), it.keys - 1) : it.keys - 1;
  const int least = __builtin_amdgcn_readfirstlane(limit);
  Running<DP> r;
  r.clear();
  Source<PAGED> src(a, it, kvh, ring);
  const int chunks = a.d / 8, last = it.key1 - 1;
  u32x4* kimg = smem + wave * (S::kShare ? 1 : 2) * IMG;
  u32x4* vimg = S::kShare ? kimg : kimg + IMG;
  constexpr int STEP = 32 * kWaves;
  int key = it.key0 + 32 * wave;
  int64_t ko, vo;
  if (key < it.key1) src.reach(key, key + STEP + 31, lane);
  if constexpr (PAGED) wait_vm<0>();  // the table and the queries
  if (key < it.key1) {
    src.at(key + lane % 32, ko, vo);
    load_rows<DP, 32, 1, false, FULL>(src, kimg, key, ko, chunks, 0, lane);
    if constexpr (!S::kShare) load_rows<DP, 32, 1, true, FULL>(src, vimg, key, vo, chunks, 0, lane);
  }
  if constexpr (!PAGED) wait_vm<0>();  // the queries
  for (; key < it.key1; key += STEP) {
    const bool more = key + STEP < it.key1;
    if constexpr (S::kShare) wait_vm<0>();
    else wait_vm<LOADS>();  // the keys: only the values' loads are younger
    f32x16 s[1] = {scores<T, DP>(kimg, 0, q, lane)};
    u32x4 p[1][2];
    wait_lds();  // the keys are in registers: their image is free
    if constexpr (S::kShare) load_rows<DP, 32, 1, true, FULL>(src, vimg, key, vo, chunks, 0, lane);
    if (more) {
      src.reach(key, key + 2 * STEP + 31, lane);
      src.at(key + STEP + lane % 32, ko, vo);
      if constexpr (!S::kShare) load_rows<DP, 32, 1, false, FULL>(src, kimg, key + STEP, ko, chunks, 0, lane);
    }
    softmax_step<T, DP, 1>(s, p, r, a.scale_log2, key, min(limit, last), key + 31 > min(least, last), lane);
    if (!S::kShare && more) wait_vm<LOADS>();
    else wait_vm<0>();
    weighted<T, DP>(vimg, 0, p[0], r.o, lane);
    wait_lds();
    if (more) {
      if constexpr (S::kShare) load_rows<DP, 32, 1, false, FULL>(src, kimg, key + STEP, ko, chunks, 0, lane);
      else load_rows<DP, 32, 1, true, FULL>(src, vimg, key + STEP, vo, chunks, 0, lane);
    }
  }
  if (PAGED && __any(src.bad)) r.l = NAN;
  join_waves<T, DP, S::G>(a, it, kvh, r, smem, stats);
}

// 256 columns: a wave's sums alone are 128 registers, so one workgroup a CU with all of them.
template <class T, int DP, bool PAGED, bool FULL>
__global__ __launch_bounds__(kThreads, DP > 128 ? 1 : 2) void attention_kernel(Args a) {
  using S = Shape<DP>;
  __shared__ __align__(16) u32x4 smem[S::kChunks];
  __shared__ float stats[32 * (2 * kWaves + 1)];
  __shared__ int rings[PAGED ? kWaves * kRing : 1];
  const int* ring = rings + (PAGED ? threadIdx.x / kWave * kRing : 0);
  const int index = a.hk(blockIdx.x), kvh = blockIdx.x - index * a.hk.d;
  const Item it = find_item<false>(a, index);
  if (it.b < 0) {
    fill_rest(a, kvh, it.extra, a.hk(gridDim.x) - (index - it.extra));
    return;
  }
  if (it.key0 >= it.key1 && it.split > 0) return;
  if constexpr (!FULL) {
    for (int i = threadIdx.x; i < S::kChunks; i += kThreads) smem[i] = u32x4{};
    __syncthreads();
  }
  if (it.small) small_tile<T, DP, PAGED, FULL>(a, it, kvh, smem, stats, ring);
  else large_tile<T, DP, PAGED, FULL>(a, it, kvh, smem, ring);
}

// A unit's rows, a thread 4 columns of one, whose parts it loads kMergeParts at a time. MORE: there are more parts than that (the
// form without the running sums is 5 us faster where there are not: prompts of 2047 and 1300 tokens, heads of 64, in 3 and 2 parts
// a tile, 45 us in all against 40).
template <class T, int DP, bool MORE>
__device__ __forceinline__ void merge_rows(const Args& a, const Item& it, int kvh, const float* ws, int64_t step) {
  const int pieces = a.d / 4;
  for (int i = threadIdx.x; i < it.rows * pieces; i += kThreads) {
    const int row = it.split + i / pieces, col = 4 * (i % pieces);
    float top = -INFINITY, sum = 0.f;
    f32x4 o = {};
    for (int s0 = 0; s0 < (MORE ? it.splits : 1); s0 += kMergeParts) {
      float m[kMergeParts], l[kMergeParts];
      f32x4 x[kMergeParts];
#pragma unroll
      for (int s = 0; s < kMergeParts; ++s) {
        if (s0 + s >= it.splits) break;
        const float* p = ws + (s0 + s) * step;
        m[s] = p[a.ws_rows * DP + row];
        l[s] = p[a.ws_rows * (DP + 1) + row];
        x[s] = *reinterpret_cast<const f32x4*>(p + row * DP + col);
      }
      float now = top;
#pragma unroll
      for (int s = 0; s < kMergeParts; ++s) {
        if (s0 + s >= it.splits) break;
        now = fmaxf(now, m[s]);
      }
      if constexpr (MORE) {
        const float before = rescaled(top, now, a.scale_log2);
        sum *= before;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] *= before;
      }
      top = now;
#pragma unroll
      for (int s = 0; s < kMergeParts; ++s) {
        if (s0 + s >= it.splits) break;
        const float f = rescaled(m[s], top, a.scale_log2);
        sum += l[s] * f;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += x[s][e] * f;
      }
    }
    const float inv = inverse(sum);
    *reinterpret_cast<u32x2*>(out_row(a, it, kvh, it.row0 + row) + col) =
        u32x2{T::result(o[0] * inv, o[1] * inv), T::result(o[2] * inv, o[3] * inv)};
  }
}

// Joins the partials of a unit's rows: the parts' sums, each times exp2 of its maximum less the greatest. Few parts or many
// rows: merge_rows. Few rows of many parts: the workgroup has one row, whose parts its groups of d / 4 threads share (one
// thread after another part took 30 us for 80 parts of 36 rows).
template <class T, int DP, class P>
__global__ __launch_bounds__(kThreads) void merge_kernel(Args a) {
  __shared__ float red[kWaves];
  __shared__ f32x4 sums[kThreads];
  __shared__ float total[kThreads];
  const int index = a.hk(blockIdx.x), kvh = blockIdx.x - index * a.hk.d;
  const int tid = threadIdx.x, pieces = a.d / 4;
  const int64_t step = static_cast<int64_t>(a.hk.d) * a.ws_rows * (DP + 2);
  for (int unit = index;; unit += a.hk(gridDim.x)) {
    const Item it = find_item<true, P>(a, unit);
    if (it.b < 0) return;
    if (it.slot + it.splits > a.slots) continue;
    const float* ws = slot_at<DP>(a, it.slot, kvh);
    if (it.splits <= kMergeParts) {
      merge_rows<T, DP, false>(a, it, kvh, ws, step);
      continue;
    }
    if (!it.small) {
      merge_rows<T, DP, true>(a, it, kvh, ws, step);
      continue;
    }
    const int row = it.split;
    const float* stats = ws + a.ws_rows * DP + row;
    float top = -INFINITY;
    for (int s = tid; s < it.splits; s += kThreads) top = fmaxf(top, stats[s * step]);
    top = xor_butterfly<true>(top, MaxOp());
    __syncthreads();  // the last unit's sums are read
    if ((tid & 63) == 0) red[tid / kWave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const int groups = kThreads / pieces, g = tid / pieces, piece = tid - g * pieces;
    float sum = 0.f;
    f32x4 o = {};
    if (g < groups) {
#pragma unroll 8
      for (int s = g; s < it.splits; s += groups) {
        const float ms = stats[s * step];
        const f32x4 xs = *reinterpret_cast<const f32x4*>(ws + s * step + row * DP + 4 * piece);
        const float f = rescaled(ms, top, a.scale_log2);
        sum += stats[s * step + a.ws_rows] * f;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += xs[e] * f;
      }
      sums[tid] = o;
      total[tid] = sum;
    }
    __syncthreads();
    if (g == 0) {
      for (int n = 1; n < groups; ++n) {
        sum += total[n * pieces + piece];
        o += sums[n * pieces + piece];
      }
      const float inv = inverse(sum);
      *reinterpret_cast<u32x2*>(out_row(a, it, kvh, it.row0 + row) + 4 * piece) =
          u32x2{T::result(o[0] * inv, o[1] * inv), T::result(o[2] * inv, o[3] * inv)};
    }
  }
}

// The append: piece c of head h of token tok goes to the token's place in its sequence's pages.
struct Append {
  const void* k;
  const void* v;
  void* k_pages;
  void* v_pages;
  const int* cu;
  const int* lengths;
  const int* table;
  int64_t k_t, k_h, v_t, v_h, kp_p, kp_t, kp_h, vp_p, vp_t, vp_h, table_stride;  // bytes, table_stride in entries
  Div page;
  int tokens, seqs, pool, max_keys, hk, pieces;
};

// E: a piece, 16 bytes where every row is made of aligned ones, else one element. Bound by memory: 7889 tokens of 16 heads of 128
// in 21 us, 6.2 TB/s read and written.
template <class E>
__global__ __launch_bounds__(kThreads) void append_kernel(Append a) {
  const int64_t per = static_cast<int64_t>(a.hk) * a.pieces, total = a.tokens * per;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int tok = static_cast<int>(i / per), rest = static_cast<int>(i - tok * per), h = rest / a.pieces, c = rest % a.pieces;
    int lo = 0, hi = a.seqs;  // the last sequence that begins at or before tok
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (a.cu[mid] <= tok) lo = mid;
      else hi = mid;
    }
    const int end = a.cu[lo + 1];
    if (tok < a.cu[lo] || tok >= end) continue;
    const int pos = max(a.lengths[lo], 0) - (min(end, a.tokens) - tok);  // offsets are cut as the attention cuts them
    if (static_cast<unsigned>(pos) >= static_cast<unsigned>(a.max_keys)) continue;
    const int n = a.page(pos), slot = pos - n * a.page.d;
    const int id = a.table[lo * a.table_stride + n];
    if (static_cast<unsigned>(id) >= static_cast<unsigned>(a.pool)) continue;
    const auto from = [&](const void* p, int64_t t, int64_t hs) {
      return reinterpret_cast<const E*>(static_cast<const char*>(p) + tok * t + h * hs) + c;
    };
    const auto to = [&](void* p, int64_t ps, int64_t t, int64_t hs) {
      return reinterpret_cast<E*>(static_cast<char*>(p) + id * ps + slot * t + h * hs) + c;
    };
    *to(a.k_pages, a.kp_p, a.kp_t, a.kp_h) = *from(a.k, a.k_t, a.k_h);
    *to(a.v_pages, a.vp_p, a.vp_t, a.vp_h) = *from(a.v, a.v_t, a.v_h);
  }
}

template <class T, int DP, bool PAGED>
int launch(const Args& a, const Launch& n, hipStream_t st) {
  const unsigned grid = static_cast<unsigned>(n.index * a.hk.d);
  if (a.d == DP) attention_kernel<T, DP, PAGED, true><<<grid, kThreads, 0, st>>>(a);
  else attention_kernel<T, DP, PAGED, false><<<grid, kThreads, 0, st>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return static_cast<int>(e);
  return n.merges > 0 ? launch_merge<Tiles32>(std::is_same<T, Bf16>::value ? BP_DT_BF16 : BP_DT_F16, a, n, st) : BP_OK;
}

template <class T, bool PAGED>
int launch_dim(const Args& a, const Launch& n, hipStream_t st) {
  switch (padded_dim(a.d)) {
    case 64: return launch<T, 64, PAGED>(a, n, st);
    case 96: return launch<T, 96, PAGED>(a, n, st);
    case 128: return launch<T, 128, PAGED>(a, n, st);
    default: return launch<T, 256, PAGED>(a, n, st);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int run(int dtype, Args& a, bool paged, size_t ws_bytes, hipStream_t st) {
  const int hk = a.hk.d;
  if (dtype != BP_DT_BF16 && dtype != BP_DT_F16) return BP_E_UNSUPPORTED;
  if (a.tokens < 0 || a.seqs < 0 || hk <= 0 || a.hq <= 0 || a.hq % hk != 0 || !(a.scale_log2 > 0.f && a.scale_log2 <= FLT_MAX) ||
      a.max_keys < 0)
    return BP_E_INVALID_ARG;
  if (a.d <= 0 || a.d % 8 != 0 || a.d > 256) return BP_E_UNSUPPORTED;
  if (a.tokens == 0) return BP_OK;
  if (a.q == nullptr || a.out == nullptr || (a.seqs > 0 && a.cu == nullptr)) return BP_E_INVALID_ARG;
  // a stride that nothing is multiplied with may be anything
  if (a.tokens == 1) a.q_t = 0;
  if (a.hq == 1) a.q_h = 0;
  if (hk == 1) a.k_h = a.v_h = 0;
  if (paged ? a.page.d == 1 : a.tokens == 1) a.k_t = a.v_t = 0;
  if (a.pool == 1) a.k_p = a.v_p = 0;
  if (!aligned16(a.q) || !aligned16(a.k) || !aligned16(a.v) || !aligned16(a.out) ||
      ((a.q_t | a.q_h | a.k_p | a.k_t | a.k_h | a.v_p | a.v_t | a.v_h) & 7) != 0)
    return BP_E_INVALID_ARG;
  // rows of a sequence, keys plus a split, and the byte offsets inside a load instruction, in 32 bits
  if (static_cast<int64_t>(a.tokens) * a.hq >= (1ll << 30) || a.max_keys >= (1 << 29) || a.k_t < 0 || a.v_t < 0 ||
      a.k_t >= (1 << 28) || a.v_t >= (1 << 28))
    return BP_E_UNSUPPORTED;
  Launch n;
  if (!plan_launch(a, n)) return BP_E_UNSUPPORTED;
  if (n.workspace > 0 && (a.ws == nullptr || ws_bytes < n.workspace || !aligned16(a.ws))) return BP_E_WORKSPACE;
  if (n.workspace == 0) a.ws = nullptr;
  // A row of q is read by the tile that writes its result and by no other, so out may be q itself.
  const auto bytes = [&](int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t n2, int64_t s2) {
    return n0 > 0 ? 2 * ((n0 - 1) * s0 + (n1 - 1) * s1 + (n2 - 1) * s2 + a.d) : 0;
  };
  const int64_t dense = static_cast<int64_t>(a.hq) * a.d, out = 2 * dense * a.tokens, keys = paged ? a.page.d : a.tokens;
  const bool in_place = a.out == a.q && (a.tokens == 1 || a.q_t == dense) && (a.hq == 1 || a.q_h == a.d);
  if ((!in_place && ranges_overlap(a.out, out, a.q, bytes(a.tokens, a.q_t, a.hq, a.q_h, 1, 0))) ||
      ranges_overlap(a.out, out, a.k, bytes(paged ? a.pool : 1, a.k_p, keys, a.k_t, hk, a.k_h)) ||
      ranges_overlap(a.out, out, a.v, bytes(paged ? a.pool : 1, a.v_p, keys, a.v_t, hk, a.v_h)))
    return BP_E_INVALID_ARG;
  if (dtype == BP_DT_BF16)
    return paged ? launch_dim<Bf16, true>(a, n, st) : launch_dim<Bf16, false>(a, n, st);
  return paged ? launch_dim<F16, true>(a, n, st) : launch_dim<F16, false>(a, n, st);
}

}  // namespace

template <class T, class P>
void merge(const Args& a, unsigned grid, hipStream_t st) {
  switch (padded_dim(a.d)) {
    case 64: merge_kernel<T, 64, P><<<grid, kThreads, 0, st>>>(a); break;
    case 96: merge_kernel<T, 96, P><<<grid, kThreads, 0, st>>>(a); break;
    case 128: merge_kernel<T, 128, P><<<grid, kThreads, 0, st>>>(a); break;
    default: merge_kernel<T, 256, P><<<grid, kThreads, 0, st>>>(a);
  }
}

template <class P>
int launch_merge(int dtype, const Args& a, const Launch& n, hipStream_t st) {
  const unsigned grid = static_cast<unsigned>(n.merges * a.hk.d);
  if (dtype == BP_DT_BF16) merge<Bf16, P>(a, grid, st);
  else merge<F16, P>(a, grid, st);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? BP_OK : static_cast<int>(e);
}
template int launch_merge<Tiles32>(int, const Args&, const Launch&, hipStream_t);
template int launch_merge<FewTiles<1>>(int, const Args&, const Launch&, hipStream_t);
template int launch_merge<FewTiles<2>>(int, const Args&, const Launch&, hipStream_t);
template int launch_merge<FewTiles<3>>(int, const Args&, const Launch&, hipStream_t);

}  // namespace attn
}  // namespace bp

extern "C" {

size_t bp_attn_workspace_bytes(int64_t tokens, int64_t seqs, int64_t hq, int64_t hk, int64_t head_dim, int64_t max_keys) {
  return bp::attn::workspace_bytes(tokens, seqs, hq, hk, head_dim, max_keys);
}

int bp_attn_packed(int dtype, const void* q, const void* k, const void* v, void* out, const int32_t* cu, int tokens, int seqs,
                   int hq, int hk, int head_dim, int64_t q_t, int64_t q_h, int64_t k_t, int64_t k_h, int64_t v_t, int64_t v_h,
                   int causal, float scale, void* workspace, size_t workspace_bytes, void* stream) {
  bp::attn::Args a = {};
  if (tokens > 0 && (k == nullptr || v == nullptr)) return BP_E_INVALID_ARG;
  a.q = q, a.k = k, a.v = v, a.out = out, a.cu = cu;
  a.ws = static_cast<float*>(workspace);
  a.q_t = q_t, a.q_h = q_h, a.k_t = k_t, a.k_h = k_h, a.v_t = v_t, a.v_h = v_h;
  a.tokens = tokens, a.seqs = seqs, a.hq = hq, a.hk.d = hk, a.d = head_dim, a.causal = causal != 0;
  a.max_keys = tokens;
  a.page = bp::attn::Div::of(1);
  a.scale_log2 = scale * 1.44269504088896340736f;
  return bp::attn::run(dtype, a, false, workspace_bytes, static_cast<hipStream_t>(stream));
}

int bp_attn_paged(int dtype, const void* q, const void* k_pages, const void* v_pages, void* out, const int32_t* table,
                  int64_t table_stride, const int32_t* lengths, const int32_t* cu, int tokens, int seqs, int pool, int page,
                  int max_pages, int hq, int hk, int head_dim, int64_t q_t, int64_t q_h, int64_t k_p, int64_t k_t, int64_t k_h,
                  int64_t v_p, int64_t v_t, int64_t v_h, float scale, void* workspace, size_t workspace_bytes, void* stream) {
  if (page <= 0 || pool < 0 || max_pages < 0 || static_cast<int64_t>(page) * max_pages >= (1ll << 29)) return BP_E_INVALID_ARG;
  if (tokens > 0 && seqs > 0 &&
      (lengths == nullptr || (max_pages > 0 && (table == nullptr || k_pages == nullptr || v_pages == nullptr || pool == 0))))
    return BP_E_INVALID_ARG;
  bp::attn::Args a = {};
  a.q = q, a.k = k_pages, a.v = v_pages, a.out = out, a.cu = cu, a.lengths = lengths, a.table = table;
  a.ws = static_cast<float*>(workspace);
  a.q_t = q_t, a.q_h = q_h, a.k_p = k_p, a.k_t = k_t, a.k_h = k_h, a.v_p = v_p, a.v_t = v_t, a.v_h = v_h;
  a.table_stride = table_stride;
  a.tokens = tokens, a.seqs = seqs, a.hq = hq, a.hk.d = hk, a.d = head_dim, a.causal = 1;
  a.pool = pool, a.page = bp::attn::Div::of(page);
  a.max_keys = page * max_pages;
  a.scale_log2 = scale * 1.44269504088896340736f;
  return bp::attn::run(dtype, a, true, workspace_bytes, static_cast<hipStream_t>(stream));
}

int bp_paged_append(int element_bytes, const void* k, const void* v, void* k_pages, void* v_pages, const int32_t* table,
                    int64_t table_stride, const int32_t* lengths, const int32_t* cu, int tokens, int seqs, int pool, int page,
                    int max_pages, int hk, int head_dim, int64_t k_t, int64_t k_h, int64_t v_t, int64_t v_h, int64_t kp_p,
                    int64_t kp_t, int64_t kp_h, int64_t vp_p, int64_t vp_t, int64_t vp_h, void* stream) {
  if ((element_bytes != 1 && element_bytes != 2 && element_bytes != 4) || tokens < 0 || seqs < 0 || pool < 0 || page <= 0 ||
      max_pages < 0 || static_cast<int64_t>(page) * max_pages >= (1ll << 29) || hk < 0 || head_dim < 0)
    return BP_E_INVALID_ARG;
  if (tokens == 0 || seqs == 0 || pool == 0 || max_pages == 0 || hk == 0 || head_dim == 0) return BP_OK;
  if (k == nullptr || v == nullptr || k_pages == nullptr || v_pages == nullptr || table == nullptr || lengths == nullptr ||
      cu == nullptr)
    return BP_E_INVALID_ARG;
  const int64_t row = static_cast<int64_t>(head_dim) * element_bytes;
  if (hk * row >= (1ll << 31)) return BP_E_UNSUPPORTED;
  bp::attn::Append a = {};
  a.k = k, a.v = v, a.k_pages = k_pages, a.v_pages = v_pages, a.cu = cu, a.lengths = lengths, a.table = table;
  a.k_t = k_t * element_bytes, a.k_h = k_h * element_bytes, a.v_t = v_t * element_bytes, a.v_h = v_h * element_bytes;
  a.kp_p = kp_p * element_bytes, a.kp_t = kp_t * element_bytes, a.kp_h = kp_h * element_bytes;
  a.vp_p = vp_p * element_bytes, a.vp_t = vp_t * element_bytes, a.vp_h = vp_h * element_bytes;
  a.table_stride = table_stride;
  a.tokens = tokens, a.seqs = seqs, a.pool = pool, a.page = bp::attn::Div::of(page);
  a.max_keys = page * max_pages, a.hk = hk;
  const bool wide = bp::attn::aligned16(k) && bp::attn::aligned16(v) && bp::attn::aligned16(k_pages) &&
                    bp::attn::aligned16(v_pages) && row % 16 == 0 &&
                    ((a.k_t | a.k_h | a.v_t | a.v_h | a.kp_p | a.kp_t | a.kp_h | a.vp_p | a.vp_t | a.vp_h) & 15) == 0;
  a.pieces = wide ? static_cast<int>(row / 16) : head_dim;
  const int64_t total = static_cast<int64_t>(tokens) * hk * a.pieces;
  int64_t blocks = (total + bp::attn::kThreads - 1) / bp::attn::kThreads;
  if (blocks > 16384) blocks = 16384;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(blocks));
  if (wide) bp::attn::append_kernel<bp::u32x4><<<grid, bp::attn::kThreads, 0, st>>>(a);
  else if (element_bytes == 1) bp::attn::append_kernel<uint8_t><<<grid, bp::attn::kThreads, 0, st>>>(a);
  else if (element_bytes == 2) bp::attn::append_kernel<uint16_t><<<grid, bp::attn::kThreads, 0, st>>>(a);
  else bp::attn::append_kernel<uint32_t><<<grid, bp::attn::kThreads, 0, st>>>(a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? BP_OK : static_cast<int>(e);
}

}  // extern "C"
