// Log probabilities of given tokens, the entropy and the most likely tokens of rows of logits, in one pass over the logits.
//
//   m = max x, z = sum exp(x - m), w = sum exp(x - m) (x - m):  log p(t) = x_t - m - ln z,  H = ln z - w / z
//
// in units of log2: d = x log2(e) - m2 is one fused multiply-add, with m2 = m log2(e) rounded once and used everywhere. A wave
// keeps one running m2 (all lanes the same) and its lanes' own z and w relative to it; a batch of logits that holds a greater
// one rescales them: z' = f z, w' = f (w + dm z) with f = exp2(dm), dm = m2 - m2'. Held in fp32: logits as they are,
// exponentials, sums. m2 starts at -kFar: what lies far below it (masked tokens, whatever value masks them) adds nothing.
//
// The most likely tokens, greater logit first, then lower index: a wave appends the batch's logits above its threshold to a
// list in LDS; a full list is cut to its best `top`, whose last is the new threshold, and every wave uses the greatest
// threshold of its workgroup (`top` entries reach each of them, so no answer depends on which it saw).
//
// Two kinds of rows are done again by plain passes over memory: the order of those whose z is NaN (a NaN or +inf among the
// logits makes every log probability NaN, as log softmax does; NaN counts as greatest in the order), and the statistics of those
// whose m2 is kFar = 2^24 or more either way. There a step of m2 is more than 1: what its rounding leaves goes into the exponent
// of every term, and from 2^31 on out of exp2's range. Those take the difference of the logits first.

#include "byteprof_amd.h"
#include "common.h"

namespace bp {
namespace logprobs {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kMaxTop = 32;
constexpr int kFull = 64;      // entries of a wave's list that a piece of every lane may come to
constexpr int kCap = kFull + kWave * 8;
constexpr int kVectors = 4;    // 16-byte loads of a lane in flight
constexpr int kStatWords = 4;
constexpr int kMaxParts = 64;  // workgroups of a row: one lane each in the merge
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr int kNoIndex = 0x7fffffff;
constexpr float kFar = 16777216.f;

struct Args {
  const void* logits;
  const int64_t* targets;  // or null
  float* logprob;          // with targets
  float* entropy;
  int64_t* top_ids;
  float* top_logprobs;
  float* ws;  // [rows][parts][kStatWords + 2 top]: m, z, w, then the best entries' keys
  int64_t stride;  // elements
  int vocab, top, parts, per_part;  // per_part: 16-byte pieces of a part
};

// An entry of a list: the logit's bits in the order of the numbers, then the index counted down; a greater key comes earlier.
// 0 is none.
using Key = unsigned long long;
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 as +0
  return b ^ (static_cast<uint32_t>(static_cast<int>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return __uint_as_float(o ^ (static_cast<uint32_t>(static_cast<int>(~o) >> 31) | 0x80000000u));
}
__device__ __forceinline__ Key key_of(float x, int i) {
  return static_cast<Key>(order_of(x)) << 32 | static_cast<uint32_t>(kNoIndex - i);
}
__device__ __forceinline__ float logit_of(Key k) { return value_of(static_cast<uint32_t>(k >> 32)); }
__device__ __forceinline__ int index_of(Key k) { return kNoIndex - static_cast<int>(k & 0xffffffffu); }

template <class E>
struct Type;
template <>
struct Type<uint16_t> {  // bf16
  static __device__ __forceinline__ float value(uint16_t v) { return bf16_bits_to_float(v); }
  static __device__ __forceinline__ uint16_t lowest() { return 0xff80; }
};
template <>
struct Type<_Float16> {
  static __device__ __forceinline__ float value(_Float16 v) { return static_cast<float>(v); }
  static __device__ __forceinline__ _Float16 lowest() { return static_cast<_Float16>(-INFINITY); }
};
template <>
struct Type<float> {
  static __device__ __forceinline__ float value(float v) { return v; }
  static __device__ __forceinline__ float lowest() { return -INFINITY; }
};

__device__ __forceinline__ float wave_max(float v) { return xor_butterfly<true>(v, MaxOp()); }
__device__ __forceinline__ float wave_sum(float v) { return xor_butterfly<true>(v, AddOp()); }

// The number of the `count` entries that come before `mine`; the list is readable kPad entries past its end.
constexpr int kPad = 8;
__device__ __forceinline__ int rank_in(const Key* list, int count, Key mine) {
  int rank = 0;
  for (int n = 0; n < count; n += kPad) {
    Key e[kPad];
#pragma unroll
    for (int u = 0; u < kPad; ++u) e[u] = list[n + u];
    if (n + kPad <= count) {
#pragma unroll
      for (int u = 0; u < kPad; ++u) rank += static_cast<int>(e[u] > mine);
    } else {
#pragma unroll
      for (int u = 0; u < kPad; ++u) rank += static_cast<int>((n + u < count) & (e[u] > mine));
    }
  }
  return rank;
}

// The best `keep` of the `count` entries of a wave's list to its front, in order. Returns how many that are.
__device__ __forceinline__ int cut(Key* list, Key* out, int count, int keep, int lane) {
  for (int n = 0; n < count; n += kWave) {
    const Key mine = n + lane < count ? list[n + lane] : 0;
    const int rank = rank_in(list, count, mine);
    if (mine != 0 && rank < keep) out[rank] = mine;
  }
  __builtin_amdgcn_wave_barrier();
  const int left = min(count, keep);
  if (lane < left) list[lane] = out[lane];
  __builtin_amdgcn_wave_barrier();
  return left;
}

// The lanes' entries (those with `in`) to the end of the list.
__device__ __forceinline__ void append(Key* list, int& count, bool in, Key e) {
  const uint64_t mask = __ballot(in);
  if (in)
    list[count + __builtin_amdgcn_mbcnt_hi(static_cast<unsigned>(mask >> 32),
                                           __builtin_amdgcn_mbcnt_lo(static_cast<unsigned>(mask), 0))] = e;
  count += __popcll(mask);
  __builtin_amdgcn_wave_barrier();
}

struct Stats {
  float m, z, w;  // m and w in units of log2
};

__device__ __forceinline__ Stats join(const Stats& a, const Stats& b) {
  Stats r;
  r.m = fmaxf(a.m, b.m);
  const auto part = [&](const Stats& s, float& z, float& w) {
    const float dm = s.m == r.m ? 0.f : s.m - r.m;  // (both may be +inf)
    const float f = s.m == r.m ? 1.f : __builtin_amdgcn_exp2f(dm);
    z += f * s.z;
    w += f == 0.f ? 0.f * s.z : f * (s.w + dm * s.z);
  };
  r.z = r.w = 0.f;
  part(a, r.z, r.w);
  part(b, r.z, r.w);
  return r;
}

// The wave's part of a row: pieces of 16 bytes from `first` to `last`, the workgroup's waves in turn.
template <class E>
struct Pass {
  static constexpr int PER = 16 / sizeof(E);
  static constexpr int N = kVectors * PER;
  const E* row;
  int vocab, head, last, top, lane;
  int least, whole;  // the pieces from least to whole are inside the row (whole: inside the part as well)
  Key* list;
  Key* out;
  Stats s;
  Key threshold;  // keys above it are taken
  float tx;       // its logit
  int count;

  // A lane's pieces of a batch: piece p holds elements p PER - head ...; the first and the last may reach over the row's ends.
  __device__ __forceinline__ void fetch(int p0, u32x4 (&raw)[kVectors]) const {
    if (p0 >= least && p0 + (kVectors - 1) * kThreads + kWave <= whole) {  // all inside the row and the part
#pragma unroll
      for (int v = 0; v < kVectors; ++v)
        raw[v] = *as_global(reinterpret_cast<const u32x4*>(row + ((p0 + v * kThreads + lane) * PER - head)));
      return;
    }
#pragma unroll
    for (int v = 0; v < kVectors; ++v) {
      const int p = p0 + v * kThreads + lane, at = p * PER - head;
      E part[PER];
#pragma unroll
      for (int e = 0; e < PER; ++e) part[e] = Type<E>::lowest();
      if (p >= least && p < whole) {
        const u32x4 r = *as_global(reinterpret_cast<const u32x4*>(row + at));
        __builtin_memcpy(part, &r, 16);
      } else if (p < last) {
#pragma unroll
        for (int e = 0; e < PER; ++e)
          if (inside(p, at + e)) part[e] = as_global(row)[at + e];
      }
      __builtin_memcpy(&raw[v], part, 16);
    }
  }
  __device__ __forceinline__ static void unpack(const u32x4 (&raw)[kVectors], float (&x)[N], float (&most)[kVectors], float& best) {
    best = -INFINITY;
#pragma unroll
    for (int v = 0; v < kVectors; ++v) {
      E part[PER];
      __builtin_memcpy(part, &raw[v], 16);
      most[v] = -INFINITY;
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        x[v * PER + e] = Type<E>::value(part[e]);
        most[v] = fmaxf(most[v], x[v * PER + e]);
      }
      best = fmaxf(best, most[v]);
    }
  }
  __device__ __forceinline__ bool inside(int p, int at) const { return (p < last) & (at >= 0) & (at < vocab); }
  __device__ __forceinline__ void raise(Key to) {
    // what lies below -inf is no number: everything is taken
    const bool any = (to >> 32) < order_of(-INFINITY);
    threshold = any ? 0 : to;
    tx = any ? -INFINITY : logit_of(to);
  }

  // The batches from `first` on. lanes: LDS for the workgroup's first maxima; shared: for the waves' thresholds.
  __device__ __forceinline__ void run(int first, uint32_t* lanes, volatile uint32_t* shared, int wave) {
    s = Stats{-kFar, 0.f, 0.f};
    raise(0);
    count = 0;
    least = head > 0 ? 1 : 0;
    whole = min(last, (vocab + head) / PER);
    float x[N], most[kVectors], best;
    u32x4 raw[kVectors];
    fetch(first + wave * kWave, raw);
    if (top > 0) {
      // the first threshold: the `top`-th greatest of the lanes' best of the first batch, over the workgroup (`top` entries
      // reach it)
      unpack(raw, x, most, best);
      // (with the thread in place of the last 8 bits: no two are alike, and the threshold is a little lower)
      const uint32_t mine = (order_of(best) & ~0xffu) | (0xffu - (wave * kWave + lane));
      lanes[wave * kWave + lane] = mine;
      __syncthreads();
      int rank = 0;
#pragma unroll 8
      for (int n = 0; n < kThreads; n += 4) {
        const u32x4 o = *reinterpret_cast<const u32x4*>(lanes + n);
#pragma unroll
        for (int u = 0; u < 4; ++u) rank += static_cast<int>(o[u] > mine);
      }
      if (rank == top - 1) shared[kWaves] = mine & ~0xffu;
      __syncthreads();
      raise(static_cast<Key>(shared[kWaves]) << 32);
    }
    for (int p0 = first + wave * kWave; p0 < last; p0 += kThreads * kVectors) {
      unpack(raw, x, most, best);
      if (p0 + kThreads * kVectors < last) fetch(p0 + kThreads * kVectors, raw);  // while this batch is worked on
      if (__any(best * kLog2e > s.m)) {
        const float m = wave_max(best) * kLog2e;
        const float dm = s.m - m, f = __builtin_amdgcn_exp2f(dm);
        s.w = f == 0.f ? 0.f * s.z : f * (s.w + dm * s.z);
        s.z *= f;
        s.m = m;
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float d = fmaf(x[i], kLog2e, -s.m), e = __builtin_amdgcn_exp2f(d);
        s.z += e;
        s.w += e * fmaxf(d, -256.f);  // 0 at -inf
      }
      if (top > 0) {
        uint32_t o = static_cast<uint32_t>(threshold >> 32);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) o = max(o, shared[w]);
        if (o > static_cast<uint32_t>(threshold >> 32)) raise(static_cast<Key>(o) << 32);
        if (__any(best >= tx)) {
          take(p0, x, most);
          if (lane == 0) shared[wave] = static_cast<uint32_t>(threshold >> 32);
        }
      }
    }
    if (top > 0) count = cut(list, out, count, top, lane);
  }

  // Appends the batch's entries before the threshold, piece by piece (one body for all: the pieces move down the registers).
  __device__ __forceinline__ void take(int p0, float (&x)[N], float (&most)[kVectors]) {
    for (int v = 0; v < kVectors; ++v) {
      if (__any(most[0] >= tx)) {
        if (count > min(2 * top, kFull)) {
          count = cut(list, out, count, top, lane);
          raise(list[top - 1]);  // there is one: the list held more
        }
        const int p = p0 + v * kThreads + lane, at = p * PER - head;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          if (!__any(x[e] >= tx)) continue;
          const Key key = key_of(x[e], at + e);
          append(list, count, (key > threshold) & inside(p, at + e), key);
        }
      }
#pragma unroll
      for (int i = 0; i + PER < N; ++i) x[i] = x[i + PER];
#pragma unroll
      for (int i = 0; i + 1 < kVectors; ++i) most[i] = most[i + 1];
    }
  }
};

// The `top` greatest entries' indexes in the order in which NaN is greatest, a pass over the row in memory for each.
template <class E>
__device__ void order_with_nan(const E* row, int vocab, int top, int64_t* ids, int lane) {
  uint64_t prev = ~0ull;
  for (int k = 0; k < top; ++k) {
    uint64_t best = 0;
    for (int i = lane; i < vocab; i += kWave) {
      const float x = Type<E>::value(as_global(row)[i]) + 0.f;
      const uint32_t b = __float_as_uint(x);
      const uint32_t key = x != x ? 0xffffffffu : (b & 0x80000000u) ? ~b : (b | 0x80000000u);
      const uint64_t c = (static_cast<uint64_t>(key) << 32) | static_cast<uint32_t>(kNoIndex - i);
      if (c < prev && c > best) best = c;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const uint64_t other = __shfl_xor(static_cast<unsigned long long>(best), o);
      best = other > best ? other : best;
    }
    if (lane == 0) ids[k] = kNoIndex - static_cast<int>(best & 0xffffffffu);
    prev = best;
  }
}

// A row whose m2 is kFar or more: the statistics again, with the difference taken first. Relative to m = 0 in the form that
// finish() takes: the greatest logit itself comes back in `greatest`. One wave a row (2048 rows of 100352 that are all such: 2.2
// ms).
template <class E>
__device__ Stats far_row(const E* row, int vocab, float& greatest, int lane) {
  float m = -INFINITY, z = 0.f, w = 0.f;
  for (int i = lane; i < vocab; i += kWave) m = fmaxf(m, Type<E>::value(as_global(row)[i]));
  m = wave_max(m);
  for (int i = lane; i < vocab; i += kWave) {
    const float d = (Type<E>::value(as_global(row)[i]) - m) * kLog2e, e = __builtin_amdgcn_exp2f(d);
    z += e;
    w += e * fmaxf(d, -256.f);
  }
  greatest = m;
  return Stats{0.f, wave_sum(z), wave_sum(w)};
}

// The results of a row from its statistics and its `count` best entries, by one wave.
template <class E>
__device__ __forceinline__ void finish(const Args& a, int64_t r, Stats s, const Key* list, int count, int lane) {
  const E* row = static_cast<const E*>(a.logits) + r * a.stride;
  float base = 0.f;
  if (!(fabsf(s.m) < kFar)) s = far_row(row, a.vocab, base, lane);
  const float lz = log2f(s.z);
  const auto logprob = [&](float x) {
    const float d = x - base;  // next to the type's lowest value the product would pass its range
    return fabsf(d) < 1e30f ? (fmaf(d, kLog2e, -s.m) - lz) * kLn2 : d - (s.m + lz) * kLn2;
  };
  const bool nan = s.z != s.z;
  if (lane == 0) {
    a.entropy[r] = (lz - s.w / s.z) * kLn2;
    if (a.targets != nullptr) {
      const int64_t t = a.targets[r];
      // a token outside the vocabulary has no probability: NaN
      a.logprob[r] = t >= 0 && t < a.vocab ? logprob(Type<E>::value(row[t])) : NAN;
    }
  }
  if (lane < a.top) {
    const Key e = lane < count ? list[lane] : 0;
    if (!nan) a.top_ids[r * a.top + lane] = index_of(e);
    a.top_logprobs[r * a.top + lane] = nan ? NAN : logprob(logit_of(e));
  }
  if (nan && a.top > 0) order_with_nan<E>(row, a.vocab, a.top, a.top_ids + r * a.top, lane);
}

// Bound by memory without alternatives (2048 rows of 100352 in bf16: 82 us, 5.0 TB/s), by the vector unit with them (20: 105 us;
// a logit costs about seven instructions, a quarter of the time goes to thresholds and lists). Four 16-byte pieces a thread in
// flight while the four before are worked on: with two and six workgroups a CU 113 us.
template <class E>
__global__ __launch_bounds__(kThreads, 4) void logprobs_kernel(Args a) {
  __shared__ __align__(16) Key lists[kWaves][kCap + kPad];
  __shared__ Key best[kMaxTop];
  __shared__ Key outs[kWaves][kMaxTop];
  __shared__ __align__(16) uint32_t lanes[kThreads];
  __shared__ Stats parts[kWaves];
  __shared__ int counts[kWaves];
  __shared__ uint32_t thresholds[kWaves + 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t r = blockIdx.x / a.parts;
  const int part = blockIdx.x % a.parts;
  const E* row = static_cast<const E*>(a.logits) + r * a.stride;
  const int head = static_cast<int>(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(E));
  const int64_t pieces = (static_cast<int64_t>(a.vocab) + head + Pass<E>::PER - 1) / Pass<E>::PER;
  const int first = static_cast<int>(min(pieces, static_cast<int64_t>(part) * a.per_part));
  const int last = static_cast<int>(min(pieces, first + static_cast<int64_t>(a.per_part)));
  if (tid < kWaves) thresholds[tid] = 0;
  Pass<E> pass;
  pass.row = row, pass.vocab = a.vocab, pass.head = head, pass.last = last, pass.top = a.top, pass.lane = lane;
  pass.list = lists[wave], pass.out = outs[wave];
  pass.run(first, lanes, thresholds, wave);
  pass.s.z = wave_sum(pass.s.z);
  pass.s.w = wave_sum(pass.s.w);
  if (lane == 0) {
    parts[wave] = pass.s;
    counts[wave] = pass.count;
  }
  __syncthreads();
  Stats s = parts[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) s = join(s, parts[w]);
  int all = 0;
  if (a.top > 0) {
    // every entry's rank among all waves' best, an entry a thread
    const int w = tid / kMaxTop % kWaves, n = tid % kMaxTop;
    const Key mine = tid < kWaves * kMaxTop && n < counts[w] ? lists[w][n] : 0;
    int rank = 0;
#pragma unroll
    for (int o = 0; o < kWaves; ++o) {
      rank += rank_in(lists[o], counts[o], mine);
      all += counts[o];
    }
    if (mine != 0 && rank < a.top) best[rank] = mine;
    __syncthreads();
  }
  if (wave != 0) return;
  const int count = min(all, a.top);
  if (a.parts > 1) {
    float* ws = a.ws + blockIdx.x * static_cast<int64_t>(kStatWords + 2 * a.top);
    if (lane == 0) {
      ws[0] = s.m;
      ws[1] = s.z;
      ws[2] = s.w;
    }
    if (lane < a.top) reinterpret_cast<Key*>(ws + kStatWords)[lane] = lane < count ? best[lane] : 0;
    return;
  }
  finish<E>(a, r, s, best, count, lane);
}

// Joins a row's parts, lane p part p. Where n parts have r entries each that reach a value, n r >= top, it is a threshold: the
// n-th greatest of the parts' r-th entries, with the least r that the number of parts allows; so is every part's last entry.
// What reaches them goes into one list that is put in order.
template <class E>
__global__ __launch_bounds__(kWave) void merge_kernel(Args a) {
  __shared__ __align__(16) Key list[kCap + kPad];
  __shared__ Key out[kMaxTop];
  const int lane = threadIdx.x;
  const int64_t r = blockIdx.x;
  const int words = kStatWords + 2 * a.top;
  const float* ws = a.ws + r * a.parts * static_cast<int64_t>(words);
  Stats s = {-kFar, 0.f, 0.f};
  const int deep = max(1, (a.top + a.parts - 1) / a.parts);
  uint32_t head = 0;
  if (lane < a.parts) {
    s = Stats{ws[lane * words], ws[lane * words + 1], ws[lane * words + 2]};
    if (a.top > 0) head = static_cast<uint32_t>(reinterpret_cast<const Key*>(ws + lane * words + kStatWords)[deep - 1] >> 32);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s = join(s, Stats{__shfl_xor(s.m, o), __shfl_xor(s.z, o), __shfl_xor(s.w, o)});
  int count = 0;
  if (a.top > 0) {
    head = (head & ~63u) | (63u - lane);
    int rank = 0;
#pragma unroll 16
    for (int l = 0; l < kWave; ++l) rank += static_cast<int>(static_cast<uint32_t>(__builtin_amdgcn_readlane(head, l)) > head);
    const int nth = __builtin_ctzll(__ballot(rank == (a.top + deep - 1) / deep - 1));
    Key threshold = static_cast<Key>(static_cast<uint32_t>(__builtin_amdgcn_readlane(head, nth)) & ~63u) << 32;
    // nor can an entry below a part's last one be among the best, if the part has as many as are asked for
    Key tail = lane < a.parts ? reinterpret_cast<const Key*>(ws + lane * words + kStatWords)[a.top - 1] : 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const Key other = __shfl_xor(tail, o);
      tail = other > tail ? other : tail;
    }
    if (tail > threshold) threshold = tail - 1;
    constexpr int kAhead = 4;  // entries of a lane loaded together
    for (int i0 = 0; i0 < a.parts * a.top; i0 += kAhead * kWave) {
      Key e[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int i = i0 + u * kWave + lane, p = i / a.top, k = i - p * a.top;
        e[u] = p < a.parts ? reinterpret_cast<const Key*>(ws + p * words + kStatWords)[k] : 0;
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        append(list, count, e[u] > threshold, e[u]);
        if (count > kFull) {
          count = cut(list, out, count, a.top, lane);
          threshold = list[a.top - 1];
        }
      }
    }
    count = cut(list, out, count, a.top, lane);
  }
  finish<E>(a, r, s, list, count, lane);
}

constexpr int kTarget = 1024;    // workgroups that splitting rows aims at
constexpr int kLeastPart = 1024;  // least pieces of a part: a batch of every thread (with a quarter of it 126 rows of 23908 took 25 us, so 17)

int parts_of(int64_t rows, int64_t vocab, int per) {
  const int64_t pieces = (vocab + per - 1) / per + 1;  // + 1: a row that begins inside a piece
  int64_t parts = kTarget / rows;  // no more than the card holds at once
  const int64_t most = (pieces + kLeastPart - 1) / kLeastPart;
  parts = parts < most ? parts : most;
  return static_cast<int>(parts < 1 ? 1 : parts < kMaxParts ? parts : kMaxParts);
}

int element_bytes(int dtype) { return dtype == BP_DT_F32 ? 4 : 2; }

template <class E>
int launch(const Args& a, int64_t rows, hipStream_t st) {
  logprobs_kernel<E><<<static_cast<unsigned>(rows * a.parts), kThreads, 0, st>>>(a);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && a.parts > 1) {
    merge_kernel<E><<<static_cast<unsigned>(rows), kWave, 0, st>>>(a);
    e = hipGetLastError();
  }
  return e == hipSuccess ? BP_OK : static_cast<int>(e);
}

}  // namespace
}  // namespace logprobs
}  // namespace bp

extern "C" {

size_t bp_logprobs_workspace_bytes(int dtype, int64_t rows, int64_t vocab, int top) {
  if (rows <= 0 || vocab <= 0 || top < 0 || top > bp::logprobs::kMaxTop) return 0;
  const int parts = bp::logprobs::parts_of(rows, vocab, 16 / bp::logprobs::element_bytes(dtype));
  return parts > 1 ? static_cast<size_t>(rows) * parts * (bp::logprobs::kStatWords + 2 * top) * sizeof(float) : 0;
}

int bp_logprobs(int dtype, const void* logits, int64_t row_stride, const int64_t* targets, float* logprob, float* entropy,
                int64_t* top_ids, float* top_logprobs, int64_t rows, int64_t vocab, int top, void* workspace,
                size_t workspace_bytes, void* stream) {
  if (dtype != BP_DT_BF16 && dtype != BP_DT_F16 && dtype != BP_DT_F32) return BP_E_UNSUPPORTED;
  if (rows < 0 || vocab < 0 || top < 0 || row_stride < 0) return BP_E_INVALID_ARG;
  if (top > bp::logprobs::kMaxTop || vocab >= (1ll << 30) || rows >= (1ll << 24)) return BP_E_UNSUPPORTED;
  if (rows == 0) return BP_OK;
  if (vocab == 0 || top > vocab || logits == nullptr || entropy == nullptr || (targets != nullptr && logprob == nullptr) ||
      (top > 0 && (top_ids == nullptr || top_logprobs == nullptr)) ||
      reinterpret_cast<uintptr_t>(logits) % bp::logprobs::element_bytes(dtype) != 0)
    return BP_E_INVALID_ARG;
  const size_t need = bp_logprobs_workspace_bytes(dtype, rows, vocab, top);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 8 != 0)) return BP_E_WORKSPACE;
  bp::logprobs::Args a = {};
  a.logits = logits, a.targets = targets, a.logprob = logprob, a.entropy = entropy, a.top_ids = top_ids;
  a.top_logprobs = top_logprobs, a.ws = static_cast<float*>(workspace), a.stride = row_stride;
  a.vocab = static_cast<int>(vocab), a.top = top;
  const int per = 16 / bp::logprobs::element_bytes(dtype);
  a.parts = bp::logprobs::parts_of(rows, vocab, per);
  const int64_t pieces = (vocab + per - 1) / per + 1;
  a.per_part = static_cast<int>((pieces + a.parts - 1) / a.parts);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == BP_DT_BF16) return bp::logprobs::launch<uint16_t>(a, rows, st);
  if (dtype == BP_DT_F16) return bp::logprobs::launch<_Float16>(a, rows, st);
  return bp::logprobs::launch<float>(a, rows, st);
}

}  // extern "C"
