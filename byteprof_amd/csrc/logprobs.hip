// Log probabilities of given tokens, the entropy and the most likely tokens of rows of logits, in one pass over the logits.
//
//   m = max x, z = sum exp(x - m), w = sum exp(x - m) (x - m):  log p(t) = x_t - m - ln z,  H = ln z - w / z
//
// A wave keeps one running maximum (all lanes the same) and its lanes' own z and w relative to it; a batch of logits that
// holds a greater one rescales them: z' = f z, w' = f (w + dm z) with f = exp(dm), dm = m - m'. The
// most likely tokens: a wave appends the batch's logits above its threshold to a list in LDS; a full list is cut to its best
// `top`, whose last is the new threshold. Order: greater logit first, then lower index.
// Held in fp32: logits as they are, exponentials, sums. A NaN or +inf among the logits makes z NaN, and with it every log
// probability of the row (as log softmax does); the order of such a row comes from a second pass that counts NaN as greatest.

#include "byteprof_amd.h"
#include "common.h"

namespace bp {
namespace logprobs {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kMaxTop = 32;
constexpr int kCap = 256;      // entries of a wave's list
constexpr int kVectors = 4;    // 16-byte loads of a lane in flight
constexpr int kMaxParts = 64;  // workgroups of a row: one lane each in the merge
constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kNoIndex = 0x7fffffff;

struct Args {
  const void* logits;
  const int64_t* targets;  // or null
  float* logprob;          // with targets
  float* entropy;
  int64_t* top_ids;
  float* top_logprobs;
  float* ws;  // [rows][parts][3 + 2 top]: m, z, w, values, indices
  int64_t stride;  // elements
  int vocab, top, parts, per_part;  // per_part: 16-byte pieces of a part
};

struct Entry {
  float x;
  int i;
};

// a before b: greater, or equal and of lower index.
__device__ __forceinline__ bool before(float ax, int ai, float bx, int bi) { return ax > bx || (ax == bx && ai < bi); }

template <class E>
struct Type;
template <>
struct Type<uint16_t> {  // bf16
  static __device__ __forceinline__ float value(uint16_t v) { return bf16_bits_to_float(v); }
};
template <>
struct Type<_Float16> {
  static __device__ __forceinline__ float value(_Float16 v) { return static_cast<float>(v); }
};
template <>
struct Type<float> {
  static __device__ __forceinline__ float value(float v) { return v; }
};

__device__ __forceinline__ float wave_max(float v) { return xor_butterfly<true>(v, MaxOp()); }
__device__ __forceinline__ float wave_sum(float v) { return xor_butterfly<true>(v, AddOp()); }

// The best `keep` of the `count` entries of a wave's list to its front, in order (by every entry's number of entries before
// it). Returns how many that are.
__device__ int cut(Entry* list, int count, int keep, int lane) {
  constexpr int PER = kCap / kWave;
  Entry mine[PER];
  int rank[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int at = j * kWave + lane;
    mine[j] = at < count ? list[at] : Entry{-INFINITY, kNoIndex};
    rank[j] = at < count ? 0 : kCap;
  }
  for (int n = 0; n < count; ++n) {
    const Entry e = list[n];
#pragma unroll
    for (int j = 0; j < PER; ++j) rank[j] += before(e.x, e.i, mine[j].x, mine[j].i) ? 1 : 0;
  }
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int j = 0; j < PER; ++j)
    if (rank[j] < keep) list[rank[j]] = mine[j];
  __builtin_amdgcn_wave_barrier();
  return min(count, keep);
}

struct Stats {
  float m, z, w;
};

// The difference is taken before the product: logits of the type's lowest value times log2(e) would pass its range.
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

__device__ __forceinline__ Stats join(const Stats& a, const Stats& b) {
  Stats r;
  r.m = fmaxf(a.m, b.m);
  const float base = r.m == -INFINITY ? 0.f : r.m;
  const auto part = [&](const Stats& s, float& z, float& w) {
    const float dm = s.m == r.m ? 0.f : s.m - base;  // s.m = -inf: nothing in it, z = w = 0
    const float f = s.m == r.m ? 1.f : exp_of(dm);
    z += f * s.z;
    w += f == 0.f ? 0.f * s.z : f * (s.w + dm * s.z);
  };
  r.z = r.w = 0.f;
  part(a, r.z, r.w);
  part(b, r.z, r.w);
  return r;
}

// The wave's part of a row: pieces of 16 bytes from `first` to `last`, every kWaves x 64th.
template <class E>
struct Pass {
  static constexpr int PER = 16 / sizeof(E);
  static constexpr int N = kVectors * PER;
  Stats s;
  float tx;  // threshold: entries before (tx, ti) are taken
  int ti, count;

  __device__ __forceinline__ void run(const E* row, int vocab, int head, int first, int last, int top, Entry* list, int wave,
                                      int lane) {
    s = Stats{-INFINITY, 0.f, 0.f};
    tx = -INFINITY;
    ti = kNoIndex;
    count = 0;
    for (int p0 = first + wave * kWave * kVectors; p0 < last; p0 += kThreads * kVectors) {
      float x[N];
      uint32_t raw[kVectors][4];
#pragma unroll
      for (int v = 0; v < kVectors; ++v) {
        // piece p: elements p PER - head ...; the first and the last may reach over the row's ends
        const int p = p0 + v * kWave + lane, at = p * PER - head;
        if (p < last && at >= 0 && at + PER <= vocab) {
          const u32x4 r = *as_global(reinterpret_cast<const u32x4*>(row + at));
#pragma unroll
          for (int j = 0; j < 4; ++j) raw[v][j] = r[j];
        } else {
          E part[PER];
#pragma unroll
          for (int e = 0; e < PER; ++e) {
            const bool in = p < last && at + e >= 0 && at + e < vocab;
            part[e] = in ? as_global(row)[at + e] : lowest();
          }
          __builtin_memcpy(raw[v], part, 16);
        }
      }
      float best = -INFINITY;
#pragma unroll
      for (int v = 0; v < kVectors; ++v) {
        E part[PER];
        __builtin_memcpy(part, raw[v], 16);
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          x[v * PER + e] = Type<E>::value(part[e]);
          best = fmaxf(best, x[v * PER + e]);
        }
      }
      if (__any(best > s.m)) {
        const float m = wave_max(best);
        if (s.m != -INFINITY) {
          const float dm = s.m - m, f = exp_of(dm);
          s.w = f == 0.f ? 0.f * s.z : f * (s.w + dm * s.z);
          s.z *= f;
        }
        s.m = m;
      }
      const float base = s.m == -INFINITY ? 0.f : s.m;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float d = x[i] - base, e = exp_of(d);
        s.z += e;
        s.w += e * fmaxf(d, -256.f);  // 0 at -inf
      }
      if (top > 0 && __any(best >= tx)) take(x, best, vocab, head, p0, last, top, list, lane);
    }
    if (top > 0) count = cut(list, count, top, lane);
  }

  static __device__ __forceinline__ E lowest() {
    if constexpr (sizeof(E) == 4) return -INFINITY;
    else if constexpr (__is_same(E, _Float16)) return static_cast<_Float16>(-INFINITY);
    else return static_cast<E>(0xff80);
  }

  // Appends the batch's entries before the threshold. Where `top` lanes or more have one, the threshold first rises to the
  // `top`-th greatest of the lanes' best: that many entries reach it.
  __device__ void take(const float (&x)[N], float best, int vocab, int head, int p0, int last, int top, Entry* list, int lane) {
    if (__popcll(__ballot(best >= tx)) >= top) {
      int rank = 0;
      for (int l = 0; l < kWave; ++l) {
        const float o = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(best), l));
        rank += o > best || (o == best && l < lane) ? 1 : 0;
      }
      const float at = __int_as_float(
          __builtin_amdgcn_readlane(__float_as_int(best), __builtin_ctzll(__ballot(rank == top - 1))));
      if (at > tx) {
        tx = at;
        ti = kNoIndex;
      }
    }
#pragma unroll
    for (int v = 0; v < kVectors; ++v) {
      const int p = p0 + v * kWave + lane, at = p * PER - head;
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const bool in = p < last && at + e >= 0 && at + e < vocab;
        const float xe = x[v * PER + e];
        const uint64_t mask = __ballot(in && before(xe, at + e, tx, ti));
        if (mask == 0) continue;
        if (in && before(xe, at + e, tx, ti))
          list[count + __builtin_amdgcn_mbcnt_hi(static_cast<unsigned>(mask >> 32),
                                                 __builtin_amdgcn_mbcnt_lo(static_cast<unsigned>(mask), 0))] = Entry{xe, at + e};
        count += __popcll(mask);
        __builtin_amdgcn_wave_barrier();
        if (count > kCap - kWave) {
          count = cut(list, count, top, lane);
          tx = list[top - 1].x;  // count >= top: the list was nearly full
          ti = list[top - 1].i;
        }
      }
    }
  }
};

// Greatest entry of the wave that comes after (px, pi) in the order in which NaN is greatest, over a row in memory.
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

template <class E>
__device__ __forceinline__ void finish(const Args& a, int64_t r, const Stats& s, int lane) {
  const E* row = static_cast<const E*>(a.logits) + r * a.stride;
  const float lz = logf(s.z);
  if (lane == 0) {
    a.entropy[r] = lz - s.w / s.z;
    if (a.targets != nullptr) {
      const int64_t t = a.targets[r];
      // a token outside the vocabulary has no probability: NaN
      a.logprob[r] = t >= 0 && t < a.vocab ? Type<E>::value(row[t]) - s.m - lz : NAN;
    }
  }
}

template <class E>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(Args a) {
  __shared__ Entry lists[kWaves][kCap];
  __shared__ Stats parts[kWaves];
  __shared__ int counts[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t r = blockIdx.x / a.parts;
  const int part = blockIdx.x % a.parts;
  const E* row = static_cast<const E*>(a.logits) + r * a.stride;
  const int head = static_cast<int>(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(E));
  const int64_t pieces = (static_cast<int64_t>(a.vocab) + head + Pass<E>::PER - 1) / Pass<E>::PER;
  const int first = static_cast<int>(min(pieces, static_cast<int64_t>(part) * a.per_part));
  const int last = static_cast<int>(min(pieces, first + static_cast<int64_t>(a.per_part)));
  Pass<E> pass;
  pass.run(row, a.vocab, head, first, last, a.top, lists[wave], wave, lane);
  pass.s.z = wave_sum(pass.s.z);
  pass.s.w = wave_sum(pass.s.w);
  if (lane == 0) {
    parts[wave] = pass.s;
    counts[wave] = pass.count;
  }
  __syncthreads();
  if (wave != 0) return;
  Stats s = parts[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) s = join(s, parts[w]);
  int count = counts[0];
  for (int w = 1; w < kWaves; ++w) {  // the other waves' entries behind the first's
    if (lane < counts[w]) lists[0][count + lane] = lists[w][lane];
    count += counts[w];
  }
  __builtin_amdgcn_wave_barrier();
  if (a.top > 0) count = cut(lists[0], count, a.top, lane);
  if (a.parts > 1) {
    float* ws = a.ws + blockIdx.x * static_cast<int64_t>(3 + 2 * a.top);
    if (lane == 0) {
      ws[0] = s.m;
      ws[1] = s.z;
      ws[2] = s.w;
    }
    if (lane < a.top) {
      const Entry e = lane < count ? lists[0][lane] : Entry{-INFINITY, kNoIndex};
      ws[3 + lane] = e.x;
      ws[3 + a.top + lane] = __int_as_float(e.i);
    }
    return;
  }
  finish<E>(a, r, s, lane);
  const bool nan = s.z != s.z;
  if (lane < a.top) {
    if (!nan) a.top_ids[r * a.top + lane] = lists[0][lane].i;
    a.top_logprobs[r * a.top + lane] = nan ? NAN : lists[0][lane].x - s.m - logf(s.z);
  }
  if (nan && a.top > 0) order_with_nan<E>(row, a.vocab, a.top, a.top_ids + r * a.top, lane);
}

// Joins a row's parts: lane p holds part p; the greatest of the parts' next entries, `top` times.
template <class E>
__global__ __launch_bounds__(kWave) void merge_kernel(Args a) {
  __shared__ Entry lists[kMaxParts][kMaxTop + 1];
  const int lane = threadIdx.x;
  const int64_t r = blockIdx.x;
  const int words = 3 + 2 * a.top;
  const float* ws = a.ws + r * a.parts * static_cast<int64_t>(words);
  Stats s = {-INFINITY, 0.f, 0.f};
  if (lane < a.parts) s = Stats{ws[lane * words], ws[lane * words + 1], ws[lane * words + 2]};
  for (int i = lane; i < a.parts * a.top; i += kWave) {
    const int p = i / a.top, k = i % a.top;
    lists[p][k] = Entry{ws[p * words + 3 + k], __float_as_int(ws[p * words + 3 + a.top + k])};
  }
  lists[lane][a.top] = Entry{-INFINITY, kNoIndex};
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s = join(s, Stats{__shfl_xor(s.m, o), __shfl_xor(s.z, o), __shfl_xor(s.w, o)});
  finish<E>(a, r, s, lane);
  if (s.z != s.z) {
    if (lane < a.top) a.top_logprobs[r * a.top + lane] = NAN;
    if (a.top > 0)
      order_with_nan<E>(static_cast<const E*>(a.logits) + r * a.stride, a.vocab, a.top, a.top_ids + r * a.top, lane);
    return;
  }
  const float lz = logf(s.z);
  int at = 0;
  Entry mine = lane < a.parts ? lists[lane][0] : Entry{-INFINITY, kNoIndex};
  for (int k = 0; k < a.top; ++k) {
    float x = mine.x;
    int i = mine.i;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const float ox = __shfl_xor(x, o);
      const int oi = __shfl_xor(i, o);
      if (before(ox, oi, x, i)) x = ox, i = oi;
    }
    if (lane == 0) {
      a.top_ids[r * a.top + k] = i;
      a.top_logprobs[r * a.top + k] = x - s.m - lz;
    }
    if (mine.i == i && at < a.top) mine = lists[lane][++at];
  }
}

constexpr int kTarget = 1024;    // workgroups that splitting rows aims at
constexpr int kLeastPart = 256;  // least pieces of a part: one a thread

int parts_of(int64_t rows, int64_t vocab, int per) {
  const int64_t pieces = (vocab + per - 1) / per + 1;  // + 1: a row that begins inside a piece
  int64_t parts = (kTarget + rows - 1) / rows;
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
  return parts > 1 ? static_cast<size_t>(rows) * parts * (3 + 2 * top) * sizeof(float) : 0;
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
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return BP_E_WORKSPACE;
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
