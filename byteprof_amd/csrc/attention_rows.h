// What a tile of the attention kernels reads and writes besides its keys and values: the queries' rows, the result, the partial sums
// of divided tiles, and the rows that belong to no sequence.
#pragma once

#include "attention.h"

namespace bp {
namespace attn {

// Rows that belong to no sequence: zeros, dealt to the workgroups past the last tile.
__device__ __forceinline__ void fill_rest(const Args& a, int kvh, int extra, int extras) {
  const int lo = a.seqs > 0 ? min(max(a.cu[0], 0), a.tokens) : a.tokens;
  int hi = a.seqs > 0 ? min(max(a.cu[a.seqs], lo), a.tokens) : a.tokens;
  const int64_t rest = lo + (a.tokens - hi), per = static_cast<int64_t>(a.group.d) * a.d / 8;
  for (int64_t i = static_cast<int64_t>(extra) * kThreads + threadIdx.x; i < rest * per;
       i += static_cast<int64_t>(extras) * kThreads) {
    const int64_t n = i / per, c = i % per;
    const int64_t tok = n < lo ? n : hi + (n - lo);
    uint16_t* at = static_cast<uint16_t*>(a.out) + (tok * a.hq + static_cast<int64_t>(kvh) * a.group.d) * a.d + 8 * c;
    *reinterpret_cast<u32x4*>(at) = u32x4{};
  }
}

__device__ __forceinline__ uint16_t* out_row(const Args& a, const Item& it, int kvh, int row) {
  const int n = a.group(row);
  const int64_t head = static_cast<int64_t>(it.begin + n) * a.hq + kvh * a.group.d + (row - n * a.group.d);
  return static_cast<uint16_t*>(a.out) + head * a.d;
}

// A split's slot: [ws_rows][DP] sums, then ws_rows maxima and ws_rows sums of probabilities.
template <int DP>
__device__ __forceinline__ float* slot_at(const Args& a, int64_t slot, int kvh) {
  return a.ws + (slot * a.hk.d + kvh) * a.ws_rows * (DP + 2);
}

template <class T, int DP, bool FULL>
__device__ __forceinline__ void load_q(const Args& a, const Item& it, int kvh, int row, u32x4 (&q)[DP / 16], int lane) {
  const int n = a.group(row);
  const uint16_t* p = static_cast<const uint16_t*>(a.q) + static_cast<int64_t>(it.begin + n) * a.q_t +
                      static_cast<int64_t>(kvh * a.group.d + row - n * a.group.d) * a.q_h;
#pragma unroll
  for (int i = 0; i < DP / 16; ++i) {
    const int c = 2 * i + (lane >> 5);
    q[i] = FULL || 8 * c < a.d ? *reinterpret_cast<const u32x4*>(p + 8 * c) : u32x4{};
  }
}

__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }

// The result of a large tile's row (lane's row `row`, of which rows past the tile's are not written), or the row's partial sums.
template <class T, int DP>
__device__ __forceinline__ void write_rows(const Args& a, const Item& it, int kvh, int row, const Running<DP>& r, int lane) {
  const int top = it.row0 + it.rows - 1, mine = min(row, top);
  const float l = add_halves(r.l);
  if (!it.divided) {
    const float inv = inverse(l);
    uint16_t* out = out_row(a, it, kvh, mine);
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // columns 16 i + 4 half + 0..3 and 8 further, as 8 columns a lane: the halves exchange a group of 4
        u32x2 x, y;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          x[e] = T::result(r.o[db][8 * i + 2 * e] * inv, r.o[db][8 * i + 2 * e + 1] * inv);
          y[e] = T::result(r.o[db][8 * i + 4 + 2 * e] * inv, r.o[db][8 * i + 4 + 2 * e + 1] * inv);
        }
        const auto w0 = __builtin_amdgcn_permlane32_swap(x[0], y[0], false, false);
        const auto w1 = __builtin_amdgcn_permlane32_swap(x[1], y[1], false, false);
        const int col = 32 * db + 16 * i + 8 * (lane >> 5);
        if (row <= top && col < a.d) *reinterpret_cast<u32x4*>(out + col) = u32x4{w0[0], w1[0], w0[1], w1[1]};
      }
    return;
  }
  float* ws = slot_at<DP>(a, it.slot + it.split, kvh);
  const int at = row - it.row0;
  if (row > top || it.slot + it.split >= a.slots) return;
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<f32x4*>(ws + at * DP + 32 * db + 8 * i + 4 * (lane >> 5)) =
          f32x4{r.o[db][4 * i], r.o[db][4 * i + 1], r.o[db][4 * i + 2], r.o[db][4 * i + 3]};
  if (lane < 32) {
    ws[a.ws_rows * DP + at] = r.m;
    ws[a.ws_rows * (DP + 1) + at] = l;
  }
}

// Joins the four waves' parts of a small tile (every wave has all rows) into the result or the tile's partial sums. G: 32-column
// blocks of a round through smem.
template <class T, int DP, int G>
__device__ __forceinline__ void join_waves(const Args& a, const Item& it, int kvh, Running<DP>& r, u32x4* smem, float* stats) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  r.l = add_halves(r.l);
  // stats: [wave][32] maxima, [wave][32] sums, [32] factors of the result
  if (lane < 32) {
    stats[32 * wave + lane] = r.m;
    stats[32 * (kWaves + wave) + lane] = r.l;
  }
  __syncthreads();
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) m = fmaxf(m, stats[32 * w + (lane & 31)]);
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float mw = stats[32 * w + (lane & 31)];
    l += stats[32 * (kWaves + w) + (lane & 31)] * rescaled(mw, m, a.scale_log2);
  }
  const float f = rescaled(r.m, m, a.scale_log2);
  const bool whole = !it.divided;
  float* ws = whole ? nullptr : slot_at<DP>(a, it.slot + it.split, kvh);
  const bool keep = whole || it.slot + it.split < a.slots;
  if (wave == 0 && lane < 32) {
    stats[32 * 2 * kWaves + lane] = whole ? inverse(l) : 1.f;
    if (!whole && keep && lane < it.rows) {
      ws[a.ws_rows * DP + lane] = m;
      ws[a.ws_rows * (DP + 1) + lane] = l;
    }
  }
  f32x4* parts = reinterpret_cast<f32x4*>(smem);
#pragma unroll
  for (int g = 0; g < DP / 32 / G; ++g) {
    if ((lane & 31) < it.rows) {
#pragma unroll
      for (int db = 0; db < G; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x16& o = r.o[g * G + db];
          parts[(wave * G * 8 + db * 8 + 2 * i + (lane >> 5)) * 32 + (lane & 31)] =
              f32x4{o[4 * i] * f, o[4 * i + 1] * f, o[4 * i + 2] * f, o[4 * i + 3] * f};
        }
    }
    __syncthreads();
    for (int i = tid; i < it.rows * G * 8; i += kThreads) {
      const int row = i / (G * 8), piece = i % (G * 8), col = 4 * piece + 32 * G * g;
      f32x4 x = parts[piece * 32 + row];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) x += parts[(w * G * 8 + piece) * 32 + row];
      if (whole) {
        const float inv = stats[32 * 2 * kWaves + row];
        if (col < a.d)
          *reinterpret_cast<u32x2*>(out_row(a, it, kvh, it.row0 + row) + col) =
              u32x2{T::result(x[0] * inv, x[1] * inv), T::result(x[2] * inv, x[3] * inv)};
      } else if (keep) {
        *reinterpret_cast<f32x4*>(ws + row * DP + col) = x;
      }
    }
    if (g + 1 < DP / 32 / G) __syncthreads();
  }
}

// Joins the partial sums of divided tiles (n.merges > 0). dtype: BP_DT_BF16 or BP_DT_F16.
template <class P>
int launch_merge(int dtype, const Args& a, const Launch& n, hipStream_t st);

}  // namespace attn
}  // namespace bp
