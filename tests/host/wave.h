// A wave of 64 lanes on the CPU, for device code whose control flow is the same in all lanes: a fiber per lane, and every
// operation between lanes hands on to the next lane until all have given their value.
#pragma once

#include <setjmp.h>
#include <stdint.h>
#include <string.h>
#include <ucontext.h>

#include <algorithm>
#include <functional>
#include <vector>

#define __device__
#define __host__
#define __forceinline__ inline

using std::max;
using std::min;

namespace wave {

constexpr int kLanes = 64;
constexpr size_t kStack = 64 * 1024;

struct Fiber {
  jmp_buf at;
  ucontext_t start;
  std::vector<char> stack;
  int phase;
  bool started, done;
};

inline Fiber fibers[kLanes];
inline jmp_buf outside;
inline ucontext_t home;
inline int current;
inline uint32_t values[2][kLanes];
inline std::function<void(int)> body;

// To the next lane that still runs, or out.
inline void hand_on() {
  for (int i = 1; i <= kLanes; ++i) {
    const int next = (current + i) % kLanes;
    Fiber& f = fibers[next];
    if (f.done) continue;
    if (next == current) return;
    current = next;
    if (f.started) _longjmp(f.at, 1);
    f.started = true;
    setcontext(&f.start);
  }
  _longjmp(outside, 1);
}

inline void enter() {
  body(current);
  fibers[current].done = true;
  hand_on();
}

inline const uint32_t* gather(uint32_t v) {
  Fiber& f = fibers[current];
  const int phase = f.phase;
  f.phase ^= 1;
  values[phase][current] = v;
  if (_setjmp(f.at) == 0) hand_on();
  return values[phase];
}

inline void run(const std::function<void(int)>& fn) {
  body = fn;
  for (Fiber& f : fibers) {
    f.stack.resize(kStack);
    f.phase = 0;
    f.started = f.done = false;
    getcontext(&f.start);
    f.start.uc_stack.ss_sp = f.stack.data();
    f.start.uc_stack.ss_size = kStack;
    f.start.uc_link = nullptr;
    makecontext(&f.start, enter, 0);
  }
  current = 0;
  fibers[0].started = true;
  if (_setjmp(outside) == 0) setcontext(&fibers[0].start);
}

}  // namespace wave

struct ThreadIdx {
  struct X {
    operator int() const { return wave::current; }
  } x;
};
inline ThreadIdx threadIdx;

inline float __int_as_float(int v) {
  float f;
  memcpy(&f, &v, 4);
  return f;
}
inline int __float_as_int(float f) {
  int v;
  memcpy(&v, &f, 4);
  return v;
}
inline uint32_t __umulhi(uint32_t a, uint32_t b) { return static_cast<uint64_t>(a) * b >> 32; }

inline int wave_readlane(int v, int lane) { return static_cast<int>(wave::gather(static_cast<uint32_t>(v))[lane]); }
inline uint64_t __ballot(bool v) {
  const uint32_t* all = wave::gather(v);
  uint64_t mask = 0;
  for (int i = 0; i < wave::kLanes; ++i) mask |= static_cast<uint64_t>(all[i] != 0) << i;
  return mask;
}
// row_shr:1..8 within rows of 16 and the broadcasts of a row's last lane into the rows behind it; a lane without a source keeps
// `old`, as does a row outside the mask.
inline int wave_update_dpp(int old, int v, int ctrl, int row_mask, int bank_mask, bool) {
  const uint32_t* all = wave::gather(static_cast<uint32_t>(v));
  const int lane = wave::current, row = lane / 16;
  int from = -1;
  if (ctrl > 0x110 && ctrl < 0x120) from = lane % 16 >= ctrl - 0x110 ? lane - (ctrl - 0x110) : -1;
  else if (ctrl == 0x142) from = row > 0 ? 16 * row - 1 : -1;
  else if (ctrl == 0x143) from = row > 1 ? 31 : -1;
  else __builtin_trap();
  if (!(row_mask >> row & 1) || bank_mask != 0xF || from < 0) return old;
  return static_cast<int>(all[from]);
}
#define __builtin_amdgcn_readlane wave_readlane
#define __builtin_amdgcn_readfirstlane(v) wave_readlane(v, 0)
#define __builtin_amdgcn_update_dpp wave_update_dpp

// What a plan takes of common.h.
namespace bp {
constexpr int kWave = wave::kLanes;
struct AddOp {
  float operator()(float a, float b) const { return a + b; }
};
template <bool DOWN, class Op>
float xor_butterfly(float v, Op op) {
  static_assert(DOWN, "the order 32, 16, ..., 1");
  for (int d = 32; d > 0; d >>= 1) {
    const uint32_t* all = wave::gather(static_cast<uint32_t>(__float_as_int(v)));
    v = op(v, __int_as_float(static_cast<int>(all[wave::current ^ d])));
  }
  return v;
}
}  // namespace bp
