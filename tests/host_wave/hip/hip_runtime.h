// Stands in for HIP's header where device code that reads tables is compiled for the host: the
// threads of one work-group are fibers that run in turn from one exchange (ballot, shuffle,
// barrier) to the next, so a wrong index is an assertion of the test instead of a fault.
#pragma once
#include <ucontext.h>

#include <cassert>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <functional>
#include <memory>
#include <vector>

#define __device__
#define __host__
#define __global__
#define __forceinline__ inline
#define __shared__ static

struct float2 {
  float x, y;
};
struct dim3 {
  unsigned x = 1, y = 1, z = 1;
};
static dim3 threadIdx, blockIdx;

using std::max;
using std::min;

namespace host_wave {
constexpr int kMost = 512, kStack = 1 << 16;
struct Thread {
  ucontext_t at;
  bool done;
  int exchanges;
};
static Thread threads[kMost];
static ucontext_t caller;
static int current, count;
static uint64_t slots[2][kMost];  // of this exchange and the next: a thread may be one ahead
static std::function<void()> body;

static void begin() {
  body();
  threads[current].done = true;
}
// what every thread gives, when all have given it
static const uint64_t* exchange(uint64_t x) {
  Thread& t = threads[current];
  uint64_t* bank = slots[t.exchanges++ & 1];
  bank[current] = x;
  swapcontext(&t.at, &caller);
  return bank;
}
static void run(int n, std::function<void()> f) {
  static std::unique_ptr<char[]> stacks(new char[kMost * kStack]);
  assert(n <= kMost);
  body = f;
  count = n;
  for (int i = 0; i < n; ++i) {
    getcontext(&threads[i].at);
    threads[i].at.uc_stack.ss_sp = &stacks[i * kStack];
    threads[i].at.uc_stack.ss_size = kStack;
    threads[i].at.uc_link = &caller;
    threads[i].done = false;
    threads[i].exchanges = 0;
    makecontext(&threads[i].at, begin, 0);
  }
  for (bool more = true; more;) {
    more = false;
    for (current = 0; current < n; ++current) {
      if (threads[current].done) continue;
      threadIdx.x = current;
      swapcontext(&caller, &threads[current].at);
      more = more || !threads[current].done;
    }
  }
}
template <class T>
inline uint64_t bits(T x) {
  uint64_t y = 0;
  memcpy(&y, &x, sizeof x);
  return y;
}
template <class T>
inline T value(uint64_t y) {
  T x;
  memcpy(&x, &y, sizeof x);
  return x;
}
}  // namespace host_wave

inline uint64_t __ballot(bool x) {
  const uint64_t* all = host_wave::exchange(x);
  const int wave = threadIdx.x & ~63u;
  uint64_t y = 0;
  for (int i = 0; i < 64 && wave + i < host_wave::count; ++i) y |= all[wave + i] << i;
  return y;
}
inline int __popcll(uint64_t x) { return __builtin_popcountll(x); }
inline void __syncthreads() { host_wave::exchange(0); }
template <class T>
inline T __shfl_up(T x, int by, int) {
  const uint64_t* all = host_wave::exchange(host_wave::bits(x));
  const int lane = threadIdx.x & 63;
  return host_wave::value<T>(all[threadIdx.x - (lane >= by ? by : 0)]);
}
template <class T>
inline T __shfl_xor(T x, int with, int) {
  return host_wave::value<T>(host_wave::exchange(host_wave::bits(x))[threadIdx.x ^ with]);
}
inline int read_lane(int x, int lane) {
  return host_wave::value<int>(host_wave::exchange(host_wave::bits(x))[(threadIdx.x & ~63u) + lane]);
}
inline unsigned __umulhi(unsigned a, unsigned b) { return static_cast<uint64_t>(a) * b >> 32; }
inline float __int_as_float(int x) { return host_wave::value<float>(host_wave::bits(x)); }
inline int __float_as_int(float x) { return host_wave::value<int>(host_wave::bits(x)); }

// values that the code says are uniform; and what other headers name and these tests never call
#define __builtin_amdgcn_readfirstlane(x) (x)
#define __builtin_amdgcn_readlane(x, lane) read_lane(x, lane)
#define __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, x, y, z) (c)
#define __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, x, y, z) (c)
#define __builtin_amdgcn_mov_dpp(x, c, r, b, z) (x)
#define __builtin_amdgcn_rcpf(x) (1.0f / (x))
#define __builtin_amdgcn_exp2f(x) exp2f(x)
typedef void* hipStream_t;
