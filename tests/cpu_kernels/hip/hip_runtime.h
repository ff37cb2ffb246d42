// A HIP kernel on the CPU, for tests: a workgroup's threads are coroutines of one host thread, which switch at
// barriers and lane exchanges only.  What dpft_norm.hip uses, no more.
#pragma once
#include <ucontext.h>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <vector>

#define __global__
#define __device__
#define __forceinline__ inline
#define __launch_bounds__(...)
#define __shared__ static
#define __restrict__

struct dim3 {
  unsigned x;
  dim3(unsigned n = 1) : x(n) {}
};
typedef void* hipStream_t;
struct float2 {
  float x, y;
};
struct float4 {
  float x, y, z, w;
};
inline float2 make_float2(float a, float b) { return {a, b}; }
inline float4 make_float4(float a, float b, float c, float d) { return {a, b, c, d}; }

namespace cpu {
struct Thread {
  ucontext_t context;
  std::vector<uint64_t> sent;  // lane exchanges since the last barrier
  bool done;
};
extern std::vector<Thread> threads;
extern ucontext_t scheduler;
extern int current, alive, arrived, generation;
void fail(const char* why);
void run(unsigned grid, int threads, std::function<void()> kernel);
inline void yield() { swapcontext(&threads[current].context, &scheduler); }
// Sends v to the workgroup and takes what `partner` sends as its exchange of the same number.
inline uint64_t exchange(uint64_t v, int partner) {
  const size_t number = threads[current].sent.size();
  threads[current].sent.push_back(v);
  while (threads[partner].sent.size() <= number) {
    if (threads[partner].done) fail("exchange with a lane that has ended");
    yield();
  }
  return threads[partner].sent[number];
}
struct Index {
  unsigned x;
};
}  // namespace cpu
extern cpu::Index blockIdx, gridDim;
struct ThreadIndex {
  struct {
    operator unsigned() const { return (unsigned)cpu::current; }
  } x;
};
extern ThreadIndex threadIdx;

inline void __syncthreads() {
  const int before = cpu::generation;
  if (++cpu::arrived == cpu::alive) {
    cpu::arrived = 0;
    ++cpu::generation;
    for (auto& t : cpu::threads) t.sent.clear();
  }
  while (cpu::generation == before) cpu::yield();
}
template <typename T>
T __shfl_xor(T v, int o) {
  uint64_t bits = 0;
  memcpy(&bits, &v, sizeof v);
  bits = cpu::exchange(bits, cpu::current ^ o);
  memcpy(&v, &bits, sizeof v);
  return v;
}
inline int cpu_dpp(int v, int control) {  // quad_perm [1,0,3,2], quad_perm [2,3,0,1], row_half_mirror
  const int flip = control == 0xB1 ? 1 : control == 0x4E ? 2 : control == 0x141 ? 7 : 0;
  if (!flip) cpu::fail("unknown lane pattern");
  return (int)cpu::exchange((uint32_t)v, cpu::current ^ flip);
}
#define __builtin_amdgcn_mov_dpp(v, control, row, bank, bound) cpu_dpp(v, control)
#define __builtin_amdgcn_rcpf(v) (1.0f / (v))
inline uint32_t __umulhi(uint32_t a, uint32_t b) { return (uint32_t)(((uint64_t)a * b) >> 32); }
inline float __expf(float x) { return std::exp(x); }
inline uint32_t __float_as_uint(float f) { return __builtin_bit_cast(uint32_t, f); }
inline float __uint_as_float(uint32_t u) { return __builtin_bit_cast(float, u); }
template <typename T>
T max(T a, T b) {
  return a > b ? a : b;
}
template <typename T>
T min(T a, T b) {
  return a < b ? a : b;
}
#define hipLaunchKernelGGL(kernel, grid, block, lds, stream, ...) \
  cpu::run((grid).x, (int)(block).x, [=]() { kernel(__VA_ARGS__); })
