// dpft_norm.hip -- the encoder's normalisation for gfx950 (MI355X): group normalisation with an
// activation on channels_last maps, forward and backward, and activation checkpoints in 8 bits.
// ABI and semantics: include/dpft_ic.h (dpft_group_norm_act*, dpft_act_checkpoint / _restore).
//
// A sample is L = pixels * C values in a row.  Threads walk it as a matrix of rows of
// Cv = lcm(C, V) values, V = the 16-byte load's values, so that a thread's V values belong to the
// same channels in every row it visits, whatever C is: its channel sums and its affine coefficients
// stay in registers.  A row that L cuts short is handled value by value.
//
// Everything here moves far more bytes than it computes on (12 to 40 flops per value of 2 to 20
// bytes): bound by memory at the large sizes, by launches at the small ones.  The rates beside the kernels
// are the bytes that they ask for over their time, in graphs of calls on many sets of inputs: a call's inputs
// come from HBM, and of what a second pass reads again the Infinity Cache still holds a part, which is why some
// exceed the 6.22 TB/s (read and written) of dpft_copy_probe on 1 GiB.
// Two passes over x, not one: kernels that held a sample's values in registers from the statistics to
// the result, workgroups waiting for each other's sums, took 198 to 303 us where two passes took 213 to
// 291 -- all of them load, join and store at the same time, and the memory idles in between.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <numeric>
#include <type_traits>

#include "dpft_ic.h"
#include "dpft_internal.h"

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kBlock8 = 32;  // values that share a scale in a checkpoint

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));  // a 16-byte access at any value's address

template <typename T>
struct Vec {
  static constexpr int V = 16 / (int)sizeof(T);
  typedef T type __attribute__((ext_vector_type(V)));
};

// At a uniform base and a thread's 32-bit offset in values (the access's scalar-base form).
template <typename T>
__device__ __forceinline__ T* at(T* base, uint32_t off) {
  typedef std::conditional_t<std::is_const_v<T>, const char, char> Byte;
  return reinterpret_cast<T*>(reinterpret_cast<Byte*>(base) + (size_t)(off * (uint32_t)sizeof(T)));
}
template <typename T>
__device__ __forceinline__ u32x4 load_raw(const T* p) {
  return *reinterpret_cast<const u32x4_any*>(p);
}
template <typename T>
__device__ __forceinline__ void widen(u32x4 raw, float (&v)[Vec<T>::V]) {
  const auto r = __builtin_bit_cast(typename Vec<T>::type, raw);
#pragma unroll
  for (int j = 0; j < Vec<T>::V; ++j) v[j] = (float)r[j];
}
template <typename T>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[Vec<T>::V]) {
  widen<T>(load_raw(p), v);
}
// The first m of V values, zeros behind them.
template <typename T>
__device__ __forceinline__ u32x4 load_first(const T* p, int m) {
  typename Vec<T>::type r = {};
#pragma unroll
  for (int j = 0; j < Vec<T>::V; ++j)
    if (j < m) r[j] = p[j];
  return __builtin_bit_cast(u32x4, r);
}
template <typename T>
__device__ __forceinline__ void store_first(T* p, const float (&v)[Vec<T>::V], int m) {
#pragma unroll
  for (int j = 0; j < Vec<T>::V; ++j)
    if (j < m) p[j] = (T)v[j];
}
// Rounds to T to nearest even: the values' own type.  Non-temporal: kept in L2, the results drive out
// what the next pass reads (8 x 32 x 480 x 640 fp32: 205 -> 178 us).
template <typename T>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[Vec<T>::V]) {
  typename Vec<T>::type r;
#pragma unroll
  for (int j = 0; j < Vec<T>::V; ++j) r[j] = (T)v[j];
  __builtin_nontemporal_store(__builtin_bit_cast(u32x4, r), reinterpret_cast<u32x4_any*>(p));
}

__device__ __forceinline__ float load_param(const void* p, int type, int i, float none) {
  if (!p) return none;
  if (type == DPFT_TYPE_F32) return static_cast<const float*>(p)[i];
  if (type == DPFT_TYPE_BF16) return (float)static_cast<const __bf16*>(p)[i];
  return (float)static_cast<const _Float16*>(p)[i];
}
__device__ __forceinline__ void store_param(void* p, int type, int i, float v) {
  if (type == DPFT_TYPE_F32) static_cast<float*>(p)[i] = v;
  else if (type == DPFT_TYPE_BF16) static_cast<__bf16*>(p)[i] = (__bf16)v;
  else static_cast<_Float16*>(p)[i] = (_Float16)v;
}

// ------------------------------------------------------------------ activations
// expm1 on z <= 0: its Taylor polynomial to z^6 above -1/4 (the next term is 4.8e-8 of the value
// there), exp(z) - 1 below (whose error of 1.2 x 2^-24 is at most 5.5 x 2^-24 of the value).  Both are
// computed and one is selected: as branches, which lanes part at, a value after the other.
template <typename T>
__device__ __forceinline__ float expm1_neg(float z) {
  if constexpr (sizeof(T) < 4) {
    // for a result of 16 bits: to z^3 above -1/16 (the next term is at most 2^-16.5 of the value), and
    // exp(z) - 1 below (2^-19): against half a step of 2^-8 (bf16) or 2^-11 (fp16)
    const float near = fmaf(z * z, fmaf(z, 1.0f / 6, 0.5f), z), far = __expf(z) - 1.0f;
    return z > -0.0625f ? near : far;
  }
  float q = 1.0f / 720;
  q = fmaf(q, z, 1.0f / 120);
  q = fmaf(q, z, 1.0f / 24);
  q = fmaf(q, z, 1.0f / 6);
  q = fmaf(q, z, 0.5f);
  const float near = fmaf(z * z, q, z), far = __expf(z) - 1.0f;
  return z > -0.25f ? near : far;
}
template <int ACT, typename T>
__device__ __forceinline__ float act_fwd(float z) {
  if constexpr (ACT == DPFT_ACT_RELU) return z < 0.0f ? 0.0f : z;
  if constexpr (ACT == DPFT_ACT_ELU) {
    const float below = expm1_neg<T>(z);
    return z > 0.0f ? z : below;
  }
  if constexpr (ACT == DPFT_ACT_SILU) return z * __builtin_amdgcn_rcpf(1.0f + __expf(-z));
  return z;
}
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == DPFT_ACT_RELU) return z <= 0.0f ? 0.0f : 1.0f;
  if constexpr (ACT == DPFT_ACT_ELU) return z > 0.0f ? 1.0f : __expf(z);
  if constexpr (ACT == DPFT_ACT_SILU) {
    const float t = __expf(fminf(-z, 87.0f)), s = __builtin_amdgcn_rcpf(1.0f + t);
    return s * fmaf(z, t * s, 1.0f);  // 1 - s = t s without cancellation
  }
  return 1.0f;
}

// ------------------------------------------------------------------ checkpoints in 8 bits
// The step of a block is a power of two, so x / step and q * step are exact: a value is rounded
// once, and is the same in every type it is restored to.
__device__ __forceinline__ float step_of(int scale) {  // 255: NaN
  return scale == 255 ? __builtin_nanf("") : __uint_as_float((uint32_t)(scale - 6) << 23);
}
__device__ __forceinline__ int scale_of(float top) {
  const int e = (int)(__float_as_uint(top) >> 23) & 255;
  return e == 255 ? 255 : max(7, min(e, 254));
}
__device__ __forceinline__ int quantise(float x, float per_step) {
  return (int)fminf(fmaxf(rintf(x * per_step), -127.0f), 127.0f);
}
__device__ __forceinline__ float per_step_of(int scale) {
  return scale == 255 ? 0.0f : __uint_as_float((uint32_t)(260 - scale) << 23);
}

// max over the 32 / V neighbouring lanes that hold a block (aligned groups of 4 or 8 lanes).
template <int LANES>
__device__ __forceinline__ uint32_t block_max(uint32_t m) {
  static_assert(LANES == 4 || LANES == 8);
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xF, 0xF, true));  // quad_perm [1,0,3,2]
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xF, 0xF, true));  // quad_perm [2,3,0,1]
  if constexpr (LANES == 8) m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x141, 0xF, 0xF, true));
  return m;
}
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <int V>
struct Bytes;  // V signed bytes
template <>
struct Bytes<4> {
  typedef uint32_t type;
};
template <>
struct Bytes<8> {
  typedef u32x2 type;
};
__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
  return (a & 255) | (b & 255) << 8 | (c & 255) << 16 | (uint32_t)d << 24;
}
// One thread's V values of a block that 32 / V neighbouring lanes share: their bytes, and the
// block's scale (the largest magnitude's bits carry its exponent; NaN and infinity have 255).
template <int V>
__device__ __forceinline__ typename Bytes<V>::type quantise_vec(const float (&v)[V], int& scale) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
  scale = scale_of(__uint_as_float(block_max<kBlock8 / V>(m)));
  const float ps = per_step_of(scale);
  int q[V];
#pragma unroll
  for (int j = 0; j < V; ++j) q[j] = quantise(v[j], ps);
  const uint32_t keep = scale == 255 ? 0u : ~0u;
  if constexpr (V == 4) return pack4(q[0], q[1], q[2], q[3]) & keep;
  else return u32x2{pack4(q[0], q[1], q[2], q[3]) & keep, pack4(q[4], q[5], q[6], q[7]) & keep};
}
template <int V>
__device__ __forceinline__ void restore_vec(typename Bytes<V>::type b, float step, float (&v)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) {
    uint32_t word;
    if constexpr (V == 4) word = b;
    else word = b[j / 4];
    v[j] = (float)(int8_t)(word >> (8 * (j % 4))) * step;
  }
}

// 16 bytes of x per thread and step, kUnroll steps in flight; the block's maximum by lane shifts.
// Bound by memory (8 x 32 x 480 x 640 fp32: 64 us, 6.2 TB/s).
constexpr int kUnroll = 4;
template <typename T>
__global__ __launch_bounds__(kThreads) void act_checkpoint_kernel(const T* __restrict__ x, int64_t n,
                                                                  int8_t* __restrict__ q, uint8_t* __restrict__ scale) {
  constexpr int V = Vec<T>::V;
  typedef typename Bytes<V>::type Q;
  const int64_t chunk = (int64_t)kThreads * V, stride = (int64_t)gridDim.x * kUnroll * chunk;
  for (int64_t c0 = (int64_t)blockIdx.x * kUnroll * chunk; c0 < n; c0 += stride) {
    const int64_t i0 = c0 + threadIdx.x * V;
    if (c0 + kUnroll * chunk <= n) {
      float v[kUnroll][V];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) load_vec(x + i0 + u * chunk, v[u]);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int64_t i = i0 + u * chunk;
        int sc;
        *reinterpret_cast<Q*>(q + i) = quantise_vec<V>(v[u], sc);
        if (i % kBlock8 == 0) scale[i / kBlock8] = (uint8_t)sc;
      }
    } else {
      for (int u = 0; u < kUnroll; ++u) {  // every lane takes part in its block's maximum
        const int64_t i = i0 + u * chunk;
        float v[V];
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = i + j < n ? (float)x[i + j] : 0.0f;
        int sc;
        const Q b = quantise_vec<V>(v, sc);
        if (i % kBlock8 == 0 && i < n) scale[i / kBlock8] = (uint8_t)sc;
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (i + j < n) q[i + j] = reinterpret_cast<const int8_t*>(&b)[j];
      }
    }
  }
}

// As the other way (8 x 32 x 480 x 640 fp32, just checkpointed: 56 us, 7.1 TB/s).
template <typename T>
__global__ __launch_bounds__(kThreads) void act_restore_kernel(const int8_t* __restrict__ q,
                                                               const uint8_t* __restrict__ scale, int64_t n,
                                                               T* __restrict__ out) {
  constexpr int V = Vec<T>::V;
  typedef typename Bytes<V>::type Q;
  const int64_t chunk = (int64_t)kThreads * V, stride = (int64_t)gridDim.x * kUnroll * chunk;
  for (int64_t c0 = (int64_t)blockIdx.x * kUnroll * chunk; c0 < n; c0 += stride) {
    const int64_t i0 = c0 + threadIdx.x * V;
    if (c0 + kUnroll * chunk <= n) {
      Q b[kUnroll];
      int sc[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        b[u] = *reinterpret_cast<const Q*>(q + i0 + u * chunk);
        sc[u] = scale[(i0 + u * chunk) / kBlock8];
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        float v[V];
        restore_vec<V>(b[u], step_of(sc[u]), v);
        store_vec(out + i0 + u * chunk, v);
      }
    } else {
      for (int u = 0; u < kUnroll; ++u)
        for (int64_t i = i0 + u * chunk; i < min(i0 + u * chunk + V, n); ++i)
          out[i] = (T)((float)q[i] * step_of(scale[i / kBlock8]));
    }
  }
}

// ------------------------------------------------------------------ the walk over a sample
// A workgroup (n, part, tile) visits the blocks part, part + parts, ... of sample n: a block is `deep`
// vectors a thread of RS rows side by side, so that the grid reads one stretch of memory at a time.
struct Walk {
  int64_t L;      // values of a sample
  int64_t rows;   // rows of Cv values, the last one cut short where L % Cv != 0
  int64_t full;   // whole rows
  int32_t N, C, D, G;
  int32_t Cv, S;  // values and 16-byte slots of a row
  int32_t W, tiles;  // slots of a tile (at most kThreads), tiles of a row
  int32_t RS;     // rows that a workgroup visits side by side
  int32_t parts, blocks;  // workgroups (per tile) and blocks of a sample
  int32_t in_block;     // a thread's V values lie in one checkpoint block
  int32_t lanes_block;  // ... and the rows that a workgroup visits side by side are whole blocks
};

// Vectors of a block, which a thread has in flight: of the statistics, of the apply pass, of the backward's two.
constexpr int kDeep = 8, kDeepApply = 4, kDeepSums = 4, kDeepGrad = 2;

struct Place {
  int n, part, tile, slot, rr;
  bool active;
  uint32_t off;     // the thread's first value in RS rows
  int channel;      // of the thread's first value
  __device__ __forceinline__ Place(const Walk& w, int V, int b) {
    tile = b % w.tiles;
    const int np = b / w.tiles;
    n = np / w.parts;
    part = np - n * w.parts;
    const int t = threadIdx.x;
    rr = t / w.W;
    slot = tile * w.W + (t - rr * w.W);
    active = rr < w.RS && slot < w.S;
    if (!active) {
      rr = 0;
      slot = tile * w.W;
    }
    off = rr * w.Cv + slot * V;
    channel = slot * V % w.C;
  }
};
// Of block b: vectors 0 .. whole - 1 of every thread are the sample's, of vector `whole` the first
// `tail` values (0 where there is none: whole == deep), none behind it.
struct Block {
  int whole, tail;
  int64_t at;  // the block's first value
  __device__ __forceinline__ Block(const Walk& w, const Place& p, int b, int deep, int V) {
    const int64_t r0 = (int64_t)b * deep * w.RS;
    at = p.n * w.L + r0 * w.Cv;
    whole = deep;
    tail = 0;
    if (b == w.blocks - 1) {  // (the others are whole: the division stays out of the loops)
      whole = (int)min((w.full - r0) / w.RS, (int64_t)deep);
      const int64_t r = r0 + (int64_t)whole * w.RS + p.rr;
      tail = whole == deep ? 0 : r < w.full ? V : r == w.full ? tail_values(w, p.slot, V) : 0;
    }
  }
  // Values of the cut row that fall to `slot`.
  static __device__ __forceinline__ int tail_values(const Walk& w, int slot, int V) {
    const int64_t left = w.L - w.full * w.Cv - (int64_t)slot * V;
    return (int)max((int64_t)0, min(left, (int64_t)V));
  }
};

// Threads that share a group's (or a position's) sum: a power of two, at most a wave.
__device__ __forceinline__ int sharers(int things, int threads = kThreads) {
  int q = 64;
  while (q > 1 && q * things > threads) q >>= 1;
  return q;
}
template <typename F>
__device__ __forceinline__ F lanes_sum(F v, int q) {
  for (int o = q >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
// f(i) by Q lanes over `rows` x `n` entries r * row + i, i < n, in a fixed order.
template <typename F>
__device__ __forceinline__ void over_box(int rows, int row, int n, int lane, int Q, F&& f) {
  const uint32_t by_n = n > 1 ? 0xffffffffu / (uint32_t)n + 1 : 0;  // r = e / n, exact for e n < 2^32
#pragma unroll 4
  for (int e = lane; e < rows * n; e += Q) {
    const int r = n > 1 ? (int)__umulhi((uint32_t)e, by_n) : e;
    f(r * row + (e - r * n));
  }
}
// f(i) by Q lanes over the entries i of group g in shared memory that lie in a tile: an entry for each
// `per` values of a tile's row, RS rows.
template <typename F>
__device__ __forceinline__ void over_entries(const Walk& w, int tile, int V, int per, int g, int lane, int Q, F&& f) {
  const int lo = tile * w.W * V, hi = min(lo + w.W * V, w.Cv), RE = w.W * V / per;
#pragma unroll 1
  for (int k = g * w.D; k < hi; k += w.C) {  // the row's copies of the group's channels
    const int e0 = (max(k, lo) - lo) / per, e1 = (min(k + w.D, hi) - lo) / per;
    if (e1 > e0) over_box(w.RS, RE, e1 - e0, lane, Q, [&](int i) { f(e0 + i); });
  }
}

// ------------------------------------------------------------------ forward
// Records [n][parts * tiles][G]: mean, sum of squares about it and count of the workgroup's values of a
// group.  A thread takes the exact mean of kDeep values of a position, then their squares about it, and
// joins the batches by the parallel-variance rule; the threads are joined in the same way: nothing
// cancels, whatever the mean is.  Bound by memory: 8 x 32 x 480 x 640 fp32 53.0 us, 5.9 TB/s; 16 x 64 x
// 240 x 320 bf16 30.7 us, 5.1 TB/s.
template <typename T>
__global__ __launch_bounds__(kThreads) void gn_stats_kernel(const T* __restrict__ x, Walk w, float4* __restrict__ rec) {
  constexpr int V = Vec<T>::V;
  __shared__ float s_mean[kThreads * V], s_m2[kThreads * V], s_cnt[kThreads * V];
  const Place p(w, V, blockIdx.x);
  const int step = w.RS * w.Cv;
  float mean[V] = {}, m2[V] = {};
  int cnt = 0, tail = 0;
  // The exact means of the first n vectors, their squares about them, and both joined to what there is.
  // (Selects where n < kDeep: branches cost registers, and a branch a vector a fifth of the rate.)
  auto join = [&](const u32x4(&raw)[kDeep], int n, auto whole) {
    float s[V] = {}, q[V] = {};
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
      float v[V];
      widen<T>(raw[u], v);
#pragma unroll
      for (int j = 0; j < V; ++j) s[j] += whole || u < n ? v[j] : 0.0f;
    }
    const float r = whole ? 1.0f / kDeep : 1.0f / (float)n;
#pragma unroll
    for (int j = 0; j < V; ++j) s[j] *= r;
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
      float v[V];
      widen<T>(raw[u], v);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = whole || u < n ? v[j] - s[j] : 0.0f;
        q[j] = fmaf(d, d, q[j]);
      }
    }
    const float f = (float)n * __builtin_amdgcn_rcpf((float)(cnt + n)), c = (float)cnt * f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float d = s[j] - mean[j];
      mean[j] = fmaf(d, f, mean[j]);
      m2[j] += fmaf(d * d, c, q[j]);
    }
    cnt += n;
  };
#pragma unroll 1
  for (int b = p.part; b < w.blocks; b += w.parts) {
    const Block blk(w, p, b, kDeep, V);
    const T* src = x + blk.at;
    u32x4 raw[kDeep];
    if (blk.whole == kDeep) {
#pragma unroll
      for (int u = 0; u < kDeep; ++u) raw[u] = load_raw(at(src + (int64_t)u * step, p.off));
      join(raw, kDeep, std::true_type{});
    } else {  // the sample's last block
      if (blk.whole) {
#pragma unroll
        for (int u = 0; u < kDeep; ++u) raw[u] = load_raw(at(src + (int64_t)min(u, blk.whole - 1) * step, p.off));
        join(raw, blk.whole, std::false_type{});
      }
      tail = blk.tail;
      float v[V];
      widen<T>(load_first(at(src + (int64_t)blk.whole * step, p.off), tail), v);
      const float f = 1.0f / (float)(cnt + 1);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < tail) {
          const float d = v[j] - mean[j];
          mean[j] = fmaf(d, f, mean[j]);
          m2[j] = fmaf(d, v[j] - mean[j], m2[j]);
        }
    }
  }
  const bool merged = w.D % V == 0;  // a thread's V values are one group's: one entry
  const float none = p.active ? 1.0f : 0.0f;
  if (merged) {
    float mu = 0.0f, sq = 0.0f;
    const float n = (float)(cnt * V + tail);
#pragma unroll
    for (int j = 0; j < V; ++j) mu = fmaf((float)(cnt + (j < tail)), mean[j], mu);
    mu = n > 0.0f ? mu / n : 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) sq += fmaf((float)(cnt + (j < tail)) * (mean[j] - mu), mean[j] - mu, m2[j]);
    s_mean[threadIdx.x] = mu;
    s_m2[threadIdx.x] = sq;
    s_cnt[threadIdx.x] = n * none;
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      s_mean[threadIdx.x * V + j] = mean[j];
      s_m2[threadIdx.x * V + j] = m2[j];
      s_cnt[threadIdx.x * V + j] = (float)(cnt + (j < tail)) * none;
    }
  }
  __syncthreads();
  const int Q = sharers(w.G), lane = threadIdx.x & (Q - 1), per = merged ? V : 1;
  rec += ((int64_t)(p.n * w.parts + p.part) * w.tiles + p.tile) * w.G;
#pragma unroll 1
  for (int g = threadIdx.x / Q; g < w.G; g += kThreads / Q) {
    float cn = 0.0f, cs = 0.0f, cq = 0.0f;
    over_entries(w, p.tile, V, per, g, lane, Q, [&](int i) {
      cn += s_cnt[i];
      cs = fmaf(s_cnt[i], s_mean[i], cs);
    });
    cn = lanes_sum(cn, Q);
    cs = lanes_sum(cs, Q);
    const float mu = cn > 0.0f ? cs / cn : 0.0f;
    over_entries(w, p.tile, V, per, g, lane, Q, [&](int i) {
      cq += fmaf(s_cnt[i] * (s_mean[i] - mu), s_mean[i] - mu, s_cnt[i] > 0.0f ? s_m2[i] : 0.0f);
    });
    cq = lanes_sum(cq, Q);
    if (lane == 0) rec[g] = make_float4(mu, cq, cn, 0.0f);
  }
}

// Sample n's statistics of group g from its records, by Q lanes in a fixed order: in fp64, where the
// sums of n, n mean and m2 + n mean^2 do for the spread.  All Q lanes return them.
__device__ __forceinline__ float2 join_stats(const float4* rec, int R, int G, int n, int g, int lane, int Q, float eps) {
  const float4* r = rec + (int64_t)n * R * G + g;
  double cn = 0.0, cs = 0.0, cq = 0.0;
#pragma unroll 4
  for (int i = lane; i < R; i += Q) {
    const float4 a = r[(int64_t)i * G];
    const double m = a.x, c = a.z;
    cn += c;
    cs += c * m;
    cq += a.y + c * m * m;
  }
  cn = lanes_sum(cn, Q);
  cs = lanes_sum(cs, Q);
  cq = lanes_sum(cq, Q);
  const double mu = cs / cn, sq = cq - cs * mu;
  return make_float2((float)mu, (float)(1.0 / sqrt((sq < 0.0 ? 0.0 : sq) / cn + (double)eps)));  // keeps a NaN
}

// Where a workgroup cannot join a sample's groups itself: a wave per (sample, group).
__global__ __launch_bounds__(kThreads) void gn_finish_stats_kernel(const float4* __restrict__ rec, int R, int N, int G,
                                                                   float eps, float* __restrict__ mean,
                                                                   float* __restrict__ rstd) {
  const int lane = threadIdx.x & 63;
#pragma unroll 1
  for (int64_t i = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6); i < (int64_t)N * G; i += (int64_t)gridDim.x * kWaves) {
    const int n = (int)(i / G), g = (int)(i - (int64_t)n * G);
    const float2 r = join_stats(rec, R, G, n, g, lane, 64, eps);
    if (lane == 0) {
      mean[i] = r.x;
      rstd[i] = r.y;
    }
  }
}

struct Affine {
  const void *weight, *bias;
  const float *mean, *rstd;
  int32_t type;
};

// y = act((x - mean) a + bias), a = rstd * weight.
// MODE: y as x is stored, in the channel-quad layout, or with x's checkpoint (w.lanes_block).
// rec: the workgroup joins the statistics itself (kFold groups at most), its part 0 stores them.
// Bound by memory: 8 x 32 x 480 x 640 fp32 100.6 us, 6.3 TB/s; 16 x 64 x 240 x 320 bf16 52.9 us, 5.9; with
// a checkpoint, 8 x 64 x 240 x 320 fp32 64.4 us, 5.5.
constexpr int kFold = 128;
enum { kPlain, kPacked, kCheckpoint };
template <typename T, int ACT, int MODE>
__global__ __launch_bounds__(kThreads) void gn_apply_kernel(const T* __restrict__ x, Walk w, Affine f,
                                                            const float4* __restrict__ rec, int R, float eps,
                                                            float* mean_out, float* rstd_out, T* __restrict__ y,
                                                            int8_t* __restrict__ q, uint8_t* __restrict__ scale) {
  constexpr int V = Vec<T>::V;
  __shared__ float s_mu[kFold], s_rs[kFold];
  const Place p(w, V, blockIdx.x);
  const int step = w.RS * w.Cv;
  // The blocks backwards: the statistics' pass has read the last ones last.  The next block's loads are
  // issued as the vectors of this one are used, the first one's before the statistics are joined.
  int b = w.blocks - 1 - p.part;
  u32x4 raw[kDeepApply], end{};
  Block blk(w, p, b, kDeepApply, V);
  auto load = [&](int u) { raw[u] = load_raw(at(x + blk.at + (int64_t)u * step, p.off)); };
#pragma unroll
  for (int u = 0; u < kDeepApply; ++u)
    if (u < blk.whole) load(u);
  if (blk.whole < kDeepApply) end = load_first(at(x + blk.at + (int64_t)blk.whole * step, p.off), blk.tail);
  float mu[V], a[V], bias[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c0 = p.channel + j, c = c0 < w.C ? c0 : c0 % w.C;
    a[j] = load_param(f.weight, f.type, c, 1.0f);
    bias[j] = load_param(f.bias, f.type, c, 0.0f);
  }
  if (rec) {
    const int Q = sharers(w.G), lane = threadIdx.x & (Q - 1);
#pragma unroll 1
    for (int g = threadIdx.x / Q; g < w.G; g += kThreads / Q) {
      const float2 r = join_stats(rec, R, w.G, p.n, g, lane, Q, eps);
      if (lane == 0) {
        s_mu[g] = r.x;
        s_rs[g] = r.y;
        if (mean_out && p.part == 0 && p.tile == 0) {
          mean_out[p.n * w.G + g] = r.x;
          rstd_out[p.n * w.G + g] = r.y;
        }
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c0 = p.channel + j, g = (c0 < w.C ? c0 : c0 % w.C) / w.D;
    mu[j] = rec ? s_mu[g] : f.mean[p.n * w.G + g];
    a[j] *= rec ? s_rs[g] : f.rstd[p.n * w.G + g];
  }
  // in the channel-quad layout a slot's rows follow one another
  const int out_step = MODE == kPacked ? w.RS * V : step;
  auto one = [&](const float(&x1)[V], int m, int64_t o, T* out) {
    float v[V];
    if constexpr (MODE == kCheckpoint) {  // rows come in whole blocks: m is V or 0, alike over a block
      int sc;
      const auto bytes = quantise_vec<V>(x1, sc);
      if (m == V && p.active) {
        *reinterpret_cast<typename Bytes<V>::type*>(at(q + o, p.off)) = bytes;
        if (p.off % kBlock8 == 0) *at(scale + o / kBlock8, p.off / kBlock8) = (uint8_t)sc;  // o % 32 == 0
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = act_fwd<ACT, T>(fmaf(x1[j] - mu[j], a[j], bias[j]));
    if (!p.active) return;
    if (m == V) store_vec(out, v);
    else if (MODE != kPacked) store_first(out, v, m);
  };
  auto first_out = [&](int64_t o) {
    if constexpr (MODE == kPacked) return y + p.n * w.L + (p.slot * w.rows + (o - p.n * w.L) / w.Cv + p.rr) * V;
    else return at(y + o, p.off);
  };
  if (blk.whole < kDeepApply) {  // the sample's last block
    const int64_t o = blk.at;
    const int whole = blk.whole;
    T* out = first_out(o);
    float v[V];
#pragma unroll
    for (int u = 0; u < kDeepApply - 1; ++u)
      if (u < whole) {
        widen<T>(raw[u], v);
        one(v, V, o + (int64_t)u * step, out + (int64_t)u * out_step);
      }
    widen<T>(end, v);
    one(v, blk.tail, o + (int64_t)whole * step, out + (int64_t)whole * out_step);
    b -= w.parts;
    if (b < 0) return;
    blk = Block(w, p, b, kDeepApply, V);
#pragma unroll
    for (int u = 0; u < kDeepApply; ++u) load(u);
  }
#pragma unroll 1
  for (;;) {
    const int64_t o = blk.at;
    T* out = first_out(o);
    b -= w.parts;
    const bool more = b >= 0;
    if (more) blk = Block(w, p, b, kDeepApply, V);
#pragma unroll
    for (int u = 0; u < kDeepApply; ++u, out += out_step) {
      float v[V];
      widen<T>(raw[u], v);
      if (more) load(u);
      one(v, V, o + (int64_t)u * step, out);
    }
    if (!more) break;
  }
}

// ------------------------------------------------------------------ small maps
// A workgroup takes cw channels (whole groups) of a sample and holds all their pixels in registers: one
// launch, every value read once.  Bound by latency.  Against two passes, fp32 in a graph: 1 x 128 x 15 x
// 20 8.1 us (11.5), 32 x 128 x 30 x 34 14.4 (18.2); of one sample only, 8 vectors a thread 9.3 (11.3),
// 16 vectors 12.6 (11.5).
constexpr int kSmall = 512;       // threads
constexpr int kSmallHold = 16;    // vectors of x that a thread holds, in the backward kSmallHold / 2 of x and of dy
struct Slice {
  int64_t P;         // pixels
  int32_t C, D, G;   // channels, a group's, groups
  int32_t cw, S, RS; // channels, 16-byte slots and rows side by side of a workgroup
  int32_t nv;        // vectors that a thread holds
};
struct SliceSpot {
  int n, c0, rr, slot, c;  // sample, first channel, row, slot, the thread's first channel
  bool active;
  __device__ __forceinline__ SliceSpot(const Slice& w, int V) {
    const int per = w.C / w.cw, b = blockIdx.x, t = threadIdx.x;
    n = b / per;
    c0 = (b - n * per) * w.cw;
    rr = t / w.S;
    slot = t - rr * w.S;
    active = rr < w.RS;
    c = c0 + slot * V;
  }
};
// f(group of the workgroup, sums of v over its threads), v per thread (D % V == 0: one group's).
template <typename F>
__device__ __forceinline__ void slice_sums(const Slice& w, int V, float2 v, float2* s, F&& f) {
  const int gw = w.cw / w.D, DE = w.D / V, Q = sharers(gw, kSmall), lane = threadIdx.x & (Q - 1);
  s[threadIdx.x] = v;
  __syncthreads();
#pragma unroll 1
  for (int g = threadIdx.x / Q; g < gw; g += kSmall / Q) {
    float2 a = make_float2(0.0f, 0.0f);
    auto add = [&](float2 t) {
      a.x += t.x;
      a.y += t.y;
    };
    over_box(w.RS, w.S, DE, lane, Q, [&](int i) { add(s[g * DE + i]); });
    a.x = lanes_sum(a.x, Q);
    a.y = lanes_sum(a.y, Q);
    if (lane == 0) f(g, a);
  }
  __syncthreads();
}

template <typename T, int ACT, int MODE>
__global__ __launch_bounds__(kSmall) void gn_small_kernel(const T* __restrict__ x, Slice w, Affine f, float eps,
                                                          float* mean_out, float* rstd_out, T* __restrict__ y,
                                                          int8_t* __restrict__ q, uint8_t* __restrict__ scale) {
  constexpr int V = Vec<T>::V;
  __shared__ float2 s[kSmall];
  __shared__ float s_mu[kSmall], s_rs[kSmall];
  const SliceSpot p(w, V);
  const int64_t base = (int64_t)p.n * w.P * w.C + p.c;
  u32x4 raw[kSmallHold];
#pragma unroll
  for (int i = 0; i < kSmallHold; ++i)
    if (i < w.nv) {
      const int64_t r = p.rr + (int64_t)i * w.RS;
      raw[i] = u32x4{};
      if (p.active && r < w.P) raw[i] = load_raw(x + base + r * w.C);
    }
  float a[V], b[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    a[j] = load_param(f.weight, f.type, p.c + j, 1.0f);
    b[j] = load_param(f.bias, f.type, p.c + j, 0.0f);
  }
  // a mean of plain sums, and from the distances to it its error and the spread: exact to fp32 wherever
  // the mean lies
  float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
  for (int i = 0; i < kSmallHold; ++i)
    if (i < w.nv) {
      float v[V];
      widen<T>(raw[i], v);
#pragma unroll
      for (int j = 0; j < V; ++j) sum.x += v[j];
    }
  const float cnt = (float)(w.P * w.D);
  slice_sums(w, V, sum, s, [&](int g, float2 t) { s_mu[g] = t.x / cnt; });
  const int gl = (p.c - p.c0) / w.D;
  const float mu0 = s_mu[gl];
  sum = make_float2(0.0f, 0.0f);
#pragma unroll
  for (int i = 0; i < kSmallHold; ++i)
    if (i < w.nv) {
      float v[V];
      widen<T>(raw[i], v);
      const bool in = p.active && p.rr + (int64_t)i * w.RS < w.P;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = in ? v[j] - mu0 : 0.0f;
        sum.x += d;
        sum.y = fmaf(d, d, sum.y);
      }
    }
  slice_sums(w, V, sum, s, [&](int g, float2 t) {
    const double e = (double)t.x / cnt, var = (double)t.y / cnt - e * e;
    const float r = (float)(1.0 / sqrt((var < 0.0 ? 0.0 : var) + (double)eps));  // keeps a NaN
    s_mu[g] = (float)(s_mu[g] + e);
    s_rs[g] = r;
    if (mean_out) {
      const int i = p.n * w.G + p.c0 / w.D + g;
      mean_out[i] = s_mu[g];
      rstd_out[i] = r;
    }
  });
  const float mu = s_mu[gl];
  const float rs = s_rs[gl];
#pragma unroll
  for (int j = 0; j < V; ++j) a[j] *= rs;
#pragma unroll
  for (int i = 0; i < kSmallHold; ++i)
    if (i < w.nv) {
      const int64_t r = p.rr + (int64_t)i * w.RS;
      const bool in = p.active && r < w.P;
      float v[V];
      widen<T>(raw[i], v);
      const int64_t o = base + r * w.C;
      if constexpr (MODE == kCheckpoint) {  // cw % 32 == 0: a block is 32 channels of a pixel
        int sc;
        const auto bytes = quantise_vec<V>(v, sc);
        if (in) {
          *reinterpret_cast<typename Bytes<V>::type*>(q + o) = bytes;
          if (p.slot % (kBlock8 / V) == 0) scale[o / kBlock8] = (uint8_t)sc;
        }
      }
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = act_fwd<ACT, T>(fmaf(v[j] - mu, a[j], b[j]));
      if (!in) continue;
      if constexpr (MODE == kPacked) store_vec(y + (int64_t)p.n * w.P * w.C + ((p.c / V) * w.P + r) * V, v);
      else store_vec(y + o, v);
    }
}

// ------------------------------------------------------------------ backward
// The values of x that a thread reads: x itself, or its checkpoint restored.
template <typename T, bool Q8>
struct Source {
  const T* x;
  const int8_t* q;
  const uint8_t* scale;
  int in_block;
};
template <typename T, bool Q8>
struct Pair {  // V values of x and of dy in flight
  u32x4 xs, d;
  __device__ __forceinline__ void load(const Source<T, Q8>& x, const T* dy, int64_t o, uint32_t off) {
    xs = load_raw(at(x.x + o, off));
    d = load_raw(at(dy + o, off));
  }
  __device__ __forceinline__ void get(const Source<T, Q8>&, float (&v)[Vec<T>::V], float (&dv)[Vec<T>::V]) const {
    widen<T>(xs, v);
    widen<T>(d, dv);
  }
};
template <typename T>
struct Pair<T, true> {
  static constexpr int V = Vec<T>::V;
  typename Bytes<V>::type q;
  int s0, s1;  // the scales of the values before and from `cut` on
  int cut;
  u32x4 d;
  __device__ __forceinline__ void load(const Source<T, true>& x, const T* dy, int64_t o, uint32_t off) {
    const int64_t i = o + off;
    if (x.in_block) {
      q = *reinterpret_cast<const typename Bytes<V>::type*>(at(x.q + o, off));
      s0 = x.scale[i / kBlock8];
    } else {  // at any byte, over two blocks
      typedef typename Bytes<V>::type Any __attribute__((aligned(1)));
      q = *reinterpret_cast<const Any*>(at(x.q + o, off));
      s0 = x.scale[i / kBlock8];
      s1 = x.scale[(i + V - 1) / kBlock8];
      cut = kBlock8 - (int)(i % kBlock8);
    }
    d = load_raw(at(dy + o, off));
  }
  __device__ __forceinline__ void get(const Source<T, true>& x, float (&v)[V], float (&dv)[V]) const {
    if (x.in_block) {
      restore_vec<V>(q, step_of(s0), v);
    } else {
      restore_vec<V>(q, 1.0f, v);
      const float a = step_of(s0), b = step_of(s1);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] *= j < cut ? a : b;
    }
    widen<T>(d, dv);
  }
};
// The first m values one by one, zeros behind them.
template <typename T, bool Q8>
__device__ __forceinline__ void first_values(const Source<T, Q8>& x, const T* dy, int64_t i, int m, float (&v)[Vec<T>::V],
                                             float (&d)[Vec<T>::V]) {
#pragma unroll
  for (int j = 0; j < Vec<T>::V; ++j) {
    v[j] = d[j] = 0.0f;
    if (j < m) {
      if constexpr (Q8) v[j] = (float)x.q[i + j] * step_of(x.scale[(i + j) / kBlock8]);
      else v[j] = (float)x.x[i + j];
      d[j] = (float)dy[i + j];
    }
  }
}

template <int V>
struct Coefs {
  float mu[V], a[V], b[V];
  __device__ __forceinline__ Coefs(const Walk& w, const Place& p, const Affine& f) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c0 = p.channel + j, c = c0 < w.C ? c0 : c0 % w.C, g = p.n * w.G + c / w.D;
      mu[j] = f.mean[g];
      a[j] = f.rstd[g] * load_param(f.weight, f.type, c, 1.0f);
      b[j] = load_param(f.bias, f.type, c, 0.0f);
    }
  }
};

// With g = dy act'(z): per (sample, part, position of a row) sum g and sum g xhat, and per (sample,
// part, tile, group) sum weight g and sum weight g xhat.  Bound by memory: 16 x 64 x 240 x 320 bf16 53.6 us,
// 5.9 TB/s; from a checkpoint, 8 x 64 x 240 x 320 fp32 41.2 us, 4.8.
template <typename T, int ACT, bool Q8>
__global__ __launch_bounds__(kThreads) void gn_grad_sums_kernel(const T* __restrict__ dy, Source<T, Q8> x, Walk w,
                                                                Affine f, float2* __restrict__ pos_out,
                                                                float2* __restrict__ rec) {
  constexpr int V = Vec<T>::V;
  __shared__ float s_1[kThreads * V], s_2[kThreads * V];
  const Place p(w, V, blockIdx.x);
  const int step = w.RS * w.Cv;
  int b = p.part;
  Pair<T, Q8> h[kDeepSums];
  Block blk(w, p, b, kDeepSums, V);
  auto load = [&](int u) { h[u].load(x, dy, blk.at + (int64_t)u * step, p.off); };
#pragma unroll
  for (int u = 0; u < kDeepSums; ++u)
    if (u < blk.whole) load(u);
  const Coefs<V> k(w, p, f);
  float s1[V] = {}, s2[V] = {};
  auto add = [&](const float(&v)[V], const float(&d)[V], int m) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float xc = j < m ? v[j] - k.mu[j] : 0.0f, g = d[j] * act_slope<ACT>(fmaf(xc, k.a[j], k.b[j]));  // d is 0 behind m
      s1[j] += g;
      s2[j] = fmaf(g, xc, s2[j]);
    }
  };
  // whole blocks, the next one's loads issued as the vectors of this one are used
#pragma unroll 1
  while (b < w.blocks && blk.whole == kDeepSums) {
    b += w.parts;
    const bool more = b < w.blocks;
    if (more) blk = Block(w, p, b, kDeepSums, V);
    const bool whole = more && blk.whole == kDeepSums;
#pragma unroll
    for (int u = 0; u < kDeepSums; ++u) {
      float v[V], d[V];
      h[u].get(x, v, d);
      if (whole) load(u);
      add(v, d, V);
    }
    if (more && !whole) {
#pragma unroll
      for (int u = 0; u < kDeepSums - 1; ++u)
        if (u < blk.whole) load(u);
    }
  }
  if (b < w.blocks) {  // the sample's last block
    float v[V], d[V];
    first_values(x, dy, blk.at + (int64_t)blk.whole * step + p.off, blk.tail, v, d);
    add(v, d, blk.tail);
#pragma unroll
    for (int u = 0; u < kDeepSums - 1; ++u)
      if (u < blk.whole) {
        h[u].get(x, v, d);
        add(v, d, V);
      }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    s_1[threadIdx.x * V + j] = p.active ? s1[j] : 0.0f;
    s_2[threadIdx.x * V + j] = p.active ? s2[j] : 0.0f;
  }
  __syncthreads();
  const int PW = w.W * V;
  {
    const int P = sharers(PW), pl = threadIdx.x & (P - 1);
#pragma unroll 1
    for (int i = threadIdx.x / P; i < PW; i += kThreads / P) {
      float t1 = 0.0f, t2 = 0.0f;
#pragma unroll 4
      for (int r = pl; r < w.RS; r += P) {
        t1 += s_1[r * PW + i];
        t2 += s_2[r * PW + i];
      }
      t1 = lanes_sum(t1, P);
      t2 = lanes_sum(t2, P);
      const int pos = p.tile * PW + i;
      if (pl == 0 && pos < w.Cv) {
        const int c = pos % w.C;
        t2 *= f.rstd[p.n * w.G + c / w.D];
        pos_out[(int64_t)(p.n * w.parts + p.part) * w.Cv + pos] = make_float2(t1, t2);
        const float wt = load_param(f.weight, f.type, c, 1.0f);
        s_1[i] = wt * t1;  // row 0's place, which only these lanes have read
        s_2[i] = wt * t2;
      }
    }
  }
  __syncthreads();
  const int Q = sharers(w.G), lane = threadIdx.x & (Q - 1);
  rec += ((int64_t)(p.n * w.parts + p.part) * w.tiles + p.tile) * w.G;
  const int lo = p.tile * PW, hi = min(lo + PW, w.Cv);
#pragma unroll 1
  for (int g = threadIdx.x / Q; g < w.G; g += kThreads / Q) {
    float m1 = 0.0f, m2 = 0.0f;
#pragma unroll 1
    for (int c = g * w.D; c < hi; c += w.C)
#pragma unroll 1
      for (int i = max(c, lo) + lane; i < min(c + w.D, hi); i += Q) {
        m1 += s_1[i - lo];
        m2 += s_2[i - lo];
      }
    m1 = lanes_sum(m1, Q);
    m2 = lanes_sum(m2, Q);
    if (lane == 0) rec[g] = make_float2(m1, m2);
  }
}

// rstd E[weight g] and rstd^2 E[weight g xhat] of sample n's group g, by Q lanes as join_stats.
__device__ __forceinline__ float2 join_grads(const float2* rec, int R, const Walk& w, const Affine& f, int n, int g,
                                             int lane, int Q) {
  const float2* r = rec + (int64_t)n * R * w.G + g;
  double m1 = 0.0, m2 = 0.0;
#pragma unroll 4
  for (int i = lane; i < R; i += Q) {
    const float2 a = r[(int64_t)i * w.G];
    m1 += a.x;
    m2 += a.y;
  }
  const double rs = f.rstd[n * w.G + g], each = rs / (double)(w.L / w.G);
  return make_float2((float)(each * lanes_sum(m1, Q)), (float)(each * rs * lanes_sum(m2, Q)));
}
__global__ __launch_bounds__(kThreads) void gn_finish_grads_kernel(const float2* __restrict__ rec, int R, Walk w,
                                                                   Affine f, float2* __restrict__ means) {
  const int lane = threadIdx.x & 63;
#pragma unroll 1
  for (int64_t i = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6); i < (int64_t)w.N * w.G; i += (int64_t)gridDim.x * kWaves) {
    const int n = (int)(i / w.G), g = (int)(i - (int64_t)n * w.G);
    const float2 r = join_grads(rec, R, w, f, n, g, lane, 64);
    if (lane == 0) means[i] = r;
  }
}

// dweight and dbias from `rows` rows of (sum g, sum g xhat) per channel: 8 channels a workgroup, the
// rows dealt to 32 threads each and joined in a fixed order in fp64.
constexpr int kGradCh = 8;
__device__ __forceinline__ void param_grads(const float2* __restrict__ pos, int64_t rows, int C, int type, void* dweight,
                                            void* dbias, int block) {
  constexpr int R = kThreads / kGradCh;
  __shared__ double s_1[R][kGradCh], s_2[R][kGradCh];
  const int k = threadIdx.x % kGradCh, r = threadIdx.x / kGradCh, c = block * kGradCh + k;
  double s1 = 0.0, s2 = 0.0;
  if (c < C)
#pragma unroll 4
    for (int64_t i = r; i < rows; i += R) {
      const float2 a = pos[i * C + c];
      s1 += a.x;
      s2 += a.y;
    }
  s_1[r][k] = s1;
  s_2[r][k] = s2;
  __syncthreads();
  if (r == 0 && c < C) {
    s1 = s2 = 0.0;
    for (int i = 0; i < R; ++i) {
      s1 += s_1[i][k];
      s2 += s_2[i][k];
    }
    if (dbias) store_param(dbias, type, c, (float)s1);
    if (dweight) store_param(dweight, type, c, (float)s2);
  }
}

struct Params {  // of the parameters' gradients: the first `blocks` workgroups compute them
  const float2* pos;
  int64_t rows;
  void *dweight, *dbias;
  int32_t blocks;
};

__global__ __launch_bounds__(kThreads) void gn_param_grads_kernel(Params pg, int C, int type) {
  param_grads(pg.pos, pg.rows, C, type, pg.dweight, pg.dbias, blockIdx.x);
}

// dx = a g - rstd E[weight g] - (x - mean) rstd^2 E[weight g xhat], a = rstd * weight.  Bound by memory:
// 16 x 64 x 240 x 320 bf16 79.6 us, 5.9 TB/s; from a checkpoint, 8 x 64 x 240 x 320 fp32 59.8 us, 5.9.
template <typename T, int ACT, bool Q8>
__global__ __launch_bounds__(kThreads) void gn_grad_input_kernel(const T* __restrict__ dy, Source<T, Q8> x, Walk w,
                                                                 Affine f, Params pg, const float2* __restrict__ rec,
                                                                 int R, const float2* __restrict__ means,
                                                                 T* __restrict__ dx) {
  constexpr int V = Vec<T>::V;
  __shared__ float s_m1[kFold], s_m2[kFold];
  if ((int)blockIdx.x < pg.blocks) {
    param_grads(pg.pos, pg.rows, w.C, f.type, pg.dweight, pg.dbias, blockIdx.x);
    return;
  }
  const Place p(w, V, blockIdx.x - pg.blocks);
  const int step = w.RS * w.Cv;
  int b = w.blocks - 1 - p.part;  // backwards and ahead, as gn_apply_kernel
  Pair<T, Q8> h[kDeepGrad];
  Block blk(w, p, b, kDeepGrad, V);
  auto load = [&](int u) { h[u].load(x, dy, blk.at + (int64_t)u * step, p.off); };
#pragma unroll
  for (int u = 0; u < kDeepGrad; ++u)
    if (u < blk.whole) load(u);
  const Coefs<V> k(w, p, f);
  if (rec) {
    const int Q = sharers(w.G), lane = threadIdx.x & (Q - 1);
#pragma unroll 1
    for (int g = threadIdx.x / Q; g < w.G; g += kThreads / Q) {
      const float2 r = join_grads(rec, R, w, f, p.n, g, lane, Q);
      if (lane == 0) {
        s_m1[g] = r.x;
        s_m2[g] = r.y;
      }
    }
    __syncthreads();
  }
  float m1[V], m2[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c0 = p.channel + j, g = (c0 < w.C ? c0 : c0 % w.C) / w.D;
    m1[j] = rec ? s_m1[g] : means[p.n * w.G + g].x;
    m2[j] = rec ? s_m2[g] : means[p.n * w.G + g].y;
  }
  auto grad = [&](float(&v)[V], const float(&d)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float xc = v[j] - k.mu[j], g = d[j] * act_slope<ACT>(fmaf(xc, k.a[j], k.b[j]));
      v[j] = fmaf(-xc, m2[j], fmaf(k.a[j], g, -m1[j]));
    }
  };
  if (blk.whole < kDeepGrad) {  // the sample's last block
    float v[V], d[V];
#pragma unroll
    for (int u = 0; u < kDeepGrad - 1; ++u)
      if (u < blk.whole) {
        h[u].get(x, v, d);
        grad(v, d);
        if (p.active) store_vec(at(dx + blk.at + (int64_t)u * step, p.off), v);
      }
    const int64_t i = blk.at + (int64_t)blk.whole * step + p.off;
    first_values(x, dy, i, blk.tail, v, d);
    grad(v, d);
    if (p.active) store_first(dx + i, v, blk.tail);
    b -= w.parts;
    if (b < 0) return;
    blk = Block(w, p, b, kDeepGrad, V);
#pragma unroll
    for (int u = 0; u < kDeepGrad; ++u) load(u);
  }
#pragma unroll 1
  for (;;) {
    T* out = dx + blk.at;
    b -= w.parts;
    const bool more = b >= 0;
    if (more) blk = Block(w, p, b, kDeepGrad, V);
#pragma unroll
    for (int u = 0; u < kDeepGrad; ++u, out += step) {
      float v[V], d[V];
      h[u].get(x, v, d);
      if (more) load(u);
      grad(v, d);
      if (p.active) store_vec(at(out, p.off), v);
    }
    if (!more) break;
  }
}

// The backward of gn_small_kernel.  pos [N][C]: (sum g, sum g xhat); with one sample, dweight and dbias.
template <typename T, int ACT, bool Q8>
__global__ __launch_bounds__(kSmall) void gn_small_grad_kernel(const T* __restrict__ dy, Source<T, Q8> x, Slice w, Affine f,
                                                               float2* __restrict__ pos, void* dweight, void* dbias,
                                                               T* __restrict__ dx) {
  constexpr int V = Vec<T>::V;
  __shared__ float s_1[kSmall * V], s_2[kSmall * V], s_m1[kSmall], s_m2[kSmall];
  const SliceSpot p(w, V);
  const int64_t base = (int64_t)p.n * w.P * w.C + p.c0;
  const uint32_t off = (p.active ? p.rr * w.C : 0) + (p.active ? p.slot * V : 0);
  const int64_t step = (int64_t)w.RS * w.C;
  Pair<T, Q8> h[kSmallHold / 2];
#pragma unroll
  for (int i = 0; i < kSmallHold / 2; ++i)
    if (i < w.nv && p.active && p.rr + (int64_t)i * w.RS < w.P) h[i].load(x, dy, base + i * step, off);
  const int g0 = p.n * w.G + (p.active ? p.c : p.c0) / w.D;
  const float mu = f.mean[g0], rs = f.rstd[g0];
  float a[V], b[V], s1[V] = {}, s2[V] = {};
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = p.active ? p.c + j : p.c0;
    a[j] = rs * load_param(f.weight, f.type, c, 1.0f);
    b[j] = load_param(f.bias, f.type, c, 0.0f);
  }
#pragma unroll
  for (int i = 0; i < kSmallHold / 2; ++i)
    if (i < w.nv && p.active && p.rr + (int64_t)i * w.RS < w.P) {
      float v[V], d[V];
      h[i].get(x, v, d);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float xc = v[j] - mu, g = d[j] * act_slope<ACT>(fmaf(xc, a[j], b[j]));
        s1[j] += g;
        s2[j] = fmaf(g, xc, s2[j]);
      }
    }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    s_1[threadIdx.x * V + j] = s1[j];
    s_2[threadIdx.x * V + j] = s2[j];
  }
  __syncthreads();
  {
    const int L = sharers(w.cw, kSmall), lane = threadIdx.x & (L - 1);
#pragma unroll 1
    for (int i = threadIdx.x / L; i < w.cw; i += kSmall / L) {
      float t1 = 0.0f, t2 = 0.0f;
#pragma unroll 4
      for (int r = lane; r < w.RS; r += L) {
        t1 += s_1[r * w.cw + i];
        t2 += s_2[r * w.cw + i];
      }
      t1 = lanes_sum(t1, L);
      t2 = lanes_sum(t2, L);
      if (lane == 0) {
        const int c = p.c0 + i;
        t2 *= f.rstd[p.n * w.G + c / w.D];
        if (pos) {
          pos[(int64_t)p.n * w.C + c] = make_float2(t1, t2);
        } else {
          if (dbias) store_param(dbias, f.type, c, t1);
          if (dweight) store_param(dweight, f.type, c, t2);
        }
        const float wt = load_param(f.weight, f.type, c, 1.0f);
        s_1[i] = wt * t1;  // row 0's place, which only these lanes have read
        s_2[i] = wt * t2;
      }
    }
  }
  if (!dx) return;
  __syncthreads();
  {
    const int gw = w.cw / w.D, Q = sharers(gw, kSmall), lane = threadIdx.x & (Q - 1);
#pragma unroll 1
    for (int g = threadIdx.x / Q; g < gw; g += kSmall / Q) {
      float m1 = 0.0f, m2 = 0.0f;
#pragma unroll 1
      for (int i = g * w.D + lane; i < (g + 1) * w.D; i += Q) {
        m1 += s_1[i];
        m2 += s_2[i];
      }
      m1 = lanes_sum(m1, Q);
      m2 = lanes_sum(m2, Q);
      if (lane == 0) {
        const float r = f.rstd[p.n * w.G + p.c0 / w.D + g], each = r / (float)(w.P * w.D);
        s_m1[g] = each * m1;
        s_m2[g] = each * r * m2;
      }
    }
  }
  __syncthreads();
  const int gl = p.active ? (p.c - p.c0) / w.D : 0;
  const float m1 = s_m1[gl], m2 = s_m2[gl];
#pragma unroll
  for (int i = 0; i < kSmallHold / 2; ++i)
    if (i < w.nv && p.active && p.rr + (int64_t)i * w.RS < w.P) {
      float v[V], d[V];
      h[i].get(x, v, d);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float xc = v[j] - mu, g = d[j] * act_slope<ACT>(fmaf(xc, a[j], b[j]));
        v[j] = fmaf(-xc, m2, fmaf(a[j], g, -m1));
      }
      store_vec(at(dx + base + i * step, off), v);
    }
}

// ------------------------------------------------------------------ host side
// Workgroups of the statistics and of the gradients' sums, whose records the others join, and of those
// that write.  (Forward passes in all.  Statistics, 8 x 32 x 480 x 640 fp32: 512 168 us, 1024 175, 2048
// 186; apply, 8 x 64 x 240 x 320 bf16: 1024 55.7 us, 4096 67.2.  Both that write, forward and backward, 16 x
// 64 x 240 x 320 bf16: 1024 228.7 us, 1280 224.8, which all fit at once.)
constexpr int kStatsWorkgroups = 512, kSumsWorkgroups = 512, kApplyWorkgroups = 1280, kGradWorkgroups = 1280;

// Slots of a tile where the result is in the channel-quad layout, in which a slot's pixels lie side by side and
// slots a plane apart: 32 pixels a workgroup, 512 bytes in a row (3 x 512 x 62 x 314: a whole row's 128 slots
// and 2 pixels 356 us, 16 slots 90, 8 slots 85; 8 x 32 x 240 x 320, of 8 slots, 47 either way).
constexpr int kPackedSlots = 8;

int check(const DpftGroupNorm* d) {
  if (!d) return dpft_fail(DPFT_E_INVALID, "null descriptor");
  if (d->N < 1 || d->C < 1 || d->pixels < 1 || d->groups < 1)
    return dpft_fail(DPFT_E_INVALID, "bad shape N=%d C=%d pixels=%lld groups=%d", d->N, d->C, (long long)d->pixels,
                     d->groups);
  if (d->C % d->groups) return dpft_fail(DPFT_E_INVALID, "groups=%d does not divide C=%d", d->groups, d->C);
  if (d->C > (1 << 20) || d->pixels > (int64_t(1) << 40) / d->C || d->N > (1 << 20) ||
      (int64_t)d->N * (d->C / kThreads + 1) > (1 << 20) || (int64_t)d->N * d->C > (1 << 30))
    return dpft_fail(DPFT_E_INVALID, "too large: N=%d C=%d pixels=%lld", d->N, d->C, (long long)d->pixels);
  if (d->act < DPFT_ACT_NONE || d->act > DPFT_ACT_SILU) return dpft_fail(DPFT_E_INVALID, "unknown act %d", d->act);
  if (d->x_type < DPFT_TYPE_F32 || d->x_type > DPFT_TYPE_F16 || d->param_type < DPFT_TYPE_F32 ||
      d->param_type > DPFT_TYPE_F16)
    return dpft_fail(DPFT_E_INVALID, "unknown type (x %d, parameters %d)", d->x_type, d->param_type);
  if (!(d->eps >= 0.0f)) return dpft_fail(DPFT_E_INVALID, "eps must not be negative");
  if (d->flags & ~DPFT_GN_PACKED) return dpft_fail(DPFT_E_INVALID, "unknown flags 0x%x", d->flags);
  if ((d->flags & DPFT_GN_PACKED) && (d->x_type != DPFT_TYPE_F32 || d->C % 4))
    return dpft_fail(DPFT_E_INVALID, "DPFT_GN_PACKED needs fp32 and C %% 4 == 0 (C=%d)", d->C);
  return DPFT_OK;
}

// deep: vectors that a thread visits in a block; slots: of a tile at most.
Walk make_walk(const DpftGroupNorm& d, int deep, int workgroups, int slots = kThreads) {
  Walk w{};
  const int V = d.x_type == DPFT_TYPE_F32 ? 4 : 8;
  w.N = d.N;
  w.C = d.C;
  w.G = d.groups;
  w.D = d.C / d.groups;
  w.L = d.pixels * d.C;
  w.Cv = std::lcm(d.C, V);
  w.S = w.Cv / V;
  w.tiles = (w.S + slots - 1) / slots;
  w.W = (w.S + w.tiles - 1) / w.tiles;
  w.RS = kThreads / w.W;
  const int whole = kBlock8 / std::gcd(w.Cv, kBlock8);  // rows that make whole checkpoint blocks
  if (w.RS >= whole) w.RS -= w.RS % whole;
  w.in_block = w.L % V == 0;
  w.lanes_block = w.tiles == 1 && w.RS % whole == 0 && w.L % kBlock8 == 0;
  w.full = w.L / w.Cv;
  w.rows = (w.L + w.Cv - 1) / w.Cv;
  w.blocks = (int)((w.rows + (int64_t)deep * w.RS - 1) / ((int64_t)deep * w.RS));
  w.parts = (int)std::min<int64_t>(w.blocks, std::max<int64_t>(1, workgroups / ((int64_t)d.N * w.tiles)));
  return w;
}

constexpr int64_t kMaxValues = int64_t(1) << 48;
// Workgroups of the flat kernels for n values, at most 2^20 (a launch holds fewer than 2^32 threads).
unsigned grid_for(int type, int64_t n) {
  const int64_t per = (int64_t)kThreads * kUnroll * (type == DPFT_TYPE_F32 ? 4 : 8);
  return (unsigned)std::min<int64_t>((n + per - 1) / per, int64_t(1) << 20);
}
size_t round256(size_t n) { return (n + 255) / 256 * 256; }
// The small maps' cut, or cw = 0: whole groups of whole vectors, as few as hold 32 channels, whose pixels
// a workgroup can hold.
Slice make_slice(const DpftGroupNorm& d, int hold) {
  Slice w{};
  const int V = d.x_type == DPFT_TYPE_F32 ? 4 : 8, D = d.C / d.groups;
  if (D % V || d.C > (1 << 16)) return w;
  int gw = 1;
  while (gw < d.groups && (gw * D < 32 || d.groups % gw)) ++gw;
  const int cw = gw * D, S = cw / V;
  if (S > kSmall) return w;
  const int RS = kSmall / S;
  if (d.pixels > (int64_t)RS * hold) return w;
  w.P = d.pixels;
  w.C = d.C;
  w.D = D;
  w.G = d.groups;
  w.cw = cw;
  w.S = S;
  w.RS = RS;
  w.nv = (int)((d.pixels + RS - 1) / RS);
  return w;
}

// The workspace: the forward's records, then statistics that nobody asked for; the backward's records,
// positions and, for many groups, means.
size_t record_bytes(const Walk& w, size_t one) { return round256((size_t)w.N * w.parts * w.tiles * w.G * one); }
size_t position_bytes(const Walk& w) { return round256((size_t)w.N * w.parts * w.Cv * sizeof(float2)); }
size_t group_bytes(const Walk& w) { return round256((size_t)w.N * w.G * sizeof(float2)); }
size_t need(const DpftGroupNorm& d) {
  const Walk f = make_walk(d, kDeep, kStatsWorkgroups), b = make_walk(d, kDeepSums, kSumsWorkgroups);
  // (positions: at least a row of C a sample, which is what the small maps' backward needs)
  return std::max(record_bytes(f, sizeof(float4)) + group_bytes(f),
                  record_bytes(b, sizeof(float2)) + position_bytes(b) + group_bytes(b));
}
// The workgroups of the last pass join a sample's records themselves where there are few of them: 3 x 30
// x 61 x 79 bf16, forward and backward 35.1 us, with launches of their own 36.7; 8 x 96 x 120 x 160 fp32
// 93.1 and 94.3.  Each workgroup reads them all, 16 KiB for 1024: one sample of 384 x 16 x 636 fp16 in 16
// groups took 63.7 us with up to 8192, 52.9 so.
bool fold(const Walk& w) { return w.G <= kFold && (int64_t)w.parts * w.tiles * w.G <= 1024; }
unsigned waves_grid(int64_t waves) { return (unsigned)std::min<int64_t>((waves + kWaves - 1) / kWaves, int64_t(1) << 20); }
unsigned walk_grid(const Walk& w) { return (unsigned)(w.N * w.parts * w.tiles); }
bool misaligned(const void* p) { return reinterpret_cast<uintptr_t>(p) & 15; }

template <typename T, int ACT, int MODE>
void launch_forward(const DpftGroupNorm& d, const T* x, Affine f, float* mean_out, float* rstd_out, T* y, int8_t* q,
                    uint8_t* scale, void* ws, hipStream_t st) {
  const Slice sl = make_slice(d, kSmallHold);
  if (sl.cw) {
    hipLaunchKernelGGL((gn_small_kernel<T, ACT, MODE>), dim3((unsigned)(d.N * (d.C / sl.cw))), dim3(kSmall), 0, st, x, sl, f,
                       d.eps, mean_out, rstd_out, y, q, scale);
    return;
  }
  const Walk ws1 = make_walk(d, kDeep, kStatsWorkgroups),
             w = make_walk(d, kDeepApply, kApplyWorkgroups, MODE == kPacked ? kPackedSlots : kThreads);
  const int R = ws1.parts * ws1.tiles;
  const dim3 block(kThreads);
  float4* rec = static_cast<float4*>(ws);
  hipLaunchKernelGGL(gn_stats_kernel<T>, dim3(walk_grid(ws1)), block, 0, st, x, ws1, rec);
  if (!fold(ws1)) {
    float* stats = reinterpret_cast<float*>(static_cast<char*>(ws) + record_bytes(ws1, sizeof(float4)));
    if (!mean_out) mean_out = stats;
    if (!rstd_out) rstd_out = stats + (size_t)d.N * d.groups;
    f.mean = mean_out;
    f.rstd = rstd_out;
    hipLaunchKernelGGL(gn_finish_stats_kernel, dim3(waves_grid((int64_t)d.N * d.groups)), block, 0, st, rec, R, d.N, d.groups,
                       d.eps, mean_out, rstd_out);
    rec = nullptr;
  }
  hipLaunchKernelGGL((gn_apply_kernel<T, ACT, MODE>), dim3(walk_grid(w)), block, 0, st, x, w, f, rec, R, d.eps, mean_out,
                     rstd_out, y, q, scale);
}

template <typename T, int ACT, bool Q8>
void launch_backward(const DpftGroupNorm& d, const T* dy, Source<T, Q8> x, const Affine& f, T* dx, void* dweight,
                     void* dbias, void* ws, hipStream_t st) {
  const Walk ws1 = make_walk(d, kDeepSums, kSumsWorkgroups), w = make_walk(d, kDeepGrad, kGradWorkgroups);
  const int R = ws1.parts * ws1.tiles, param_blocks = dweight || dbias ? (d.C + kGradCh - 1) / kGradCh : 0;
  const dim3 block(kThreads);
  x.in_block = w.in_block;
  float2* rec = static_cast<float2*>(ws);
  const Slice sl = make_slice(d, kSmallHold / 2);
  if (sl.cw) {
    float2* rows = d.N > 1 && param_blocks ? rec : nullptr;
    hipLaunchKernelGGL((gn_small_grad_kernel<T, ACT, Q8>), dim3((unsigned)(d.N * (d.C / sl.cw))), dim3(kSmall), 0, st, dy, x,
                       sl, f, rows, d.N > 1 ? nullptr : dweight, d.N > 1 ? nullptr : dbias, dx);
    if (rows)
      hipLaunchKernelGGL(gn_param_grads_kernel, dim3((unsigned)param_blocks), block, 0, st,
                         Params{rows, d.N, dweight, dbias, param_blocks}, d.C, d.param_type);
    return;
  }
  float2* pos = reinterpret_cast<float2*>(static_cast<char*>(ws) + record_bytes(ws1, sizeof(float2)));
  float2* means = reinterpret_cast<float2*>(reinterpret_cast<char*>(pos) + position_bytes(ws1));
  hipLaunchKernelGGL((gn_grad_sums_kernel<T, ACT, Q8>), dim3(walk_grid(ws1)), block, 0, st, dy, x, ws1, f, pos, rec);
  const Params pg{pos, (int64_t)d.N * ws1.parts * (w.Cv / w.C), dweight, dbias, param_blocks};
  if (dx && !fold(ws1)) {
    hipLaunchKernelGGL(gn_finish_grads_kernel, dim3(waves_grid((int64_t)d.N * d.groups)), block, 0, st, rec, R, w, f, means);
    rec = nullptr;
  }
  if (dx || pg.blocks)
    hipLaunchKernelGGL((gn_grad_input_kernel<T, ACT, Q8>), dim3(pg.blocks + (dx ? walk_grid(w) : 0)), block, 0, st, dy, x,
                       w, f, pg, rec, R, means, dx);
}

// f(type tag, activation constant) for the descriptor's value type and activation.
template <typename F>
void dispatch(int type, int act, F&& f) {
  auto with = [&](auto tag) {
    switch (act) {
      case DPFT_ACT_NONE: f(tag, std::integral_constant<int, DPFT_ACT_NONE>{}); break;
      case DPFT_ACT_RELU: f(tag, std::integral_constant<int, DPFT_ACT_RELU>{}); break;
      case DPFT_ACT_ELU: f(tag, std::integral_constant<int, DPFT_ACT_ELU>{}); break;
      default: f(tag, std::integral_constant<int, DPFT_ACT_SILU>{});
    }
  };
  if (type == DPFT_TYPE_F32) with(float{});
  else if (type == DPFT_TYPE_BF16) with(__bf16{});
  else with(_Float16{});
}
}  // namespace

extern "C" {

size_t dpft_group_norm_workspace_size(const DpftGroupNorm* desc) {
  if (check(desc) != DPFT_OK) return 0;
  return need(*desc);
}

int dpft_group_norm_act(const DpftGroupNorm* desc, const void* x, const void* weight, const void* bias, void* y,
                        float* mean_out, float* rstd_out, int8_t* q_out, uint8_t* scale_out, void* ws, size_t ws_bytes,
                        void* hip_stream) {
  if (const int rc = check(desc)) return rc;
  const DpftGroupNorm& d = *desc;
  if (!x || !y || !ws || x == y) return dpft_fail(DPFT_E_INVALID, "null or aliased pointer");
  if (!mean_out != !rstd_out) return dpft_fail(DPFT_E_INVALID, "the statistics need both mean_out and rstd_out");
  if (!q_out != !scale_out) return dpft_fail(DPFT_E_INVALID, "a checkpoint needs both q_out and scale_out");
  if (q_out && (d.flags & DPFT_GN_PACKED)) return dpft_fail(DPFT_E_INVALID, "no checkpoint with DPFT_GN_PACKED");
  if (misaligned(x) || misaligned(y) || misaligned(ws) || misaligned(q_out) || misaligned(scale_out))
    return dpft_fail(DPFT_E_INVALID, "x, y, the checkpoint and the workspace must be 16-byte aligned");
  const Walk w = make_walk(d, kDeepApply, kApplyWorkgroups);
  const Slice sl = make_slice(d, kSmallHold);
  // written with y where a checkpoint's blocks are whole lanes of a workgroup; else by a pass of its own:
  // y is the same either way
  const bool with_y = q_out && (sl.cw ? sl.cw % kBlock8 == 0 : w.lanes_block != 0);
  if (ws_bytes < need(d)) return dpft_fail(DPFT_E_WORKSPACE, "workspace %zu < %zu", ws_bytes, need(d));
  hipStream_t st = static_cast<hipStream_t>(hip_stream);
  const Affine f{weight, bias, nullptr, nullptr, d.param_type};
  dispatch(d.x_type, d.act, [&](auto tag, auto act) {
    using T = decltype(tag);
    constexpr int A = decltype(act)::value;
    const T* xs = static_cast<const T*>(x);
    T* ys = static_cast<T*>(y);
    if constexpr (sizeof(T) == 4) {
      if (d.flags & DPFT_GN_PACKED)
        return launch_forward<T, A, kPacked>(d, xs, f, mean_out, rstd_out, ys, nullptr, nullptr, ws, st);
    }
    if (with_y)
      launch_forward<T, A, kCheckpoint>(d, xs, f, mean_out, rstd_out, ys, q_out, scale_out, ws, st);
    else
      launch_forward<T, A, kPlain>(d, xs, f, mean_out, rstd_out, ys, nullptr, nullptr, ws, st);
  });
  if (const int rc = dpft_hip_check("gn_apply_kernel")) return rc;
  return q_out && !with_y ? dpft_act_checkpoint(x, d.x_type, d.N * w.L, q_out, scale_out, hip_stream) : DPFT_OK;
}

int dpft_group_norm_act_backward(const DpftGroupNorm* desc, const void* dy, const void* x, const int8_t* q,
                                 const uint8_t* scale, const void* weight, const void* bias, const float* mean,
                                 const float* rstd, void* dx, void* dweight, void* dbias, void* ws, size_t ws_bytes,
                                 void* hip_stream) {
  if (const int rc = check(desc)) return rc;
  const DpftGroupNorm& d = *desc;
  if (d.flags & DPFT_GN_PACKED) return dpft_fail(DPFT_E_INVALID, "the channel-quad layout has no backward");
  if (!dy || !mean || !rstd || !ws || (!x && (!q || !scale)) || (x && (q || scale)))
    return dpft_fail(DPFT_E_INVALID, "null pointer, or not exactly one of x and its checkpoint");
  if (dx && (dx == dy || dx == x)) return dpft_fail(DPFT_E_INVALID, "aliased pointer");
  if (misaligned(dy) || misaligned(x) || misaligned(dx) || misaligned(q) || misaligned(scale) || misaligned(ws))
    return dpft_fail(DPFT_E_INVALID, "dy, x, dx, the checkpoint and the workspace must be 16-byte aligned");
  if (ws_bytes < need(d)) return dpft_fail(DPFT_E_WORKSPACE, "workspace %zu < %zu", ws_bytes, need(d));
  hipStream_t st = static_cast<hipStream_t>(hip_stream);
  const Affine f{weight, bias, mean, rstd, d.param_type};
  dispatch(d.x_type, d.act, [&](auto tag, auto act) {
    using T = decltype(tag);
    constexpr int A = decltype(act)::value;
    const T* g = static_cast<const T*>(dy);
    T* gx = static_cast<T*>(dx);
    if (x)
      launch_backward<T, A, false>(d, g, Source<T, false>{static_cast<const T*>(x), nullptr, nullptr, 0}, f, gx, dweight,
                                   dbias, ws, st);
    else
      launch_backward<T, A, true>(d, g, Source<T, true>{nullptr, q, scale, 0}, f, gx, dweight, dbias, ws, st);
  });
  return dpft_hip_check("gn_grad_input_kernel");
}

int dpft_act_checkpoint(const void* x, int32_t type, int64_t n, int8_t* q, uint8_t* scale, void* hip_stream) {
  if (!x || !q || !scale) return dpft_fail(DPFT_E_INVALID, "null pointer");
  if (type < DPFT_TYPE_F32 || type > DPFT_TYPE_F16) return dpft_fail(DPFT_E_INVALID, "unknown type %d", type);
  if (n < 1 || n > kMaxValues) return dpft_fail(DPFT_E_INVALID, "bad size %lld", (long long)n);
  if (misaligned(x) || misaligned(q) || misaligned(scale))
    return dpft_fail(DPFT_E_INVALID, "x, q and scale must be 16-byte aligned");
  const dim3 grid(grid_for(type, n)), block(kThreads);
  dispatch(type, DPFT_ACT_NONE, [&](auto tag, auto) {
    using T = decltype(tag);
    hipLaunchKernelGGL(act_checkpoint_kernel<T>, grid, block, 0, static_cast<hipStream_t>(hip_stream),
                       static_cast<const T*>(x), n, q, scale);
  });
  return dpft_hip_check("act_checkpoint_kernel");
}

int dpft_act_restore(const int8_t* q, const uint8_t* scale, int64_t n, void* out, int32_t type, void* hip_stream) {
  if (!out || !q || !scale) return dpft_fail(DPFT_E_INVALID, "null pointer");
  if (type < DPFT_TYPE_F32 || type > DPFT_TYPE_F16) return dpft_fail(DPFT_E_INVALID, "unknown type %d", type);
  if (n < 1 || n > kMaxValues) return dpft_fail(DPFT_E_INVALID, "bad size %lld", (long long)n);
  if (misaligned(out) || misaligned(q) || misaligned(scale))
    return dpft_fail(DPFT_E_INVALID, "out, q and scale must be 16-byte aligned");
  const dim3 grid(grid_for(type, n)), block(kThreads);
  dispatch(type, DPFT_ACT_NONE, [&](auto tag, auto) {
    using T = decltype(tag);
    hipLaunchKernelGGL(act_restore_kernel<T>, grid, block, 0, static_cast<hipStream_t>(hip_stream), q, scale, n,
                       static_cast<T*>(out));
  });
  return dpft_hip_check("act_restore_kernel");
}

}  // extern "C"
