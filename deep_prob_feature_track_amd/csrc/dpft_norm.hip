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
// bytes): HBM bound at the large sizes, launch bound at the small ones.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <numeric>

#include "dpft_ic.h"
#include "dpft_internal.h"

namespace {

constexpr int kThreads = 256;
constexpr int kBlock8 = 32;  // values that share a scale in a checkpoint

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));  // a 16-byte access at any value's address

template <typename T>
struct Vec {
  static constexpr int V = 16 / (int)sizeof(T);
  typedef T type __attribute__((ext_vector_type(V)));
};

template <typename T>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[Vec<T>::V]) {
  const auto r = __builtin_bit_cast(typename Vec<T>::type, *reinterpret_cast<const u32x4_any*>(p));
#pragma unroll
  for (int j = 0; j < Vec<T>::V; ++j) v[j] = (float)r[j];
}
// Rounds to T to nearest even: the values' own type.
template <typename T>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[Vec<T>::V]) {
  typename Vec<T>::type r;
#pragma unroll
  for (int j = 0; j < Vec<T>::V; ++j) r[j] = (T)v[j];
  *reinterpret_cast<u32x4_any*>(p) = __builtin_bit_cast(u32x4, r);
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
// expm1 on z <= 0: its Taylor polynomial to z^8 above -1/2 (the next term is 1.4e-8 of the value
// there), exp(z) - 1 below (no cancellation beyond a factor 2.5).
__device__ __forceinline__ float expm1_neg(float z) {
  float q = 1.0f / 40320;
  q = fmaf(q, z, 1.0f / 5040);
  q = fmaf(q, z, 1.0f / 720);
  q = fmaf(q, z, 1.0f / 120);
  q = fmaf(q, z, 1.0f / 24);
  q = fmaf(q, z, 1.0f / 6);
  q = fmaf(q, z, 0.5f);
  return z > -0.5f ? fmaf(z * z, q, z) : __expf(z) - 1.0f;
}
template <int ACT>
__device__ __forceinline__ float act_fwd(float z) {
  if constexpr (ACT == DPFT_ACT_RELU) return z < 0.0f ? 0.0f : z;
  if constexpr (ACT == DPFT_ACT_ELU) return z > 0.0f ? z : expm1_neg(z);
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
// Bound by HBM.
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
struct Walk {
  int64_t L;      // values of a sample
  int64_t rows;   // rows of Cv values, the last one cut short where L % Cv != 0
  int64_t full;   // whole rows
  int64_t rpp;    // rows of a part
  int32_t C, D, G;
  int32_t Cv, S;  // values and 16-byte slots of a row
  int32_t W, tiles;  // slots of a tile (at most kThreads), tiles of a row
  int32_t RS;     // rows that a workgroup visits side by side
  int32_t parts;  // row ranges of a sample, one workgroup (per tile) each
  int32_t in_block;   // a thread's V values lie in one checkpoint block
  int32_t lanes_block;  // ... and the rows that a workgroup visits side by side are whole blocks
};

struct Place {
  int n, part, tile, slot, rr;
  bool active;
  int64_t r, r1;  // the thread's first row, the part's end
};
__device__ __forceinline__ Place place(const Walk& w) {
  Place p;
  const int b = blockIdx.x;
  p.tile = b % w.tiles;
  const int np = b / w.tiles;
  p.n = np / w.parts;
  p.part = np - p.n * w.parts;
  const int t = threadIdx.x;
  p.rr = t / w.W;
  p.slot = p.tile * w.W + (t - p.rr * w.W);
  p.active = p.rr < w.RS && p.slot < w.S;
  p.r = p.part * w.rpp + p.rr;
  p.r1 = min(w.rows, (int64_t)(p.part + 1) * w.rpp);
  return p;
}
// Values of the cut row that fall to `slot`.
__device__ __forceinline__ int tail_values(const Walk& w, int slot, int V) {
  const int64_t left = w.L - w.full * w.Cv - (int64_t)slot * V;
  return (int)max((int64_t)0, min(left, (int64_t)V));
}

// ------------------------------------------------------------------ forward
constexpr int kBatch = 8;  // rows whose mean and spread a thread takes at once

// Per (sample, part, position of a row): count, mean and sum of squares about that mean of the
// part's values.  Each thread takes the exact mean of kBatch values, then their squares about it,
// and joins the batches by the parallel-variance rule: no cancellation, whatever the mean is.
template <typename T>
__global__ __launch_bounds__(kThreads) void gn_stats_kernel(const T* __restrict__ x, Walk w, float4* __restrict__ part) {
  constexpr int V = Vec<T>::V;
  __shared__ float s_mean[kThreads * V], s_m2[kThreads * V], s_cnt[kThreads * V];
  const Place p = place(w);
  float mean[V] = {}, m2[V] = {};
  int cnt = 0, tail = 0;
  if (p.active) {
    const T* base = x + p.n * w.L + (int64_t)p.slot * V;
    int64_t r = p.r;
    const int64_t rf = min(p.r1, w.full);
    int k = 0;
    for (; r + (kBatch - 1) * w.RS < rf; r += kBatch * w.RS, ++k) {
      float v[kBatch][V];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) load_vec(base + (r + u * w.RS) * w.Cv, v[u]);
      const float f = __builtin_amdgcn_rcpf((float)(k + 1));
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float s = 0.0f, q = 0.0f;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) s += v[u][j];
        const float mu = s * (1.0f / kBatch);
#pragma unroll
        for (int u = 0; u < kBatch; ++u) q = fmaf(v[u][j] - mu, v[u][j] - mu, q);
        const float d = mu - mean[j];
        mean[j] = fmaf(d, f, mean[j]);
        m2[j] += fmaf(d * d, (float)(k * kBatch) * f, q);
      }
    }
    cnt = k * kBatch;
    for (; r < rf; r += w.RS) {
      float v[V];
      load_vec(base + r * w.Cv, v);
      const float f = 1.0f / (float)++cnt;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = v[j] - mean[j];
        mean[j] = fmaf(d, f, mean[j]);
        m2[j] = fmaf(d, v[j] - mean[j], m2[j]);
      }
    }
    if (r == w.full && r < p.r1) {
      tail = tail_values(w, p.slot, V);
      const float f = 1.0f / (float)(cnt + 1);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < tail) {
          const float v = (float)base[r * w.Cv + j];
          const float d = v - mean[j];
          mean[j] = fmaf(d, f, mean[j]);
          m2[j] = fmaf(d, v - mean[j], m2[j]);
        }
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    s_mean[threadIdx.x * V + j] = mean[j];
    s_m2[threadIdx.x * V + j] = m2[j];
    s_cnt[threadIdx.x * V + j] = (float)(cnt + (j < tail));
  }
  __syncthreads();
  const int PW = w.W * V;  // positions of a tile; thread (rr, slot)'s values are at rr * PW + slot * V
  for (int i = threadIdx.x; i < PW; i += kThreads) {
    const int pos = p.tile * PW + i;
    if (pos >= w.Cv) break;
    float c = 0.0f, s = 0.0f;
    for (int a = 0; a < w.RS; ++a) {
      c += s_cnt[a * PW + i];
      s = fmaf(s_cnt[a * PW + i], s_mean[a * PW + i], s);
    }
    const float mu = c > 0.0f ? s / c : 0.0f;
    float q = 0.0f;
    for (int a = 0; a < w.RS; ++a) {
      const float d = s_mean[a * PW + i] - mu;
      q += fmaf(s_cnt[a * PW + i] * d, d, s_m2[a * PW + i]);
    }
    part[((int64_t)p.n * w.parts + p.part) * w.Cv + pos] = make_float4(mu, q, c, 0.0f);
  }
}

__device__ __forceinline__ double block_sum(double v, double* s) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0;
  for (int i = 0; i < kThreads / 64; ++i) v += s[i];
  return v;
}

// One workgroup per (sample, group): the parts joined in fp64, in a fixed order.
__global__ __launch_bounds__(kThreads) void gn_finish_stats_kernel(const float4* __restrict__ part, Walk w, float eps,
                                                                   float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ double s_red[kThreads / 64];
  const int n = blockIdx.x / w.G, g = blockIdx.x - n * w.G;
  const int KD = w.Cv / w.G;
  const float4* src = part + (int64_t)n * w.parts * w.Cv;
  const int64_t total = (int64_t)w.parts * KD;
  auto at = [&](int64_t e) {
    const int64_t pt = e / KD;
    const int i = (int)(e - pt * KD), k = i / w.D;
    return src[pt * w.Cv + k * w.C + g * w.D + (i - k * w.D)];
  };
  double c = 0.0, s = 0.0;
  for (int64_t e = threadIdx.x; e < total; e += kThreads) {
    const float4 a = at(e);
    c += a.z;
    s += (double)a.z * a.x;
  }
  c = block_sum(c, s_red);
  const double mu = block_sum(s, s_red) / c;
  double q = 0.0;
  for (int64_t e = threadIdx.x; e < total; e += kThreads) {
    const float4 a = at(e);
    const double d = a.x - mu;
    q += a.y + a.z * d * d;
  }
  q = block_sum(q, s_red);
  if (threadIdx.x == 0) {
    mean[blockIdx.x] = (float)mu;
    rstd[blockIdx.x] = (float)(1.0 / sqrt(q / c + (double)eps));
  }
}

struct Affine {
  const void *weight, *bias;
  const float *mean, *rstd;
  int32_t type;
};

// y = act((x - mean) a + bias), a = rstd * weight.
// MODE: y as x is stored, in the channel-quad layout, or with x's checkpoint (w.lanes_block).
enum { kPlain, kPacked, kCheckpoint };
template <typename T, int ACT, int MODE>
__global__ __launch_bounds__(kThreads) void gn_apply_kernel(const T* __restrict__ x, Walk w, Affine f,
                                                            T* __restrict__ y, int8_t* __restrict__ q,
                                                            uint8_t* __restrict__ scale) {
  constexpr int V = Vec<T>::V;
  const Place p = place(w);
  if (!p.active) return;
  float mu[V], a[V], b[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = (p.slot * V + j) % w.C, g = p.n * w.G + c / w.D;
    mu[j] = f.mean[g];
    a[j] = f.rstd[g] * load_param(f.weight, f.type, c, 1.0f);
    b[j] = load_param(f.bias, f.type, c, 0.0f);
  }
  const T* src = x + p.n * w.L + (int64_t)p.slot * V;
  T* dst = y + p.n * w.L + (int64_t)p.slot * V;
  int64_t r = p.r;
  const int64_t rf = min(p.r1, w.full);
  for (; r < rf; r += w.RS) {
    float v[V];
    load_vec(src + r * w.Cv, v);
    if constexpr (MODE == kCheckpoint) {
      const int64_t i = p.n * w.L + r * w.Cv + (int64_t)p.slot * V;
      int sc;
      *reinterpret_cast<typename Bytes<V>::type*>(q + i) = quantise_vec<V>(v, sc);
      if (i % kBlock8 == 0) scale[i / kBlock8] = (uint8_t)sc;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = act_fwd<ACT>(fmaf(v[j] - mu[j], a[j], b[j]));
    if constexpr (MODE == kPacked) store_vec(y + p.n * w.L + (p.slot * w.rows + r) * V, v);
    else store_vec(dst + r * w.Cv, v);
  }
  if (r == w.full && r < p.r1) {
    const int tail = tail_values(w, p.slot, V);
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < tail) dst[r * w.Cv + j] = (T)act_fwd<ACT>(fmaf((float)src[r * w.Cv + j] - mu[j], a[j], b[j]));
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
  __device__ __forceinline__ float one(int64_t i) const {
    if constexpr (Q8) return (float)q[i] * step_of(scale[i / kBlock8]);
    else return (float)x[i];
  }
  __device__ __forceinline__ void vec(int64_t i, float (&v)[Vec<T>::V]) const {
    if constexpr (Q8) {
      constexpr int V = Vec<T>::V;
      if (in_block) {
        restore_vec<V>(*reinterpret_cast<const typename Bytes<V>::type*>(q + i), step_of(scale[i / kBlock8]), v);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = one(i + j);
      }
    } else {
      load_vec(x + i, v);
    }
  }
};

// Per (sample, part, position): sum g and sum g (x - mean), g = dy act'(z).
template <typename T, int ACT, bool Q8>
__global__ __launch_bounds__(kThreads) void gn_grad_sums_kernel(const T* __restrict__ dy, Source<T, Q8> x, Walk w,
                                                                Affine f, float2* __restrict__ part) {
  constexpr int V = Vec<T>::V;
  __shared__ float s_1[kThreads * V], s_2[kThreads * V];
  const Place p = place(w);
  float s1[V] = {}, s2[V] = {};
  if (p.active) {
    float mu[V], a[V], b[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (p.slot * V + j) % w.C, g = p.n * w.G + c / w.D;
      mu[j] = f.mean[g];
      a[j] = f.rstd[g] * load_param(f.weight, f.type, c, 1.0f);
      b[j] = load_param(f.bias, f.type, c, 0.0f);
    }
    const int64_t base = p.n * w.L + (int64_t)p.slot * V;
    int64_t r = p.r;
    const int64_t rf = min(p.r1, w.full);
    for (; r < rf; r += w.RS) {
      float v[V], d[V];
      x.vec(base + r * w.Cv, v);
      load_vec(dy + base + r * w.Cv, d);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float xc = v[j] - mu[j], g = d[j] * act_slope<ACT>(fmaf(xc, a[j], b[j]));
        s1[j] += g;
        s2[j] = fmaf(g, xc, s2[j]);
      }
    }
    if (r == w.full && r < p.r1) {
      const int tail = tail_values(w, p.slot, V);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < tail) {
          const int64_t i = base + r * w.Cv + j;
          const float xc = x.one(i) - mu[j], g = (float)dy[i] * act_slope<ACT>(fmaf(xc, a[j], b[j]));
          s1[j] += g;
          s2[j] = fmaf(g, xc, s2[j]);
        }
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    s_1[threadIdx.x * V + j] = s1[j];
    s_2[threadIdx.x * V + j] = s2[j];
  }
  __syncthreads();
  const int PW = w.W * V;
  for (int i = threadIdx.x; i < PW; i += kThreads) {
    const int pos = p.tile * PW + i;
    if (pos >= w.Cv) break;
    float t1 = 0.0f, t2 = 0.0f;
    for (int k = 0; k < w.RS; ++k) {
      t1 += s_1[k * PW + i];
      t2 += s_2[k * PW + i];
    }
    part[((int64_t)p.n * w.parts + p.part) * w.Cv + pos] = make_float2(t1, t2);
  }
}

// One workgroup per (sample, group): the parts' sums per channel, sums[n][c] = (sum g, sum g xhat),
// and the group's means of weight g and weight g xhat.
__global__ __launch_bounds__(kThreads) void gn_finish_grads_kernel(const float2* __restrict__ part, Walk w, Affine f,
                                                                   float2* __restrict__ sums,
                                                                   float2* __restrict__ means) {
  __shared__ double s_red[kThreads / 64];
  const int n = blockIdx.x / w.G, g = blockIdx.x - n * w.G;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int K = w.Cv / w.C;
  const float2* src = part + (int64_t)n * w.parts * w.Cv;
  const float rs = f.rstd[blockIdx.x];
  double m1 = 0.0, m2 = 0.0;
  for (int d = wave; d < w.D; d += kThreads / 64) {
    const int c = g * w.D + d;
    double s1 = 0.0, s2 = 0.0;
    for (int64_t e = lane; e < (int64_t)w.parts * K; e += 64) {
      const float2 a = src[(e / K) * w.Cv + (int)(e % K) * w.C + c];
      s1 += a.x;
      s2 += a.y;
    }
    for (int o = 32; o > 0; o >>= 1) {
      s1 += __shfl_xor(s1, o);
      s2 += __shfl_xor(s2, o);
    }
    s2 *= rs;
    if (lane == 0) {
      sums[(int64_t)n * w.C + c] = make_float2((float)s1, (float)s2);
      const double wt = load_param(f.weight, f.type, c, 1.0f);
      m1 += wt * s1;
      m2 += wt * s2;
    }
  }
  m1 = block_sum(m1, s_red);
  m2 = block_sum(m2, s_red);
  const double cnt = (double)w.L / w.G;
  if (threadIdx.x == 0) means[blockIdx.x] = make_float2((float)(m1 / cnt), (float)(m2 / cnt));
}

__global__ __launch_bounds__(kThreads) void gn_param_grads_kernel(const float2* __restrict__ sums, int N, int C,
                                                                  int type, void* dweight, void* dbias) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= C) return;
  double s1 = 0.0, s2 = 0.0;
  for (int n = 0; n < N; ++n) {
    const float2 a = sums[(int64_t)n * C + c];
    s1 += a.x;
    s2 += a.y;
  }
  if (dbias) store_param(dbias, type, c, (float)s1);
  if (dweight) store_param(dweight, type, c, (float)s2);
}

// dx = a g - rstd E[weight g] - (x - mean) rstd^2 E[weight g xhat], a = rstd * weight.
template <typename T, int ACT, bool Q8>
__global__ __launch_bounds__(kThreads) void gn_grad_input_kernel(const T* __restrict__ dy, Source<T, Q8> x, Walk w,
                                                                 Affine f, const float2* __restrict__ means,
                                                                 T* __restrict__ dx) {
  constexpr int V = Vec<T>::V;
  const Place p = place(w);
  if (!p.active) return;
  float mu[V], a[V], b[V], m1[V], m2[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = (p.slot * V + j) % w.C, g = p.n * w.G + c / w.D;
    const float rs = f.rstd[g];
    mu[j] = f.mean[g];
    a[j] = rs * load_param(f.weight, f.type, c, 1.0f);
    b[j] = load_param(f.bias, f.type, c, 0.0f);
    m1[j] = rs * means[g].x;
    m2[j] = rs * rs * means[g].y;
  }
  const int64_t base = p.n * w.L + (int64_t)p.slot * V;
  int64_t r = p.r;
  const int64_t rf = min(p.r1, w.full);
  auto grad = [&](int j, float v, float d) {
    const float xc = v - mu[j], g = d * act_slope<ACT>(fmaf(xc, a[j], b[j]));
    return fmaf(-xc, m2[j], fmaf(a[j], g, -m1[j]));
  };
  for (; r < rf; r += w.RS) {
    float v[V], d[V];
    x.vec(base + r * w.Cv, v);
    load_vec(dy + base + r * w.Cv, d);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = grad(j, v[j], d[j]);
    store_vec(dx + base + r * w.Cv, v);
  }
  if (r == w.full && r < p.r1) {
    const int tail = tail_values(w, p.slot, V);
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < tail) {
        const int64_t i = base + r * w.Cv + j;
        dx[i] = (T)grad(j, x.one(i), (float)dy[i]);
      }
  }
}

// ------------------------------------------------------------------ host side
constexpr int kMaxParts = 256, kWorkgroups = 2048;

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

Walk make_walk(const DpftGroupNorm& d) {
  Walk w{};
  const int V = d.x_type == DPFT_TYPE_F32 ? 4 : 8;
  w.C = d.C;
  w.G = d.groups;
  w.D = d.C / d.groups;
  w.L = d.pixels * d.C;
  w.Cv = std::lcm(d.C, V);
  w.S = w.Cv / V;
  w.W = std::min(w.S, kThreads);
  w.tiles = (w.S + w.W - 1) / w.W;
  w.RS = kThreads / w.W;
  const int whole = kBlock8 / std::gcd(w.Cv, kBlock8);  // rows that make whole checkpoint blocks
  if (w.RS >= whole) w.RS -= w.RS % whole;
  w.in_block = w.L % V == 0;
  w.lanes_block = w.tiles == 1 && w.RS % whole == 0 && w.L % kBlock8 == 0;
  w.full = w.L / w.Cv;
  w.rows = (w.L + w.Cv - 1) / w.Cv;
  const int64_t step = (int64_t)kBatch * w.RS;
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(kMaxParts, kWorkgroups / ((int64_t)d.N * w.tiles)));
  w.rpp = ((w.rows + want - 1) / want + step - 1) / step * step;
  w.parts = (int)((w.rows + w.rpp - 1) / w.rpp);
  return w;
}

constexpr int64_t kMaxValues = int64_t(1) << 48;
// Workgroups of the flat kernels for n values, at most 2^20 (a launch holds fewer than 2^32 threads).
unsigned grid_for(int type, int64_t n) {
  const int64_t per = (int64_t)kThreads * kUnroll * (type == DPFT_TYPE_F32 ? 4 : 8);
  return (unsigned)std::min<int64_t>((n + per - 1) / per, int64_t(1) << 20);
}
size_t round256(size_t n) { return (n + 255) / 256 * 256; }
size_t part_bytes(const DpftGroupNorm& d, const Walk& w) {
  return round256((size_t)d.N * w.parts * w.Cv * sizeof(float4));
}
size_t need(const DpftGroupNorm& d, const Walk& w) {
  return part_bytes(d, w) + round256((size_t)d.N * d.C * sizeof(float2)) +
         round256((size_t)d.N * d.groups * sizeof(float2));
}
bool misaligned(const void* p) { return reinterpret_cast<uintptr_t>(p) & 15; }

template <typename T, int ACT>
void launch_forward(const DpftGroupNorm& d, const Walk& w, const void* x, const Affine& f, void* y, int8_t* q,
                    uint8_t* scale, hipStream_t st) {
  const dim3 grid((unsigned)(d.N * w.parts * w.tiles)), block(kThreads);
  const T* xs = static_cast<const T*>(x);
  T* ys = static_cast<T*>(y);
  if constexpr (sizeof(T) == 4) {
    if (d.flags & DPFT_GN_PACKED) {
      hipLaunchKernelGGL((gn_apply_kernel<T, ACT, kPacked>), grid, block, 0, st, xs, w, f, ys, nullptr, nullptr);
      return;
    }
  }
  if (q && w.lanes_block)
    hipLaunchKernelGGL((gn_apply_kernel<T, ACT, kCheckpoint>), grid, block, 0, st, xs, w, f, ys, q, scale);
  else
    hipLaunchKernelGGL((gn_apply_kernel<T, ACT, kPlain>), grid, block, 0, st, xs, w, f, ys, nullptr, nullptr);
}

template <typename T, int ACT, bool Q8>
void launch_backward(const DpftGroupNorm& d, const Walk& w, const void* dy, Source<T, Q8> x, const Affine& f, void* dx,
                     void* dweight, void* dbias, char* ws, hipStream_t st) {
  float2* part = reinterpret_cast<float2*>(ws);
  float2* sums = reinterpret_cast<float2*>(ws + part_bytes(d, w));
  float2* means = reinterpret_cast<float2*>(ws + part_bytes(d, w) + round256((size_t)d.N * d.C * sizeof(float2)));
  const dim3 grid((unsigned)(d.N * w.parts * w.tiles)), block(kThreads);
  const T* g = static_cast<const T*>(dy);
  hipLaunchKernelGGL((gn_grad_sums_kernel<T, ACT, Q8>), grid, block, 0, st, g, x, w, f, part);
  hipLaunchKernelGGL(gn_finish_grads_kernel, dim3((unsigned)(d.N * d.groups)), block, 0, st, part, w, f, sums, means);
  if (dweight || dbias)
    hipLaunchKernelGGL(gn_param_grads_kernel, dim3((unsigned)((d.C + kThreads - 1) / kThreads)), block, 0, st, sums,
                       d.N, d.C, d.param_type, dweight, dbias);
  if (dx)
    hipLaunchKernelGGL((gn_grad_input_kernel<T, ACT, Q8>), grid, block, 0, st, g, x, w, f, means, static_cast<T*>(dx));
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
  return need(*desc, make_walk(*desc));
}

int dpft_group_norm_act(const DpftGroupNorm* desc, const void* x, const void* weight, const void* bias, void* y,
                        float* mean_out, float* rstd_out, int8_t* q_out, uint8_t* scale_out, void* ws, size_t ws_bytes,
                        void* hip_stream) {
  if (const int rc = check(desc)) return rc;
  const DpftGroupNorm& d = *desc;
  if (!x || !y || !ws || x == y) return dpft_fail(DPFT_E_INVALID, "null or aliased pointer");
  if (!q_out != !scale_out) return dpft_fail(DPFT_E_INVALID, "a checkpoint needs both q_out and scale_out");
  if (q_out && (d.flags & DPFT_GN_PACKED)) return dpft_fail(DPFT_E_INVALID, "no checkpoint with DPFT_GN_PACKED");
  if (misaligned(x) || misaligned(y) || misaligned(ws) || misaligned(q_out) || misaligned(scale_out))
    return dpft_fail(DPFT_E_INVALID, "x, y, the checkpoint and the workspace must be 16-byte aligned");
  const Walk w = make_walk(d);
  if (ws_bytes < need(d, w)) return dpft_fail(DPFT_E_WORKSPACE, "workspace %zu < %zu", ws_bytes, need(d, w));
  hipStream_t st = static_cast<hipStream_t>(hip_stream);
  float4* part = static_cast<float4*>(ws);
  float* stats = reinterpret_cast<float*>(static_cast<char*>(ws) + part_bytes(d, w));
  float* mean = mean_out ? mean_out : stats;
  float* rstd = rstd_out ? rstd_out : stats + (size_t)d.N * d.groups;
  const Affine f{weight, bias, mean, rstd, d.param_type};
  dispatch(d.x_type, d.act, [&](auto tag, auto act) {
    using T = decltype(tag);
    hipLaunchKernelGGL(gn_stats_kernel<T>, dim3((unsigned)(d.N * w.parts * w.tiles)), dim3(kThreads), 0, st,
                       static_cast<const T*>(x), w, part);
    hipLaunchKernelGGL(gn_finish_stats_kernel, dim3((unsigned)(d.N * d.groups)), dim3(kThreads), 0, st, part, w, d.eps,
                       mean, rstd);
    launch_forward<T, decltype(act)::value>(d, w, x, f, y, q_out, scale_out, st);
  });
  if (const int rc = dpft_hip_check("gn_apply_kernel")) return rc;
  // blocks that cross a thread's values or a workgroup's rows: a pass of their own
  return q_out && !w.lanes_block ? dpft_act_checkpoint(x, d.x_type, d.N * w.L, q_out, scale_out, hip_stream) : DPFT_OK;
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
  const Walk w = make_walk(d);
  if (ws_bytes < need(d, w)) return dpft_fail(DPFT_E_WORKSPACE, "workspace %zu < %zu", ws_bytes, need(d, w));
  hipStream_t st = static_cast<hipStream_t>(hip_stream);
  const Affine f{weight, bias, mean, rstd, d.param_type};
  dispatch(d.x_type, d.act, [&](auto tag, auto act) {
    using T = decltype(tag);
    constexpr int A = decltype(act)::value;
    if (x)
      launch_backward<T, A, false>(d, w, dy, Source<T, false>{static_cast<const T*>(x), nullptr, nullptr, 0}, f, dx,
                                   dweight, dbias, static_cast<char*>(ws), st);
    else
      launch_backward<T, A, true>(d, w, dy, Source<T, true>{nullptr, q, scale, w.in_block}, f, dx, dweight, dbias,
                                  static_cast<char*>(ws), st);
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
