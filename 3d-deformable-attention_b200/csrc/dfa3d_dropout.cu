// Dropout whose mask is never stored (dfa3d_philox.cuh), alone and at the end of a residual block (sm_100a):
//
//   y = [residual +] keep * act(x) / (1 - p)                      elementwise; act: none or ReLU
//   y = LayerNorm(residual + keep * x / (1 - p))                  rows of up to 1024 columns
//
// with their backward passes, which form the mask again from (seed, site, element).  Every tensor is read once and written once;
// what bounds them is HBM, with the instructions next: a Philox block for four elements is 43 of them, twelve of which are
// 32 x 32 -> 64 bit products at half rate.  An element of a forward without activation costs 18.0 instructions in fp32 and 16.8 in 16 bits, 7.3
// and 6.1 where nothing is dropped.
//
// Measured (HBM copy 6528 GB/s): 40 000 x 512 fp32 with ReLU 28.4 us forward, 39.2 backward (5.8, 6.3 TB/s), 60.6 for both one after
// the other; 184 950 x 256 bf16 35.0 and 34.9 (5.4 TB/s, 33.8 on another device; there 41 before the upper counter word was made one value
// for a CTA and the kept bits were compared in place; four words a thread 35, CTAs that stay and ask one step ahead 36).
// Norm of 40 000 x 256 fp32 23.6 forward, 38.6 backward (5.2, 5.3 TB/s), of 80 000 x 256 bf16 28.3 and 41.6 (4.3, 4.9 TB/s: 30 and
// 40 instructions an element); 900 x 256 fp32 3.2 and 5.5.  Rows loaded into registers instead of one ahead through shared memory:
// 26 and 46, 1024 columns 66 and 138 for 49 and 80; a warp a row of four elements a lane 25 and 56, bf16 39 and 86.
#include <algorithm>
#include <atomic>

#include "dfa3d_launch.h"
#include "dfa3d_philox.cuh"
#include "dfa3d_rowvec.cuh"

namespace dfa3d {
namespace {

constexpr int kThreads = 256;

// Words of elements base + e ... + V - 1, where base is a multiple of a CTA's elements (block_of) and e below these one of 4.
template <int V>
__device__ __forceinline__ void words_from(const DropRule &d, DropKey k, long long base, unsigned e, uint32_t (&words)[V]) {
  if (!d.rng) {
#pragma unroll
    for (int i = 0; i < V; ++i) words[i] = ~0u;
    return;
  }
#pragma unroll
  for (int i = 0; i < V; i += 4) {
    const PhiloxWords w = philox_words(block_of((unsigned long long)base, e + i), d.site, k);
    words[i] = w.x; words[i + 1] = w.y; words[i + 2] = w.z; words[i + 3] = w.w;
  }
}

// ------------------------------------------------------------------------------------------------
// elementwise
// ------------------------------------------------------------------------------------------------
// One element.  A dropped one is 0 whatever it was (NaN and infinity too); a NaN passes the ReLU, as in torch.
template <bool RELU, bool RES>
__device__ __forceinline__ float drop_one(float x, float r, bool kept, float scale) {
  if (RELU) x = x <= 0.f ? 0.f : x;
  if (RES) return kept ? fmaf(x, scale, r) : r;
  return kept ? x * scale : 0.f;
}

// Threads take 16-byte words of every tensor, U of them a CTA width apart, all loads first.  A CTA's elements begin at a multiple of
// 4096 or 2048, so that the upper half of their block numbers is one value.  VEC = false: an address is off the 16-byte grid,
// elements are read and written one by one (same mask, same result).
constexpr int kUnroll = 2;

template <typename T, bool RELU, bool RES, bool VEC>
__global__ void __launch_bounds__(kThreads)
dropout_forward_kernel(const T *x, const T *__restrict__ residual, long long n, DropRule d,
                       T *y) {      // y may be x
  constexpr int V = 16 / sizeof(T), U = kUnroll;
  const DropKey key = drop_key(d);
  const long long base = (long long)blockIdx.x * (kThreads * U * V);
  if (VEC && base + kThreads * U * V <= n) {
    Word<T, V> xw[U], rw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned e = (u * kThreads + threadIdx.x) * V;
      xw[u] = load_once<T, V>(x + base + e);
      if (RES) rw[u] = load_once<T, V>(residual + base + e);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned e = (u * kThreads + threadIdx.x) * V;
      float f[V], r[V] = {};
      widen_word<T, V>(xw[u], f);
      if (RES) widen_word<T, V>(rw[u], r);
      uint32_t words[V];
      words_from<V>(d, key, base, e, words);
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = drop_one<RELU, RES>(f[i], r[i], words[i] > d.last, d.scale);
      store_word<T, V>(y + base + e, f);
    }
    return;
  }
  for (int q = threadIdx.x; q < kThreads * U * V / 4; q += kThreads) {      // the last CTA, or all of them
    const long long at = base + q * 4;
    if (at >= n) return;
    uint32_t words[4];
    words_of<4>(d, key, (unsigned long long)at, words);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + i < n)
        y[at + i] = narrow<T>(drop_one<RELU, RES>(wide(x[at + i]), RES ? wide(residual[at + i]) : 0.f,
                                                  words[i] > d.last, d.scale));
  }
}

// grad_x = keep * [ref > 0 or NaN] * grad_y / (1 - p).  With a ReLU and no residual `ref` is the forward's result, whose zeros
// are the dropped elements too (scale >= 1: no kept positive value becomes 0), and no mask is formed (RNG = false); with a
// residual it is the forward's x.
template <typename T, bool REF, bool RNG, bool VEC>
__global__ void __launch_bounds__(kThreads)
dropout_backward_kernel(const T *__restrict__ grad_y, const T *__restrict__ ref, long long n, DropRule d, T *__restrict__ grad_x) {
  constexpr int V = 16 / sizeof(T), U = kUnroll;
  const DropKey key = RNG ? drop_key(d) : DropKey{0u, 0u};
  auto one = [&](float g, float v, bool kept) { return !kept || (REF && v <= 0.f) ? 0.f : g * d.scale; };
  const long long base = (long long)blockIdx.x * (kThreads * U * V);
  if (VEC && base + kThreads * U * V <= n) {
    Word<T, V> gw[U], vw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned e = (u * kThreads + threadIdx.x) * V;
      gw[u] = load_once<T, V>(grad_y + base + e);
      if (REF) vw[u] = load_once<T, V>(ref + base + e);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned e = (u * kThreads + threadIdx.x) * V;
      float g[V], v[V] = {};
      widen_word<T, V>(gw[u], g);
      if (REF) widen_word<T, V>(vw[u], v);
      uint32_t words[V];
      if (RNG) words_from<V>(d, key, base, e, words);
#pragma unroll
      for (int i = 0; i < V; ++i) g[i] = one(g[i], v[i], !RNG || words[i] > d.last);
      store_word<T, V>(grad_x + base + e, g);
    }
    return;
  }
  for (int q = threadIdx.x; q < kThreads * U * V / 4; q += kThreads) {
    const long long at = base + q * 4;
    if (at >= n) return;
    uint32_t words[4];
    if (RNG) words_of<4>(d, key, (unsigned long long)at, words);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + i < n)
        grad_x[at + i] = narrow<T>(one(wide(grad_y[at + i]), REF ? wide(ref[at + i]) : 0.f, !RNG || words[i] > d.last));
  }
}

// ------------------------------------------------------------------------------------------------
// LayerNorm(residual + dropout(x))
// ------------------------------------------------------------------------------------------------
constexpr int kWarps = 8;
// CTAs of the forward on an SM.  40 000 x 256 fp32: 23.6 us at three, 25.6 at four, 29.1 at five (spills).
constexpr int kForwardResident = 3;
// ... on rows off the grid, whose words and weights stay in registers: 60 000 x 202 fp16 32.6 us at two, 36.5 at three.
constexpr int kOddResident = 2;

// A row's words of V elements.  VEC: V divides E and the tensors are on the grid of such words.  Else a word is four elements that
// share a Philox block, whatever row they are of: a row begins `shift` elements inside of its first word, and elements of its
// neighbours are left out (NaN and all).  A warp's rows lie a multiple of four apart, so that its shift, and with it the columns
// of each lane, stay the same.  Against rows read one element at a time, us forward / backward: 7001 x 202 fp16 6.0 / 10.0 for
// 6.9 / 10.6, 60 000 x 202 fp16 33 / 50 for 46 / 64, 100 000 x 61 bf16 16 / 26 for 44 / 59, 40 000 x 301 bf16 41 / 75 for 112 / 108,
// 30 000 x 511 fp32 65 / 98 for 107 / 113, 20 000 x 1023 79 / 157 for 125 / 141.
struct Odd {
  int E, shift;
  long long total;       // elements of a tensor
  bool wide;             // words of four can be read and written at once
  __device__ __forceinline__ bool inside(int c) const { return (unsigned)c < (unsigned)E; }
};
// A lane's words of NT tensors' rows, as they are stored.
template <typename T, int K, int LANES, int NT>
struct OddRows {
  Word<T, 4> w[NT][K];
  // A lane's words `first`, first + 1, ... of the row that begins `at` elements behind the pointers; nothing if it is not `live`.
  // All loads are under way before the first is used.
  __device__ __forceinline__ void load(const Odd &o, const T *const (&p)[NT], long long at, int lane, bool live, int first = 0) {
    if (!live) return;
    const bool whole = o.wide && at + o.E + 3 <= o.total;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int c = (lane + LANES * (first + j)) * 4 - o.shift;
      if (c < o.E) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if (whole) {
            w[t][j] = load_word<T, 4>(p[t] + at + c);
          } else {
            float f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = o.inside(c + i) ? wide(p[t][at + c + i]) : 0.f;
            w[t][j] = narrow_word<T, 4>(f);
          }
        }
      }
    }
  }
  __device__ __forceinline__ void read(const Odd &o, int j, int t, int c, float (&f)[4]) const {
    widen_word<T, 4>(w[t][j], f);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = o.inside(c + i) ? f[i] : 0.f;
  }
};
template <typename T>
__device__ __forceinline__ void store_odd(const Odd &o, T *p, long long at, int c, const float (&f)[4]) {
  const bool whole = o.wide && c >= 0 && c + 4 <= o.E;
  if (whole) store_word<T, 4>(p + at + c, f);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (!whole && o.inside(c + i)) p[at + c + i] = narrow<T>(f[i]);
}
template <int V>
__device__ __forceinline__ void load_param(const float *p, int c, float (&f)[V]) {
#pragma unroll
  for (int i = 0; i < V; i += 4) {
    const float4 t = __ldg(reinterpret_cast<const float4 *>(p + c + i));
    f[i] = t.x; f[i + 1] = t.y; f[i + 2] = t.z; f[i + 3] = t.w;
  }
}
__device__ __forceinline__ void load_param_odd(const Odd &o, const float *p, int c, float (&f)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = o.inside(c + i) ? __ldg(p + c + i) : 0.f;
}
// All of a lane's, for the rows that it will have.
template <int K, int LANES>
__device__ __forceinline__ void load_params_odd(const Odd &o, const float *p, int lane, float (&f)[K][4]) {
#pragma unroll
  for (int j = 0; j < K; ++j) load_param_odd(o, p, (lane + LANES * j) * 4 - o.shift, f[j]);
}

// Sum over the LANES lanes that share a row.
template <int LANES>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A row's words of NT tensors, asked for one row ahead by asynchronous copies: a thread's own words, so that no barrier is
// needed and the loads of a row take no registers while the row before it is worked on.
template <typename T, int V, int K, int LANES, int NT>
struct RowsAhead {
  static constexpr unsigned kWord = kWarps * 32 * 16, kStage = K * NT * kWord;
  unsigned mine, stage = 0;
  __device__ __forceinline__ explicit RowsAhead(void *ring)
      : mine((unsigned)__cvta_generic_to_shared(ring) + threadIdx.x * 16) {}
  // `at` elements behind the pointers begins the row; nothing if it is not `live`
  __device__ __forceinline__ void ask(const T *const (&p)[NT], long long at, int lane, int E, bool live) {
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int c = (lane + LANES * j) * V;
      if (live && c < E) {
#pragma unroll
        for (int t = 0; t < NT; ++t) copy_async16(mine + stage * kStage + (j * NT + t) * kWord, p[t] + at + c);
      }
    }
    copies_asked();
    stage ^= 1;
  }
  // word j of tensor t of the row that was asked for before the last one
  __device__ __forceinline__ void read(int j, int t, float (&f)[V]) const {
    widen_word<T, V>(read_shared16(mine + stage * kStage + (j * NT + t) * kWord), f);
  }
};

// LANES lanes have a row, 32 / LANES rows a warp at a time: lane l holds the groups of V columns l, l + LANES, ... (K of them, 16
// elements in most widths: enough for the sums over lanes and the loads of weights not to count).  The sum is normalised as it
// stands in 32 bits and is not written: the backward forms it again from the same x and residual, so that storage in 16 bits
// rounds nothing but y.
template <typename T, int V, int K, int LANES, bool VEC>
__global__ void __launch_bounds__(kWarps * 32, K * V > 16 ? 1 : VEC ? kForwardResident : kOddResident)
dropout_add_layer_norm_kernel(const T *__restrict__ x, const T *__restrict__ residual, const float *__restrict__ gamma,
                              const float *__restrict__ beta, long long rows, int E, bool wide_words, DropRule d, float eps,
                              T *__restrict__ y, float *__restrict__ mean_out, float *__restrict__ rstd_out) {
  constexpr int kRowsAtOnce = 32 / LANES;
  extern __shared__ __align__(16) unsigned char ring[];
  const float inv_e = 1.f / (float)E;
  const int lane = threadIdx.x & (LANES - 1), slot = (threadIdx.x & 31) / LANES;
  const long long stride = (long long)gridDim.x * kWarps * kRowsAtOnce;
  long long row = ((long long)blockIdx.x * kWarps + (threadIdx.x >> 5)) * kRowsAtOnce + slot;
  const T *const in[2] = {x, residual};
  RowsAhead<T, V, K, LANES, 2> ahead(ring);
  if constexpr (VEC) ahead.ask(in, row * E, lane, E, row < rows);
  const DropKey key = drop_key(d);
  const Odd odd = {E, VEC ? 0 : (int)(row * E & 3), rows * E, wide_words};
  constexpr bool kAhead = !VEC && K <= 2;
  float gamma_of[VEC ? 1 : K][4], beta_of[VEC ? 1 : K][4];
  if constexpr (!VEC) {
    load_params_odd<K, LANES>(odd, gamma, lane, gamma_of);
    load_params_odd<K, LANES>(odd, beta, lane, beta_of);
  }
  OddRows<T, VEC ? 1 : K, LANES, 2> odd_row, odd_next;
  if constexpr (kAhead) odd_next.load(odd, in, row * E, lane, row < rows);
  for (; row - slot < rows; row += stride) {
    const bool live = row < rows;
    const long long at = row * E;
    if constexpr (VEC) {
      ahead.ask(in, at + stride * E, lane, E, row + stride < rows);
      copies_wait<1>();
    } else if constexpr (kAhead) {
      odd_row = odd_next;
      odd_next.load(odd, in, at + stride * E, lane, row + stride < rows);
    } else {
      odd_row.load(odd, in, at, lane, live);
    }
    float v[K][V];
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int c = (lane + LANES * j) * V - odd.shift;
#pragma unroll
      for (int i = 0; i < V; ++i) v[j][i] = 0.f;
      if (c >= E || !live) continue;
      float xf[V];
      if constexpr (VEC) {
        ahead.read(j, 0, xf);
        ahead.read(j, 1, v[j]);
      } else {
        odd_row.read(odd, j, 0, c, xf);
        odd_row.read(odd, j, 1, c, v[j]);
      }
      uint32_t words[V];
      words_of<V>(d, key, (unsigned long long)(at + c), words);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float sum = fmaf(xf[i], d.scale, v[j][i]);
        v[j][i] = words[i] > d.last ? sum : v[j][i];
        s += v[j][i];
      }
    }
    const float mean = row_sum<LANES>(s) * inv_e;
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int c = (lane + LANES * j) * V - odd.shift;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[j][i] -= mean;
        const float t = (VEC ? c < E : odd.inside(c + i)) ? v[j][i] : 0.f;
        q = fmaf(t, t, q);
      }
    }
    const float rstd = rsqrtf(row_sum<LANES>(q) * inv_e + eps);
    if (!live) continue;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int c = (lane + LANES * j) * V - odd.shift;
      if (c >= E) continue;
      if constexpr (VEC) {
        float g[V], b[V];
        load_param<V>(gamma, c, g);
        load_param<V>(beta, c, b);
#pragma unroll
        for (int i = 0; i < V; ++i) g[i] = fmaf(v[j][i] * rstd, g[i], b[i]);
        store_word<T, V>(y + at + c, g);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[j][i] = fmaf(v[j][i] * rstd, gamma_of[j][i], beta_of[j][i]);
        store_odd<T>(odd, y, at, c, v[j]);
      }
    }
    if (lane == 0 && mean_out) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
  }
  copies_wait<0>();
}

__device__ __forceinline__ void launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void launch_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// grad_residual = rstd * (d - mean(d) - xhat * mean(d * xhat)) with d = grad_y * gamma; grad_x = keep * grad_residual / (1 - p).
// grad_gamma (sum of grad_y * xhat) and grad_beta (sum of grad_y) are summed over a lane's rows in registers, over the CTA in
// shared memory, and written as the CTA's own row of `partial` (ctas, 2, E): the second kernel adds these up in a fixed order, so
// that a gradient is the same bits in every run.
template <typename T, int V, int K, int LANES, bool VEC>
__global__ void __launch_bounds__(kWarps * 32)
dropout_layer_norm_backward_kernel(const T *__restrict__ grad_y, const T *__restrict__ x, const T *__restrict__ residual,
                                   const float *__restrict__ gamma, const float *__restrict__ mean_in,
                                   const float *__restrict__ rstd_in, long long rows, int E, bool wide_words, DropRule d,
                                   T *__restrict__ grad_x,
                                   T *__restrict__ grad_residual, float *__restrict__ partial) {
  constexpr int kRowsAtOnce = 32 / LANES, kSlots = kWarps * kRowsAtOnce;
  extern __shared__ __align__(16) unsigned char ring[];
  launch_next();
  const float inv_e = 1.f / (float)E;
  const int lane = threadIdx.x & (LANES - 1), slot = (threadIdx.x & 31) / LANES, warp = threadIdx.x >> 5;
  const long long stride = (long long)gridDim.x * kSlots;
  long long row = ((long long)blockIdx.x * kWarps + warp) * kRowsAtOnce + slot;
  const T *const in[3] = {grad_y, x, residual};
  RowsAhead<T, V, K, LANES, 3> ahead(ring);
  if constexpr (VEC) ahead.ask(in, row * E, lane, E, row < rows);
  const DropKey key = drop_key(d);
  const Odd odd = {E, VEC ? 0 : (int)(row * E & 3), rows * E, wide_words};
  // long rows leave no registers for the weights, the longest none for all of their words: a third of them at a time
  constexpr bool kOnce = !VEC && K <= 4, kAhead = !VEC && K <= 2;
  constexpr int kPart = VEC ? 1 : K <= 6 ? K : 3;
  float gamma_of[kOnce ? K : 1][4];
  OddRows<T, kPart, LANES, 3> odd_row, odd_next;
  if constexpr (kOnce) load_params_odd<K, LANES>(odd, gamma, lane, gamma_of);
  if constexpr (kAhead) odd_next.load(odd, in, row * E, lane, row < rows);
  float dg[K][V] = {}, db[K][V] = {};
  for (; row - slot < rows; row += stride) {
    const bool live = row < rows;
    const long long at = row * E;
    if constexpr (VEC) {
      ahead.ask(in, at + stride * E, lane, E, row + stride < rows);
    } else if constexpr (kAhead) {
      odd_row = odd_next;
      odd_next.load(odd, in, at + stride * E, lane, row + stride < rows);
    } else if constexpr (kOnce) {
      odd_row.load(odd, in, at, lane, live);
    }
    const float mean = live ? __ldg(mean_in + row) : 0.f, rstd = live ? __ldg(rstd_in + row) : 0.f;
    if constexpr (VEC) copies_wait<1>();
    float g[K][V], h[K][V];
    uint32_t words[K][V];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int c = (lane + LANES * j) * V - odd.shift;
      if constexpr (!VEC && !kOnce)
        if (j % kPart == 0) odd_row.load(odd, in, at, lane, live, j);
#pragma unroll
      for (int i = 0; i < V; ++i) g[j][i] = h[j][i] = 0.f;
      if (c >= E || !live) continue;
      float xf[V], w[V];
      if constexpr (VEC) {
        ahead.read(j, 0, g[j]);
        ahead.read(j, 1, xf);
        ahead.read(j, 2, h[j]);
      } else {
        odd_row.read(odd, j % kPart, 0, c, g[j]);
        odd_row.read(odd, j % kPart, 1, c, xf);
        odd_row.read(odd, j % kPart, 2, c, h[j]);
      }
      if constexpr (VEC) {
        load_param<V>(gamma, c, w);
      } else if constexpr (kOnce) {
#pragma unroll
        for (int i = 0; i < V; ++i) w[i] = gamma_of[j][i];
      } else {
        load_param_odd(odd, gamma, c, w);
      }
      words_of<V>(d, key, (unsigned long long)(at + c), words[j]);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float sum = fmaf(xf[i], d.scale, h[j][i]);
        h[j][i] = ((words[j][i] > d.last ? sum : h[j][i]) - mean) * rstd;
        if (!VEC && !odd.inside(c + i)) h[j][i] = 0.f;
        dg[j][i] = fmaf(g[j][i], h[j][i], dg[j][i]);
        db[j][i] += g[j][i];
        g[j][i] *= w[i];
        s1 += g[j][i];
        s2 = fmaf(g[j][i], h[j][i], s2);
      }
    }
    // by rstd already
    const float c1 = row_sum<LANES>(s1) * inv_e * rstd, c2 = row_sum<LANES>(s2) * inv_e * rstd;
    if (!live) continue;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int c = (lane + LANES * j) * V - odd.shift;
      if (c >= E) continue;
#pragma unroll
      for (int i = 0; i < V; ++i) g[j][i] = fmaf(g[j][i], rstd, -fmaf(h[j][i], c2, c1));
      if (grad_residual) {
        if constexpr (VEC) store_word<T, V>(grad_residual + at + c, g[j]);
        else store_odd<T>(odd, grad_residual, at, c, g[j]);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) g[j][i] = words[j][i] > d.last ? g[j][i] * d.scale : 0.f;
      if (grad_x) {
        if constexpr (VEC) store_word<T, V>(grad_x + at + c, g[j]);
        else store_odd<T>(odd, grad_x, at, c, g[j]);
      }
    }
  }
  if (!partial) return;
  copies_wait<0>();
  __syncthreads();                                       // the ring becomes the lanes' sums
  constexpr int kWidth = LANES * V * K;
  float *part = reinterpret_cast<float *>(ring), *mine = part + (warp * kRowsAtOnce + slot) * kWidth + lane * V - odd.shift;
#pragma unroll
  for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (VEC || odd.inside((lane + LANES * j) * V - odd.shift + i)) mine[j * LANES * V + i] = pass == 0 ? dg[j][i] : db[j][i];
    __syncthreads();
    for (int c = threadIdx.x; c < E; c += kWarps * 32) {
      float t = part[c];
#pragma unroll 8
      for (int w = 1; w < kSlots; ++w) t += part[w * kWidth + c];
      partial[((long long)blockIdx.x * 2 + pass) * E + c] = t;
    }
    __syncthreads();
  }
}

// Sums of the CTAs' rows: columns [0, E) of `partial` are grad_gamma, [E, 2E) grad_beta.  32 columns and 32 row lanes a CTA.
__global__ void __launch_bounds__(1024)
partial_sum_kernel(const float *partial, int ctas, int E, float *__restrict__ grad_gamma, float *__restrict__ grad_beta) {
  __shared__ float part[32][32];
  const int lane = threadIdx.x & 31, rl = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  launch_wait();
  float t = 0.f;
  if (col < 2 * E)
#pragma unroll 8
    for (int i = rl; i < ctas; i += 32) t += __ldcg(partial + (long long)i * 2 * E + col);
  part[rl][lane] = t;
  __syncthreads();
  if (rl != 0 || col >= 2 * E) return;
#pragma unroll
  for (int i = 1; i < 32; ++i) t += part[i][lane];
  (col < E ? grad_gamma + col : grad_beta + col - E)[0] = t;
}

bool on_grid(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

template <typename T>
unsigned elementwise_grid(long long n) {
  const long long per_cta = kThreads * kUnroll * (16 / (int)sizeof(T));
  return (unsigned)((n + per_cta - 1) / per_cta);
}

template <typename T>
cudaError_t forward(const T *x, const T *residual, long long n, bool relu, const DropRule &d, T *y, cudaStream_t s) {
  const bool vec = on_grid(x, 16) && on_grid(y, 16) && (!residual || on_grid(residual, 16));
  const unsigned grid = elementwise_grid<T>(n);
#define DFA3D_GO(RELU, RES)                                                                                        \
  (vec ? dropout_forward_kernel<T, RELU, RES, true><<<grid, kThreads, 0, s>>>(x, residual, n, d, y)                 \
       : dropout_forward_kernel<T, RELU, RES, false><<<grid, kThreads, 0, s>>>(x, residual, n, d, y))
  if (relu) {
    if (residual) DFA3D_GO(true, true);
    else DFA3D_GO(true, false);
  } else {
    if (residual) DFA3D_GO(false, true);
    else DFA3D_GO(false, false);
  }
#undef DFA3D_GO
  return cudaGetLastError();
}

template <typename T>
cudaError_t backward(const T *grad_y, const T *ref, long long n, bool rng, const DropRule &d, T *grad_x, cudaStream_t s) {
  const bool vec = on_grid(grad_y, 16) && on_grid(grad_x, 16) && (!ref || on_grid(ref, 16));
  const unsigned grid = elementwise_grid<T>(n);
#define DFA3D_GO(REF, RNG)                                                                                       \
  (vec ? dropout_backward_kernel<T, REF, RNG, true><<<grid, kThreads, 0, s>>>(grad_y, ref, n, d, grad_x)          \
       : dropout_backward_kernel<T, REF, RNG, false><<<grid, kThreads, 0, s>>>(grad_y, ref, n, d, grad_x))
  if (ref) {
    if (rng) DFA3D_GO(true, true);
    else DFA3D_GO(true, false);
  } else {
    if (rng) DFA3D_GO(false, true);
    else DFA3D_GO(false, false);
  }
#undef DFA3D_GO
  return cudaGetLastError();
}

// How a row of E is laid out over lanes: words of V elements, K words a lane; off the grid words of four.
struct RowShape {
  int lanes, K;
  bool vec;
};
template <typename T>
RowShape row_shape(int E, bool aligned) {
  constexpr int V = 16 / (int)sizeof(T);
  if (!aligned || E % V != 0) {
    const int words = (E + (E % 4 ? 3 : 0) + 3) / 4;       // that a row may have a part of
    if (words <= 16) return {8, words <= 8 ? 1 : 2, false};
    if (words <= 32) return {16, 2, false};
    return {32, words <= 64 ? 2 : words <= 128 ? 4 : words <= 192 ? 6 : 9, false};
  }
  const int words = E / V, want = 16 / V;            // 16 elements a lane
  if (words <= 8 * want) return {8, words <= 8 ? 1 : words <= 16 ? 2 : 4, true};
  if (words <= 16 * want) return {16, want, true};
  const int K = (words + 31) / 32;
  return {32, V == 8 || K <= 4 ? K : K <= 6 ? 6 : 8, true};
}
// Calls GO(V, K, LANES, VEC) with what `r` says; the K that occur are 1, 2, 4 (fp32) or 1, 2 (16 bits) for 8 lanes, 4 or 2 for 16,
// 2 to 8 for 32.
#define DFA3D_ROWS(T, r, GO)                                                                     \
  if (!r.vec) {                                                                                  \
    if (r.lanes == 8) {                                                                          \
      if (r.K == 1) GO(4, 1, 8, false);                                                          \
      else GO(4, 2, 8, false);                                                                   \
    } else if (r.lanes == 16) GO(4, 2, 16, false);                                               \
    else if (r.K == 2) GO(4, 2, 32, false);                                                      \
    else if (r.K == 4) GO(4, 4, 32, false);                                                      \
    else if (r.K == 6) GO(4, 6, 32, false);                                                      \
    else GO(4, 9, 32, false);                                                                    \
  } else if constexpr (sizeof(T) == 4) {                                                         \
    if (r.lanes == 8) {                                                                          \
      if (r.K == 1) GO(4, 1, 8, true);                                                           \
      else if (r.K == 2) GO(4, 2, 8, true);                                                      \
      else GO(4, 4, 8, true);                                                                    \
    } else if (r.lanes == 16) GO(4, 4, 16, true);                                                \
    else if (r.K <= 3) GO(4, 3, 32, true);                                                       \
    else if (r.K == 4) GO(4, 4, 32, true);                                                       \
    else if (r.K == 6) GO(4, 6, 32, true);                                                       \
    else GO(4, 8, 32, true);                                                                     \
  } else {                                                                                       \
    if (r.lanes == 8) {                                                                          \
      if (r.K == 1) GO(8, 1, 8, true);                                                           \
      else GO(8, 2, 8, true);                                                                    \
    } else if (r.lanes == 16) GO(8, 2, 16, true);                                                \
    else if (r.K <= 2) GO(8, 2, 32, true);                                                       \
    else if (r.K == 3) GO(8, 3, 32, true);                                                       \
    else GO(8, 4, 32, true);                                                                     \
  }

// CTAs for `rows` rows, a lane group of which takes `each` one after the other, at most `cap`.
long long row_ctas(long long rows, int lanes, long long each, long long cap) {
  const long long at_once = kWarps * (32 / lanes) * each;
  return std::max(1LL, std::min((rows + at_once - 1) / at_once, cap));
}

// Two rows of a thread's words of `tensors` tensors, or its columns' sums.
size_t ring_bytes(const RowShape &r, int tensors) { return r.vec ? 2u * r.K * tensors * kWarps * 32 * 16 : 0u; }

// Launches a kernel that may need more shared memory than it gets by itself: a setting of the kernel on the current device, made
// once for each of the first 64 devices.
template <auto KERNEL, typename... A>
cudaError_t launch_rows(unsigned grid, size_t shared, cudaStream_t s, A... args) {
  if (shared > 48 * 1024) {
    static std::atomic<unsigned long long> done{0};
    int device = 0;
    cudaError_t rc = cudaGetDevice(&device);
    if (rc != cudaSuccess) return rc;
    const unsigned long long bit = device < 64 ? 1ull << device : 0ull;
    if (!(done.load(std::memory_order_relaxed) & bit)) {
      rc = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared);
      if (rc != cudaSuccess) return rc;
      done.fetch_or(bit, std::memory_order_relaxed);
    }
  }
  KERNEL<<<grid, kWarps * 32, shared, s>>>(args...);
  return cudaGetLastError();
}

template <typename T>
cudaError_t norm_forward(const T *x, const T *residual, const float *gamma, const float *beta, long long rows, int E,
                         const DropRule &d, float eps, T *y, float *mean, float *rstd, cudaStream_t s) {
  const RowShape r = row_shape<T>(E, on_grid(x, 16) && on_grid(residual, 16) && on_grid(y, 16) && on_grid(gamma, 16) &&
                                         on_grid(beta, 16));
  const bool wide = on_grid(x, 4 * sizeof(T)) && on_grid(residual, 4 * sizeof(T)) && on_grid(y, 4 * sizeof(T));
  const unsigned grid = (unsigned)row_ctas(rows, r.lanes, 1, 148 * (r.vec ? kForwardResident : kOddResident));
  const size_t shared = ring_bytes(r, 2);
#define DFA3D_GO(V, K, LANES, VEC)                                                                                      \
  return launch_rows<dropout_add_layer_norm_kernel<T, V, K, LANES, VEC>>(grid, shared, s, x, residual, gamma, beta, rows, E, wide, \
                     d, eps, y, mean, rstd)
  DFA3D_ROWS(T, r, DFA3D_GO)
#undef DFA3D_GO
}

// Every CTA leaves a row of `partial` to be added up.
long long backward_ctas(long long rows, int lanes) { return row_ctas(rows, lanes, 1, 148 * 2); }

template <typename T>
cudaError_t norm_backward(const T *grad_y, const T *x, const T *residual, const float *gamma, const float *mean,
                          const float *rstd, long long rows, int E, const DropRule &d, T *grad_x, T *grad_residual,
                          float *grad_gamma, float *grad_beta, float *partial, cudaStream_t s) {
  const RowShape r = row_shape<T>(E, on_grid(x, 16) && on_grid(residual, 16) && on_grid(grad_y, 16) && on_grid(gamma, 16) &&
                                         on_grid(grad_x, 16) && on_grid(grad_residual, 16));      // null is on the grid
  const bool wide = on_grid(x, 4 * sizeof(T)) && on_grid(residual, 4 * sizeof(T)) && on_grid(grad_y, 4 * sizeof(T)) &&
                    on_grid(grad_x, 4 * sizeof(T)) && on_grid(grad_residual, 4 * sizeof(T));
  const unsigned grid = (unsigned)backward_ctas(rows, r.lanes);
  if (!grad_gamma) partial = nullptr;
  cudaError_t rc = cudaSuccess;
#define DFA3D_GO(V, K, LANES, VEC)                                                                                            \
  rc = launch_rows<dropout_layer_norm_backward_kernel<T, V, K, LANES, VEC>>(                                                   \
      grid, std::max(ring_bytes(r, 3), sizeof(float) * kWarps * 32 * V * K), s, grad_y, x, residual, gamma, mean, rstd, rows,   \
      E, wide, d, grad_x, grad_residual, partial)
  DFA3D_ROWS(T, r, DFA3D_GO)
#undef DFA3D_GO
  if (rc != cudaSuccess || !partial) return rc;
  // begins while the other's CTAs leave
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((2 * E + 31) / 32);
  cfg.blockDim = dim3(1024);
  cfg.stream = s;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, partial_sum_kernel, (const float *)partial, (int)grid, E, grad_gamma, grad_beta);
}

}  // namespace

// dtype: DFA3D_DTYPE_F32 (0), _BF16 (1) or _F16 (3)
#define DFA3D_TYPED(call)                                 \
  if (dtype == 0) { using T = float; return call; }       \
  if (dtype == 1) { using T = __nv_bfloat16; return call; } \
  { using T = __half; return call; }

cudaError_t launch_dropout_forward(const void *x, const void *residual, int dtype, long long n, bool relu, double p,
                                   const int64_t *seed, uint32_t site, void *y, cudaStream_t s) {
  const DropRule d = drop_rule(p, seed, site);
  DFA3D_TYPED(forward<T>((const T *)x, (const T *)residual, n, relu, d, (T *)y, s))
}

cudaError_t launch_dropout_backward(const void *grad_y, const void *ref, bool ref_is_result, int dtype, long long n, double p,
                                    const int64_t *seed, uint32_t site, void *grad_x, cudaStream_t s) {
  const DropRule d = drop_rule(p, seed, site);
  DFA3D_TYPED(backward<T>((const T *)grad_y, (const T *)ref, n, d.rng && !ref_is_result, d, (T *)grad_x, s))
}

cudaError_t launch_dropout_add_layer_norm(const void *x, const void *residual, const float *gamma, const float *beta, int dtype,
                                          long long rows, int E, double p, const int64_t *seed, uint32_t site, float eps, void *y,
                                          float *mean, float *rstd, cudaStream_t s) {
  const DropRule d = drop_rule(p, seed, site);
  DFA3D_TYPED(norm_forward<T>((const T *)x, (const T *)residual, gamma, beta, rows, E, d, eps, (T *)y, mean, rstd, s))
}

// For the layout with the fewest rows at a time.
long long dropout_layer_norm_workspace(long long rows, int E) { return rows > 0 ? backward_ctas(rows, 32) * 2 * E * 4 : 0; }

cudaError_t launch_dropout_layer_norm_backward(const void *grad_y, const void *x, const void *residual, const float *gamma,
                                               const float *mean, const float *rstd, int dtype, long long rows, int E, double p,
                                               const int64_t *seed, uint32_t site, void *grad_x, void *grad_residual,
                                               float *grad_gamma, float *grad_beta, float *partial, cudaStream_t s) {
  const DropRule d = drop_rule(p, seed, site);
  DFA3D_TYPED(norm_backward<T>((const T *)grad_y, (const T *)x, (const T *)residual, gamma, mean, rstd, rows, E, d, (T *)grad_x,
                               (T *)grad_residual, grad_gamma, grad_beta, partial, s))
}

}  // namespace dfa3d
