// Dropout whose mask is never stored (dfa3d_philox.cuh), alone and at the end of a residual block (sm_100a):
//
//   y = [residual +] keep * act(x) / (1 - p)                      elementwise; act: none or ReLU
//   y = LayerNorm(residual + keep * x / (1 - p))                  rows of up to 1024 columns
//
// with their backward passes, which form the mask again from (seed, site, element).  Every tensor is read once and written once;
// what bounds them is HBM, with the integer pipes next: a Philox block for four elements is about 50 instructions.
#include <algorithm>

#include "dfa3d_launch.h"
#include "dfa3d_philox.cuh"
#include "dfa3d_rowvec.cuh"

namespace dfa3d {
namespace {

constexpr int kThreads = 256;

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

// Threads take 16-byte words of every tensor, U of them a CTA width apart, all loads first.  VEC = false: an address is off the
// 16-byte grid, elements are read and written one by one (same mask, same result).
template <typename T, bool RELU, bool RES, bool VEC>
__global__ void __launch_bounds__(kThreads)
dropout_forward_kernel(const T *x, const T *__restrict__ residual, long long n, DropRule d,
                       T *y) {      // y may be x
  constexpr int V = 16 / sizeof(T), U = 2;
  const DropKey key = drop_key(d);
  const long long words = n / V, first = (long long)blockIdx.x * kThreads * U + threadIdx.x;
  if (VEC) {
    Word<T, V> xw[U], rw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long w = first + u * kThreads;
      if (w < words) {
        xw[u] = load_once<T, V>(x + w * V);
        if (RES) rw[u] = load_once<T, V>(residual + w * V);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long w = first + u * kThreads;
      if (w >= words) break;
      const uint32_t kept = kept_bits<V, true>(d, key, (unsigned long long)w * V);
      float f[V], r[V] = {};
      widen_word<T, V>(xw[u], f);
      if (RES) widen_word<T, V>(rw[u], r);
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = drop_one<RELU, RES>(f[i], r[i], kept >> i & 1u, d.scale);
      store_word<T, V>(y + w * V, f);
    }
  }
  // all elements where VEC is false, the few behind the last word otherwise (by the first CTA)
  const long long from = VEC ? words * V : 0;
  if (VEC && blockIdx.x != 0) return;
  const long long groups = (n - from + 3) / 4, step = VEC ? kThreads : (long long)gridDim.x * kThreads;
  for (long long q = VEC ? threadIdx.x : (long long)blockIdx.x * kThreads + threadIdx.x; q < groups; q += step) {
    const long long at = from + q * 4;
    const uint32_t kept = kept_bits<4, true>(d, key, (unsigned long long)at);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + i < n)
        y[at + i] = narrow<T>(drop_one<RELU, RES>(wide(x[at + i]), RES ? wide(residual[at + i]) : 0.f, kept >> i & 1u, d.scale));
  }
}

// grad_x = keep * [ref > 0 or NaN] * grad_y / (1 - p).  With a ReLU and no residual `ref` is the forward's result, whose zeros
// are the dropped elements too (scale >= 1: no kept positive value becomes 0), and no mask is formed (RNG = false); with a
// residual it is the forward's x.
template <typename T, bool REF, bool RNG, bool VEC>
__global__ void __launch_bounds__(kThreads)
dropout_backward_kernel(const T *__restrict__ grad_y, const T *__restrict__ ref, long long n, DropRule d, T *__restrict__ grad_x) {
  constexpr int V = 16 / sizeof(T), U = 2;
  const DropKey key = RNG ? drop_key(d) : DropKey{0u, 0u};
  auto one = [&](float g, float v, bool kept) { return !kept || (REF && v <= 0.f) ? 0.f : g * d.scale; };
  const long long words = n / V, first = (long long)blockIdx.x * kThreads * U + threadIdx.x;
  if (VEC) {
    Word<T, V> gw[U], vw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long w = first + u * kThreads;
      if (w < words) {
        gw[u] = load_once<T, V>(grad_y + w * V);
        if (REF) vw[u] = load_once<T, V>(ref + w * V);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long w = first + u * kThreads;
      if (w >= words) break;
      const uint32_t kept = RNG ? kept_bits<V, true>(d, key, (unsigned long long)w * V) : ~0u;
      float g[V], v[V] = {};
      widen_word<T, V>(gw[u], g);
      if (REF) widen_word<T, V>(vw[u], v);
#pragma unroll
      for (int i = 0; i < V; ++i) g[i] = one(g[i], v[i], kept >> i & 1u);
      store_word<T, V>(grad_x + w * V, g);
    }
  }
  const long long from = VEC ? words * V : 0;
  if (VEC && blockIdx.x != 0) return;
  const long long groups = (n - from + 3) / 4, step = VEC ? kThreads : (long long)gridDim.x * kThreads;
  for (long long q = VEC ? threadIdx.x : (long long)blockIdx.x * kThreads + threadIdx.x; q < groups; q += step) {
    const long long at = from + q * 4;
    const uint32_t kept = RNG ? kept_bits<4, true>(d, key, (unsigned long long)at) : ~0u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + i < n) grad_x[at + i] = narrow<T>(one(wide(grad_y[at + i]), REF ? wide(ref[at + i]) : 0.f, kept >> i & 1u));
  }
}

// ------------------------------------------------------------------------------------------------
// LayerNorm(residual + dropout(x))
// ------------------------------------------------------------------------------------------------
constexpr int kWarps = 8;

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// V elements from `c` on of a row of E.  VEC: V divides E and the row is aligned for words of V; else one by one, zeros behind
// the row's end.
template <typename T, int V, bool VEC>
__device__ __forceinline__ void load_group(const T *row, int c, int E, float (&f)[V]) {
  if (VEC) {
    widen_word<T, V>(load_once<T, V>(row + c), f);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = c + i < E ? wide(row[c + i]) : 0.f;
  }
}
template <typename T, int V, bool VEC>
__device__ __forceinline__ void store_group(T *row, int c, int E, const float (&f)[V]) {
  if (VEC) {
    store_word<T, V>(row + c, f);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (c + i < E) row[c + i] = narrow<T>(f[i]);
  }
}
template <int V>
__device__ __forceinline__ void load_param(const float *p, int c, int E, bool whole, float (&f)[V]) {
  if (whole) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 t = __ldg(reinterpret_cast<const float4 *>(p + c + i));
      f[i] = t.x; f[i + 1] = t.y; f[i + 2] = t.z; f[i + 3] = t.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = c + i < E ? __ldg(p + c + i) : 0.f;
  }
}

// A warp owns a row; lane l holds the groups of V columns l, l + 32, ... (K of them).  The sum is normalised as it stands in
// 32 bits and is not written: the backward forms it again from the same x and residual, so that storage in 16 bits rounds
// nothing but y.
template <typename T, int V, int K, bool VEC>
__global__ void __launch_bounds__(kWarps * 32)
dropout_add_layer_norm_kernel(const T *__restrict__ x, const T *__restrict__ residual, const float *__restrict__ gamma,
                              const float *__restrict__ beta, long long rows, int E, DropRule d, float eps, T *__restrict__ y,
                              float *__restrict__ mean_out, float *__restrict__ rstd_out) {
  const DropKey key = drop_key(d);
  const float inv_e = 1.f / (float)E;
  const int lane = threadIdx.x & 31;
  const long long stride = (long long)gridDim.x * kWarps;
  for (long long row = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5); row < rows; row += stride) {
    float v[K][V];
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int c = (lane + 32 * j) * V;
#pragma unroll
      for (int i = 0; i < V; ++i) v[j][i] = 0.f;
      if (c >= E) continue;
      float xf[V];
      load_group<T, V, VEC>(x + row * E, c, E, xf);
      load_group<T, V, VEC>(residual + row * E, c, E, v[j]);
      const uint32_t kept = kept_bits<V, VEC>(d, key, (unsigned long long)(row * E + c));
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[j][i] = kept >> i & 1u ? fmaf(xf[i], d.scale, v[j][i]) : v[j][i];
        s += v[j][i];
      }
    }
    const float mean = warp_sum(s) * inv_e;
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int c = (lane + 32 * j) * V;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float t = c + i < E ? v[j][i] - mean : 0.f;
        q = fmaf(t, t, q);
      }
    }
    const float rstd = rsqrtf(warp_sum(q) * inv_e + eps);
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int c = (lane + 32 * j) * V;
      if (c >= E) continue;
      float g[V], b[V];
      load_param<V>(gamma, c, E, VEC, g);
      load_param<V>(beta, c, E, VEC, b);
#pragma unroll
      for (int i = 0; i < V; ++i) g[i] = (v[j][i] - mean) * rstd * g[i] + b[i];
      store_group<T, V, VEC>(y + row * E, c, E, g);
    }
    if (lane == 0 && mean_out) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
  }
}

// grad_residual = rstd * (d - mean(d) - xhat * mean(d * xhat)) with d = grad_y * gamma; grad_x = keep * grad_residual / (1 - p).
// grad_gamma (sum of grad_y * xhat) and grad_beta (sum of grad_y) are summed over a warp's rows in registers, over the CTA's
// warps in shared memory, and written as the CTA's own row of `partial` (ctas, 2, E): the second kernel adds these up in a
// fixed order, so that a gradient is the same bits in every run.
template <typename T, int V, int K, bool VEC>
__global__ void __launch_bounds__(kWarps * 32)
dropout_layer_norm_backward_kernel(const T *__restrict__ grad_y, const T *__restrict__ x, const T *__restrict__ residual,
                                   const float *__restrict__ gamma, const float *__restrict__ mean_in,
                                   const float *__restrict__ rstd_in, long long rows, int E, DropRule d, T *__restrict__ grad_x,
                                   T *__restrict__ grad_residual, float *__restrict__ partial) {
  __shared__ float part[kWarps][32 * V * K];
  const DropKey key = drop_key(d);
  const float inv_e = 1.f / (float)E;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long stride = (long long)gridDim.x * kWarps;
  float dg[K][V] = {}, db[K][V] = {};
  for (long long row = (long long)blockIdx.x * kWarps + warp; row < rows; row += stride) {
    const float mean = __ldg(mean_in + row), rstd = __ldg(rstd_in + row);
    float g[K][V], h[K][V];
    uint32_t kept[K];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int c = (lane + 32 * j) * V;
      kept[j] = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) g[j][i] = h[j][i] = 0.f;
      if (c >= E) continue;
      float xf[V], w[V];
      load_group<T, V, VEC>(grad_y + row * E, c, E, g[j]);
      load_group<T, V, VEC>(x + row * E, c, E, xf);
      load_group<T, V, VEC>(residual + row * E, c, E, h[j]);
      load_param<V>(gamma, c, E, VEC, w);
      kept[j] = kept_bits<V, VEC>(d, key, (unsigned long long)(row * E + c));
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float sum = kept[j] >> i & 1u ? fmaf(xf[i], d.scale, h[j][i]) : h[j][i];
        h[j][i] = (sum - mean) * rstd;
        if (!VEC && c + i >= E) h[j][i] = 0.f;
        dg[j][i] = fmaf(g[j][i], h[j][i], dg[j][i]);
        db[j][i] += g[j][i];
        g[j][i] *= w[i];
        s1 += g[j][i];
        s2 = fmaf(g[j][i], h[j][i], s2);
      }
    }
    const float c1 = warp_sum(s1) * inv_e, c2 = warp_sum(s2) * inv_e;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int c = (lane + 32 * j) * V;
      if (c >= E) continue;
#pragma unroll
      for (int i = 0; i < V; ++i) g[j][i] = rstd * (g[j][i] - c1 - h[j][i] * c2);
      if (grad_residual) store_group<T, V, VEC>(grad_residual + row * E, c, E, g[j]);
#pragma unroll
      for (int i = 0; i < V; ++i) g[j][i] = kept[j] >> i & 1u ? g[j][i] * d.scale : 0.f;
      if (grad_x) store_group<T, V, VEC>(grad_x + row * E, c, E, g[j]);
    }
  }
  if (!partial) return;
#pragma unroll
  for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) part[warp][(lane + 32 * j) * V + i] = pass == 0 ? dg[j][i] : db[j][i];
    __syncthreads();
    for (int c = threadIdx.x; c < E; c += kWarps * 32) {
      float t = part[0][c];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) t += part[w][c];
      partial[((long long)blockIdx.x * 2 + pass) * E + c] = t;
    }
    __syncthreads();
  }
}

// Sums of the CTAs' rows: columns [0, E) of `partial` are grad_gamma, [E, 2E) grad_beta.  32 columns and 8 row lanes a CTA.
__global__ void __launch_bounds__(256)
partial_sum_kernel(const float *__restrict__ partial, int ctas, int E, float *__restrict__ grad_gamma, float *__restrict__ grad_beta) {
  __shared__ float part[8][32];
  const int lane = threadIdx.x & 31, rl = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  float t = 0.f;
  if (col < 2 * E)
#pragma unroll 8
    for (int i = rl; i < ctas; i += 8) t += __ldg(partial + (long long)i * 2 * E + col);
  part[rl][lane] = t;
  __syncthreads();
  if (rl != 0 || col >= 2 * E) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) t += part[i][lane];
  (col < E ? grad_gamma + col : grad_beta + col - E)[0] = t;
}

bool on_grid(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

template <typename T>
cudaError_t forward(const T *x, const T *residual, long long n, bool relu, const DropRule &d, T *y, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T), U = 2;
  const bool vec = on_grid(x, 16) && on_grid(y, 16) && (!residual || on_grid(residual, 16));
  const long long per_cta = (long long)kThreads * U * V;
  const unsigned grid = (unsigned)std::min((n + per_cta - 1) / per_cta, (1LL << 31) - 1);
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
  constexpr int V = 16 / sizeof(T), U = 2;
  const bool vec = on_grid(grad_y, 16) && on_grid(grad_x, 16) && (!ref || on_grid(ref, 16));
  const long long per_cta = (long long)kThreads * U * V;
  const unsigned grid = (unsigned)std::min((n + per_cta - 1) / per_cta, (1LL << 31) - 1);
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

long long row_ctas(long long rows, long long rows_a_warp, long long cap) {
  return std::max(1LL, std::min((rows + kWarps * rows_a_warp - 1) / (kWarps * rows_a_warp), cap));
}

template <typename T>
cudaError_t norm_forward(const T *x, const T *residual, const float *gamma, const float *beta, long long rows, int E,
                         const DropRule &d, float eps, T *y, float *mean, float *rstd, cudaStream_t s) {
  const bool vec = E % 4 == 0 && on_grid(x, 4 * sizeof(T)) && on_grid(residual, 4 * sizeof(T)) && on_grid(y, 4 * sizeof(T)) &&
                   on_grid(gamma, 16) && on_grid(beta, 16);
  const unsigned grid = (unsigned)row_ctas(rows, 1, 148 * 4);
#define DFA3D_GO(K, VEC)                                                                                                 \
  dropout_add_layer_norm_kernel<T, 4, K, VEC><<<grid, kWarps * 32, 0, s>>>(x, residual, gamma, beta, rows, E, d, eps, y, \
                                                                           mean, rstd)
  const int k = (E + 127) / 128;
  if (!vec) {
    if (k <= 2) DFA3D_GO(2, false);
    else DFA3D_GO(8, false);
  } else switch (k) {
    case 1: DFA3D_GO(1, true); break;
    case 2: DFA3D_GO(2, true); break;
    case 3: DFA3D_GO(3, true); break;
    case 4: DFA3D_GO(4, true); break;
    case 5: case 6: DFA3D_GO(6, true); break;
    default: DFA3D_GO(8, true);
  }
#undef DFA3D_GO
  return cudaGetLastError();
}

long long backward_ctas(long long rows) { return row_ctas(rows, 4, 148 * 3); }

template <typename T>
cudaError_t norm_backward(const T *grad_y, const T *x, const T *residual, const float *gamma, const float *mean,
                          const float *rstd, long long rows, int E, const DropRule &d, T *grad_x, T *grad_residual,
                          float *grad_gamma, float *grad_beta, float *partial, cudaStream_t s) {
  const bool vec = E % 4 == 0 && on_grid(x, 4 * sizeof(T)) && on_grid(residual, 4 * sizeof(T)) &&
                   on_grid(grad_y, 4 * sizeof(T)) && (!grad_x || on_grid(grad_x, 4 * sizeof(T))) &&
                   (!grad_residual || on_grid(grad_residual, 4 * sizeof(T))) && on_grid(gamma, 16);
  const unsigned grid = (unsigned)backward_ctas(rows);
#define DFA3D_GO(K, VEC)                                                                                        \
  dropout_layer_norm_backward_kernel<T, 4, K, VEC><<<grid, kWarps * 32, 0, s>>>(                                 \
      grad_y, x, residual, gamma, mean, rstd, rows, E, d, grad_x, grad_residual, grad_gamma ? partial : nullptr)
  const int k = (E + 127) / 128;
  if (!vec) {
    if (k <= 2) DFA3D_GO(2, false);
    else DFA3D_GO(8, false);
  } else switch (k) {
    case 1: DFA3D_GO(1, true); break;
    case 2: DFA3D_GO(2, true); break;
    case 3: DFA3D_GO(3, true); break;
    case 4: DFA3D_GO(4, true); break;
    case 5: case 6: DFA3D_GO(6, true); break;
    default: DFA3D_GO(8, true);
  }
#undef DFA3D_GO
  if (grad_gamma) partial_sum_kernel<<<(2 * E + 31) / 32, 256, 0, s>>>(partial, (int)grid, E, grad_gamma, grad_beta);
  return cudaGetLastError();
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

long long dropout_layer_norm_workspace(long long rows, int E) { return rows > 0 ? backward_ctas(rows) * 2 * E * 4 : 0; }

cudaError_t launch_dropout_layer_norm_backward(const void *grad_y, const void *x, const void *residual, const float *gamma,
                                               const float *mean, const float *rstd, int dtype, long long rows, int E, double p,
                                               const int64_t *seed, uint32_t site, void *grad_x, void *grad_residual,
                                               float *grad_gamma, float *grad_beta, float *partial, cudaStream_t s) {
  const DropRule d = drop_rule(p, seed, site);
  DFA3D_TYPED(norm_backward<T>((const T *)grad_y, (const T *)x, (const T *)residual, gamma, mean, rstd, rows, E, d, (T *)grad_x,
                               (T *)grad_residual, grad_gamma, grad_beta, partial, s))
}

}  // namespace dfa3d
