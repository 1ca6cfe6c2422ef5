// Group norm of channels-last feature pyramids with an activation, forward and backward (sm_100a):
//
//   x (B, N, C), N = the rows of L levels; every (image, level, group of C / G channels) is normalised by itself,
//   z = (x - mean) * rstd * gamma + beta,  y = act(z),  act: none, ReLU, SiLU = z / (1 + exp(-z)).
//
// It is the layout of the operator's `value`, so that features go from their projection to the attention without a transpose,
// and all levels share a launch.  Rows that belong to no level become 0, in y and in grad_x.
//
// Statistics: a thread keeps, for each of its V channels, the number of values, their mean and the sum of squares around it; eight
// rows at a time are reduced in registers around their own mean and merged by
//   M2 = M2a + M2b + (mb - ma)^2 na nb / (na + nb)                      (Chan, Golub, LeVeque 1979),
// so that nothing is lost where the mean is large against the spread.  Threads, warps and CTAs are merged in a fixed order: a
// result is the same bits in every run.
#include <algorithm>

#include "dfa3d_launch.h"
#include "dfa3d_rowvec.cuh"
#include "dfa3d_segments.h"

namespace dfa3d {
namespace {

enum Act { kNone = 0, kRelu = 1, kSilu = 2 };

struct GnArgs {
  const int64_t *shapes, *start;     // level table, or null: one level
  int shape_stride;
  int N, C, G, L, S, act;            // S runs of rows an image
  int weight_rows;                   // 1, or L: weights of each level's own
  const float *weight, *bias;
  float eps;
  int cpg, nv, RL;                   // channels a group, vectors a row, rows a CTA reads at a time
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ int pieces(const GnArgs &a) { return a.S + 2 * a.L + 1; }

// Rows that row lane rl of RL takes of a piece of n.
__device__ __forceinline__ int lane_rows(int n, int rl, int RL) { return n > rl ? (n - rl + RL - 1) / RL : 0; }

__device__ __forceinline__ float activate(float z, int act) {
  if (act == kRelu) return z <= 0.f ? 0.f : z;                       // a NaN passes, as in torch
  if (act == kSilu) return z / (1.f + __expf(-z));
  return z;
}
// dz of dy
__device__ __forceinline__ float activate_grad(float g, float z, int act) {
  if (act == kRelu) return z <= 0.f ? 0.f : g;
  if (act == kSilu) {
    const float s = 1.f / (1.f + __expf(-z));
    return g * s * (1.f + z * (1.f - s));
  }
  return g;
}

constexpr int kRows = 8;      // rows of a thread in flight

// Threads of a CTA: 256, or as many as a row of up to 1024 channels has vectors.
constexpr int max_threads(int V) { return V >= 4 ? 256 : 1024 / V; }

// ------------------------------------------------------------------------------------------------
// forward
// ------------------------------------------------------------------------------------------------
// partial (B, pieces, G): mean and sum of squares around it, of the piece's values of the group.
template <typename T, int V>
__global__ void __launch_bounds__(max_threads(V))
gn_stats_kernel(const T *__restrict__ x, GnArgs a, float2 *__restrict__ partial) {
  extern __shared__ float2 chan[];       // (RL, C): a thread's mean and M2 of its channels
  __shared__ SegmentTable seg;
  if (threadIdx.x == 0) make_segments(seg, a.shapes, a.shape_stride, a.start, a.L, a.N);
  __syncthreads();
  const int b = blockIdx.x / a.S, run = blockIdx.x % a.S;
  const int r0 = run_begin(run, a.S, a.N), r1 = run_begin(run + 1, a.S, a.N);
  const int cv = threadIdx.x % a.nv, rl = threadIdx.x / a.nv;
  const bool active = rl < a.RL;
  const T *base = x + ((long long)b * a.N) * a.C + cv * V;
  for (int i = 1; i < seg.count; i += 2) {
    const int lo = max(r0, seg.end[i - 1]), hi = min(r1, seg.end[i]);
    if (lo >= hi) continue;
    float n = 0.f, mean[V] = {}, m2[V] = {};
    if (active) {
      for (int r = lo + rl; r < hi; r += a.RL * kRows) {
        Word<T, V> w[kRows];
#pragma unroll
        for (int u = 0; u < kRows; ++u)
          if (r + u * a.RL < hi) w[u] = load_word<T, V>(base + (long long)(r + u * a.RL) * a.C);
        const int cnt = min(kRows, (hi - r + a.RL - 1) / a.RL);
        float f[kRows][V];
#pragma unroll
        for (int u = 0; u < kRows; ++u) widen_word<T, V>(w[u], f[u]);
        const float nc = (float)cnt, inv = 1.f / nc, total = n + nc, part = nc / total, cross = n * part;
#pragma unroll
        for (int c = 0; c < V; ++c) {
          float s = 0.f, q = 0.f;
#pragma unroll
          for (int u = 0; u < kRows; ++u)
            if (u < cnt) s += f[u][c];
          s *= inv;
#pragma unroll
          for (int u = 0; u < kRows; ++u)
            if (u < cnt) q = fmaf(f[u][c] - s, f[u][c] - s, q);
          const float delta = s - mean[c];
          mean[c] = fmaf(delta, part, mean[c]);
          m2[c] += fmaf(delta * delta, cross, q);
        }
        n = total;
      }
#pragma unroll
      for (int c = 0; c < V; ++c) chan[rl * a.C + cv * V + c] = make_float2(mean[c], m2[c]);
    }
    __syncthreads();
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5, all = a.RL * a.cpg;
    const float inv_n = 1.f / ((float)(hi - lo) * (float)a.cpg);
    for (int g = threadIdx.x >> 5; g < a.G; g += warps) {
      float s = 0.f, q = 0.f;
      for (int e = lane; e < all; e += 32) {
        const int l = e / a.cpg;
        s = fmaf((float)lane_rows(hi - lo, l, a.RL), chan[l * a.C + g * a.cpg + e - l * a.cpg].x, s);
      }
      const float m = warp_sum(s) * inv_n;
      for (int e = lane; e < all; e += 32) {
        const int l = e / a.cpg;
        const float2 t = chan[l * a.C + g * a.cpg + e - l * a.cpg];
        const float d = t.x - m;
        q += fmaf(d * d, (float)lane_rows(hi - lo, l, a.RL), t.y);
      }
      q = warp_sum(q);
      if (lane == 0) partial[((long long)b * pieces(a) + run + i) * a.G + g] = make_float2(m, q);
    }
    __syncthreads();
  }
}

// Merges the pieces of segment i of image b; every thread returns when stats[g] = (mean, rstd) is in shared memory.
__device__ __forceinline__ void merge_stats(const GnArgs &a, const SegmentTable &seg, const float2 *partial, int b, int i,
                                            float2 *stats) {
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int lo = seg.end[i - 1], hi = seg.end[i], first = run_of(lo, a.S, a.N), last = run_of(hi - 1, a.S, a.N);
  const float2 *p = partial + ((long long)b * pieces(a) + i) * a.G;
  for (int g = threadIdx.x >> 5; g < a.G; g += warps) {
    float s = 0.f, q = 0.f;
    for (int r = first + lane; r <= last; r += 32) {
      const float n = (float)(min(hi, run_begin(r + 1, a.S, a.N)) - max(lo, run_begin(r, a.S, a.N)));
      s = fmaf(n, p[(long long)r * a.G + g].x, s);
    }
    const float m = warp_sum(s) / (float)(hi - lo);
    for (int r = first + lane; r <= last; r += 32) {
      const float n = (float)(min(hi, run_begin(r + 1, a.S, a.N)) - max(lo, run_begin(r, a.S, a.N)));
      const float2 t = p[(long long)r * a.G + g];
      const float d = t.x - m;
      q += fmaf(d * d, n * (float)a.cpg, t.y);
    }
    q = warp_sum(q);
    if (lane == 0) stats[g] = make_float2(m, rsqrtf(q / ((float)(hi - lo) * (float)a.cpg) + a.eps));
  }
  __syncthreads();
}

template <typename T, int V>
__device__ __forceinline__ void zero_rows(T *base, const GnArgs &a, int lo, int hi, int rl) {
  const float zero[V] = {};
  if (rl < a.RL)
    for (int r = lo + rl; r < hi; r += a.RL) store_word<T, V>(base + (long long)r * a.C, zero);
}

template <typename T, int V>
__global__ void __launch_bounds__(max_threads(V))
gn_apply_kernel(const T *__restrict__ x, GnArgs a, const float2 *__restrict__ partial, T *__restrict__ y,
                                float *__restrict__ mean_out, float *__restrict__ rstd_out) {
  extern __shared__ float2 stats[];      // (G): mean, rstd
  __shared__ SegmentTable seg;
  if (threadIdx.x == 0) make_segments(seg, a.shapes, a.shape_stride, a.start, a.L, a.N);
  __syncthreads();
  const int b = blockIdx.x / a.S, run = blockIdx.x % a.S;
  const int r0 = run_begin(run, a.S, a.N), r1 = run_begin(run + 1, a.S, a.N);
  const int cv = threadIdx.x % a.nv, rl = threadIdx.x / a.nv;
  const long long base = ((long long)b * a.N) * a.C + cv * V;
  for (int i = 0; i < seg.count; ++i) {
    const int begin = segment_begin(seg, i), lo = max(r0, begin), hi = min(r1, seg.end[i]);
    if (lo >= hi) continue;
    if ((i & 1) == 0) {
      zero_rows<T, V>(y + base, a, lo, hi, rl);
      continue;
    }
    merge_stats(a, seg, partial, b, i, stats);
    const int l = i >> 1;
    if (mean_out && lo == begin)
      for (int g = threadIdx.x; g < a.G; g += blockDim.x) {
        mean_out[((long long)b * a.L + l) * a.G + g] = stats[g].x;
        rstd_out[((long long)b * a.L + l) * a.G + g] = stats[g].y;
      }
    if (rl < a.RL) {
      float mean[V], scale[V], shift[V];
      const int wrow = a.weight_rows == 1 ? 0 : l;
#pragma unroll
      for (int c = 0; c < V; ++c) {
        const float2 s = stats[(cv * V + c) / a.cpg];
        mean[c] = s.x;
        scale[c] = s.y * __ldg(a.weight + wrow * a.C + cv * V + c);
        shift[c] = __ldg(a.bias + wrow * a.C + cv * V + c);
      }
      for (int r = lo + rl; r < hi; r += a.RL * kRows) {
        Word<T, V> w[kRows];
#pragma unroll
        for (int u = 0; u < kRows; ++u)
          if (r + u * a.RL < hi) w[u] = load_once<T, V>(x + base + (long long)(r + u * a.RL) * a.C);
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
          if (r + u * a.RL >= hi) break;
          float f[V];
          widen_word<T, V>(w[u], f);
#pragma unroll
          for (int c = 0; c < V; ++c) f[c] = activate(fmaf(f[c] - mean[c], scale[c], shift[c]), a.act);
          store_word<T, V>(y + base + (long long)(r + u * a.RL) * a.C, f);
        }
      }
    }
    __syncthreads();      // stats are overwritten for the next piece
  }
}

// ------------------------------------------------------------------------------------------------
// backward
// ------------------------------------------------------------------------------------------------
// What a thread knows of its channels.
template <int V>
struct Channels {
  float mean[V], rstd[V], gamma[V], beta[V];
  __device__ __forceinline__ void load(const GnArgs &a, const float *mean_in, const float *rstd_in, int b, int l, int cv) {
    const int wrow = a.weight_rows == 1 ? 0 : l;
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const long long g = ((long long)b * a.L + l) * a.G + (cv * V + c) / a.cpg;
      mean[c] = __ldg(mean_in + g);
      rstd[c] = __ldg(rstd_in + g);
      gamma[c] = __ldg(a.weight + wrow * a.C + cv * V + c);
      beta[c] = __ldg(a.bias + wrow * a.C + cv * V + c);
    }
  }
  // xhat and dz; z as the forward forms it, so that a ReLU's border falls the same way
  __device__ __forceinline__ void one(float x, float g, int c, int act, float &hat, float &dz) const {
    hat = (x - mean[c]) * rstd[c];
    dz = act == kNone ? g : activate_grad(g, fmaf(x - mean[c], rstd[c] * gamma[c], beta[c]), act);
  }
};

constexpr int kGradRows = 4;

// by_channel (B, pieces, C): sums of dz and of dz * xhat over the piece's rows; by_group (B, pieces, G): the same times gamma,
// over the group's channels.
template <typename T, int V>
__global__ void __launch_bounds__(max_threads(V))
gn_grad_stats_kernel(const T *__restrict__ grad_y, const T *__restrict__ x, GnArgs a,
                                     const float *__restrict__ mean_in, const float *__restrict__ rstd_in,
                                     float2 *__restrict__ by_channel, float2 *__restrict__ by_group) {
  extern __shared__ float2 chan[];       // (RL, C)
  __shared__ SegmentTable seg;
  if (threadIdx.x == 0) make_segments(seg, a.shapes, a.shape_stride, a.start, a.L, a.N);
  __syncthreads();
  const int b = blockIdx.x / a.S, run = blockIdx.x % a.S;
  const int r0 = run_begin(run, a.S, a.N), r1 = run_begin(run + 1, a.S, a.N);
  const int cv = threadIdx.x % a.nv, rl = threadIdx.x / a.nv;
  const long long base = ((long long)b * a.N) * a.C + cv * V;
  for (int i = 1; i < seg.count; i += 2) {
    const int lo = max(r0, seg.end[i - 1]), hi = min(r1, seg.end[i]);
    if (lo >= hi) continue;
    const int l = i >> 1, wrow = a.weight_rows == 1 ? 0 : l;
    if (rl < a.RL) {
      Channels<V> ch;
      ch.load(a, mean_in, rstd_in, b, l, cv);
      float s1[V] = {}, s2[V] = {};
      for (int r = lo + rl; r < hi; r += a.RL * kGradRows) {
        Word<T, V> xw[kGradRows], gw[kGradRows];
#pragma unroll
        for (int u = 0; u < kGradRows; ++u)
          if (r + u * a.RL < hi) {
            xw[u] = load_word<T, V>(x + base + (long long)(r + u * a.RL) * a.C);
            gw[u] = load_word<T, V>(grad_y + base + (long long)(r + u * a.RL) * a.C);
          }
#pragma unroll
        for (int u = 0; u < kGradRows; ++u) {
          if (r + u * a.RL >= hi) break;
          float xf[V], gf[V];
          widen_word<T, V>(xw[u], xf);
          widen_word<T, V>(gw[u], gf);
#pragma unroll
          for (int c = 0; c < V; ++c) {
            float hat, dz;
            ch.one(xf[c], gf[c], c, a.act, hat, dz);
            s1[c] += dz;
            s2[c] = fmaf(dz, hat, s2[c]);
          }
        }
      }
#pragma unroll
      for (int c = 0; c < V; ++c) chan[rl * a.C + cv * V + c] = make_float2(s1[c], s2[c]);
    }
    __syncthreads();
    const long long piece = (long long)b * pieces(a) + run + i;
    for (int c = threadIdx.x; c < a.C; c += blockDim.x) {
      float2 t = chan[c];
      for (int k = 1; k < a.RL; ++k) {
        t.x += chan[k * a.C + c].x;
        t.y += chan[k * a.C + c].y;
      }
      by_channel[piece * a.C + c] = t;
      const float w = __ldg(a.weight + wrow * a.C + c);
      chan[c] = make_float2(t.x * w, t.y * w);
    }
    __syncthreads();
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    for (int g = threadIdx.x >> 5; g < a.G; g += warps) {
      float u = 0.f, v = 0.f;
      for (int e = lane; e < a.cpg; e += 32) {
        u += chan[g * a.cpg + e].x;
        v += chan[g * a.cpg + e].y;
      }
      u = warp_sum(u);
      v = warp_sum(v);
      if (lane == 0) by_group[piece * a.G + g] = make_float2(u, v);
    }
    __syncthreads();
  }
}

// grad_x = rstd * (d - mean(d) - xhat * mean(d * xhat)), d = dz * gamma, means over the group.
template <typename T, int V>
__global__ void __launch_bounds__(max_threads(V))
gn_grad_apply_kernel(const T *__restrict__ grad_y, const T *__restrict__ x, GnArgs a,
                                     const float *__restrict__ mean_in, const float *__restrict__ rstd_in,
                                     const float2 *__restrict__ by_group, T *__restrict__ grad_x) {
  extern __shared__ float2 means[];      // (G)
  __shared__ SegmentTable seg;
  if (threadIdx.x == 0) make_segments(seg, a.shapes, a.shape_stride, a.start, a.L, a.N);
  __syncthreads();
  const int b = blockIdx.x / a.S, run = blockIdx.x % a.S;
  const int r0 = run_begin(run, a.S, a.N), r1 = run_begin(run + 1, a.S, a.N);
  const int cv = threadIdx.x % a.nv, rl = threadIdx.x / a.nv, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const long long base = ((long long)b * a.N) * a.C + cv * V;
  for (int i = 0; i < seg.count; ++i) {
    const int begin = segment_begin(seg, i), lo = max(r0, begin), hi = min(r1, seg.end[i]);
    if (lo >= hi) continue;
    if ((i & 1) == 0) {
      zero_rows<T, V>(grad_x + base, a, lo, hi, rl);
      continue;
    }
    const int first = run_of(begin, a.S, a.N), last = run_of(seg.end[i] - 1, a.S, a.N);
    const float inv = 1.f / ((float)(seg.end[i] - begin) * (float)a.cpg);
    const float2 *p = by_group + ((long long)b * pieces(a) + i) * a.G;
    for (int g = threadIdx.x >> 5; g < a.G; g += warps) {
      float u = 0.f, v = 0.f;
      for (int r = first + lane; r <= last; r += 32) {
        u += p[(long long)r * a.G + g].x;
        v += p[(long long)r * a.G + g].y;
      }
      u = warp_sum(u);
      v = warp_sum(v);
      if (lane == 0) means[g] = make_float2(u * inv, v * inv);
    }
    __syncthreads();
    if (rl < a.RL) {
      Channels<V> ch;
      ch.load(a, mean_in, rstd_in, b, i >> 1, cv);
      float c1[V], c2[V];
#pragma unroll
      for (int c = 0; c < V; ++c) {
        c1[c] = means[(cv * V + c) / a.cpg].x;
        c2[c] = means[(cv * V + c) / a.cpg].y;
      }
      for (int r = lo + rl; r < hi; r += a.RL * kGradRows) {
        Word<T, V> xw[kGradRows], gw[kGradRows];
#pragma unroll
        for (int u = 0; u < kGradRows; ++u)
          if (r + u * a.RL < hi) {
            xw[u] = load_once<T, V>(x + base + (long long)(r + u * a.RL) * a.C);
            gw[u] = load_once<T, V>(grad_y + base + (long long)(r + u * a.RL) * a.C);
          }
#pragma unroll
        for (int u = 0; u < kGradRows; ++u) {
          if (r + u * a.RL >= hi) break;
          float xf[V], gf[V];
          widen_word<T, V>(xw[u], xf);
          widen_word<T, V>(gw[u], gf);
#pragma unroll
          for (int c = 0; c < V; ++c) {
            float hat, dz;
            ch.one(xf[c], gf[c], c, a.act, hat, dz);
            xf[c] = ch.rstd[c] * (dz * ch.gamma[c] - c1[c] - hat * c2[c]);
          }
          store_word<T, V>(grad_x + base + (long long)(r + u * a.RL) * a.C, xf);
        }
      }
    }
    __syncthreads();
  }
}

// grad_weight, grad_bias (weight_rows, C): the sums of by_channel over images and pieces, and over levels where they share the
// weights, in a fixed order.  32 channels and 8 lanes over the pieces a CTA.
__global__ void __launch_bounds__(256)
gn_param_kernel(const float2 *__restrict__ by_channel, GnArgs a, int B, float *__restrict__ grad_weight, float *__restrict__ grad_bias) {
  __shared__ SegmentTable seg;
  __shared__ float2 part[8][32];
  if (threadIdx.x == 0) make_segments(seg, a.shapes, a.shape_stride, a.start, a.L, a.N);
  __syncthreads();
  const int lane = threadIdx.x & 31, k = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  const int l0 = a.weight_rows == 1 ? 0 : blockIdx.y, l1 = a.weight_rows == 1 ? a.L : l0 + 1;
  float2 t = make_float2(0.f, 0.f);
  if (c < a.C)
    for (int l = l0; l < l1; ++l) {
      const int lo = seg.end[2 * l], hi = seg.end[2 * l + 1];
      if (lo >= hi) continue;
      const int first = run_of(lo, a.S, a.N), n = run_of(hi - 1, a.S, a.N) - first + 1;
      const long long all = (long long)n * B;
#pragma unroll 4
      for (long long e = k; e < all; e += 8) {
        const int b = (int)(e / n), r = first + (int)(e - (long long)b * n);
        const float2 v = __ldg(by_channel + ((long long)b * pieces(a) + r + 2 * l + 1) * a.C + c);
        t.x += v.x;
        t.y += v.y;
      }
    }
  part[k][lane] = t;
  __syncthreads();
  if (k != 0 || c >= a.C) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    t.x += part[i][lane].x;
    t.y += part[i][lane].y;
  }
  grad_bias[blockIdx.y * a.C + c] = t.x;
  grad_weight[blockIdx.y * a.C + c] = t.y;
}

// ------------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------------
constexpr int kCtas = 148 * 4;

int runs_of(int B, int N, int C) {
  const int rows_at_once = std::max(1, 256 * 4 / C);                          // about what a CTA reads at a time
  const long long most = std::max(1, N / (rows_at_once * 4));
  return (int)std::max(1LL, std::min<long long>({(kCtas + B - 1) / B, most, N}));
}

struct Shape {
  GnArgs a;
  unsigned grid, threads;
  size_t chan_bytes;
};

template <int V>
Shape shape_of(GnArgs a, int B) {
  Shape s;
  a.cpg = a.C / a.G;
  a.nv = a.C / V;
  s.threads = a.nv <= 256 ? 256u : (unsigned)((a.nv + 31) / 32 * 32);
  a.RL = std::max(1, (int)s.threads / a.nv);
  a.S = runs_of(B, a.N, a.C);
  s.grid = (unsigned)(a.S * B);
  s.chan_bytes = (size_t)a.RL * a.C * sizeof(float2);
  s.a = a;
  return s;
}

template <typename T, int V>
cudaError_t forward(const T *x, GnArgs args, int B, T *y, float *mean, float *rstd, void *workspace, cudaStream_t st) {
  const Shape s = shape_of<V>(args, B);
  float2 *partial = static_cast<float2 *>(workspace);
  gn_stats_kernel<T, V><<<s.grid, s.threads, s.chan_bytes, st>>>(x, s.a, partial);
  gn_apply_kernel<T, V><<<s.grid, s.threads, s.a.G * sizeof(float2), st>>>(x, s.a, partial, y, mean, rstd);
  return cudaGetLastError();
}

template <typename T, int V>
cudaError_t backward(const T *grad_y, const T *x, GnArgs args, int B, const float *mean, const float *rstd, T *grad_x,
                     float *grad_weight, float *grad_bias, void *workspace, cudaStream_t st) {
  const Shape s = shape_of<V>(args, B);
  float2 *by_channel = static_cast<float2 *>(workspace);
  float2 *by_group = by_channel + (long long)B * (s.a.S + 2 * s.a.L + 1) * s.a.C;
  gn_grad_stats_kernel<T, V><<<s.grid, s.threads, s.chan_bytes, st>>>(grad_y, x, s.a, mean, rstd, by_channel, by_group);
  if (grad_x)
    gn_grad_apply_kernel<T, V><<<s.grid, s.threads, s.a.G * sizeof(float2), st>>>(grad_y, x, s.a, mean, rstd, by_group, grad_x);
  if (grad_weight)
    gn_param_kernel<<<dim3((s.a.C + 31) / 32, s.a.weight_rows), 256, 0, st>>>(by_channel, s.a, B, grad_weight, grad_bias);
  return cudaGetLastError();
}

// Elements a thread reads at a time: as many as divide the channels and as every address is aligned for, up to 16 bytes.
int vector_width(int C, size_t size, std::initializer_list<const void *> addresses) {
  int v = 16 / (int)size;
  while (v > 1) {
    bool ok = C % v == 0;
    for (const void *p : addresses) ok = ok && reinterpret_cast<uintptr_t>(p) % (v * size) == 0;
    if (ok) break;
    v /= 2;
  }
  return v;
}

GnArgs arguments(int N, int C, int G, const int64_t *shapes, int shape_stride, const int64_t *start, int L, const float *weight,
                 const float *bias, int weight_rows, float eps, int act) {
  GnArgs a = {};
  a.shapes = shapes; a.start = start; a.shape_stride = shape_stride;
  a.N = N; a.C = C; a.G = G; a.L = L; a.act = act;
  a.weight_rows = weight_rows; a.weight = weight; a.bias = bias; a.eps = eps;
  return a;
}

}  // namespace

long long group_norm_workspace(int B, int N, int C, int G, int L, bool backward) {
  if (B == 0 || N == 0) return 0;
  const long long pieces = (long long)B * (runs_of(B, N, C) + 2 * L + 1);
  return pieces * (backward ? C + G : G) * (long long)sizeof(float2);
}

#define DFA3D_GN(fn, v, ...)                                            \
  if (dtype == 0) {                                                     \
    using T = float;                                                    \
    if (v == 4) return fn<T, 4>(__VA_ARGS__);                           \
    if (v == 2) return fn<T, 2>(__VA_ARGS__);                           \
    return fn<T, 1>(__VA_ARGS__);                                       \
  } else if (dtype == 1) {                                              \
    using T = __nv_bfloat16;                                            \
    if (v == 8) return fn<T, 8>(__VA_ARGS__);                           \
    if (v == 4) return fn<T, 4>(__VA_ARGS__);                           \
    if (v == 2) return fn<T, 2>(__VA_ARGS__);                           \
    return fn<T, 1>(__VA_ARGS__);                                       \
  } else {                                                              \
    using T = __half;                                                   \
    if (v == 8) return fn<T, 8>(__VA_ARGS__);                           \
    if (v == 4) return fn<T, 4>(__VA_ARGS__);                           \
    if (v == 2) return fn<T, 2>(__VA_ARGS__);                           \
    return fn<T, 1>(__VA_ARGS__);                                       \
  }

cudaError_t launch_group_norm_forward(const void *x, int dtype, int B, int N, int C, int G, const int64_t *shapes,
                                      int shape_stride, const int64_t *start, int L, const float *weight, const float *bias,
                                      int weight_rows, float eps, int act, void *y, float *mean, float *rstd, void *workspace,
                                      cudaStream_t s) {
  const GnArgs a = arguments(N, C, G, shapes, shape_stride, start, L, weight, bias, weight_rows, eps, act);
  const int v = vector_width(C, dtype == 0 ? 4 : 2, {x, y});
  DFA3D_GN(forward, v, (const T *)x, a, B, (T *)y, mean, rstd, workspace, s)
}

cudaError_t launch_group_norm_backward(const void *grad_y, const void *x, int dtype, int B, int N, int C, int G,
                                       const int64_t *shapes, int shape_stride, const int64_t *start, int L, const float *weight,
                                       const float *bias, int weight_rows, const float *mean, const float *rstd, int act,
                                       void *grad_x, float *grad_weight, float *grad_bias, void *workspace, cudaStream_t s) {
  const GnArgs a = arguments(N, C, G, shapes, shape_stride, start, L, weight, bias, weight_rows, 0.f, act);
  const int v = vector_width(C, dtype == 0 ? 4 : 2, {x, grad_y, grad_x ? grad_x : x});
  DFA3D_GN(backward, v, (const T *)grad_y, (const T *)x, a, B, mean, rstd, (T *)grad_x, grad_weight, grad_bias, workspace, s)
}

}  // namespace dfa3d
