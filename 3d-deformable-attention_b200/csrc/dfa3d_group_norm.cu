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
// so that nothing is lost where the mean is large against the spread, not even where the mean's square exceeds 32 bits; a group's
// sum of squares has to fit them (beyond, rstd is 0 and the result act(beta), as in any 32-bit computation of the variance).
// Threads, warps and tiles are merged in a fixed order: a result is the same bits in every run.
//
// Three launches each way: statistics of tiles of rows; a warp for every group of a level of an image merges its tiles' parts;
// the result.  They follow one another as programmatic dependent launches, so that the third has its rows on the way while the
// second runs.  All tiles of a launch are resident at once (with up to 444 images; 296 or 148 for words of two channels or one), and
// the third walks each from its end, whose rows the first has left in L2 (126 MB).  Beyond, a tile is an image.
//
// Forwards of images of up to 256 rows of 1024 channels (1024 of 256) are one launch: a cluster of CTAs has a level of an image.
//
// 6 x 30 825 x 256, 32 groups, 4 levels: fp32 (189 MB) forward 96 us, backward 156; bf16 50 and 84; 6 x 920 x 256 fp32 11 and 11.
// The result's launch runs at the rate of a copy (57 us for 378 MB, the same with rows from L2 or not), the fp32 statistics at
// 5.6 TB/s; the bf16 ones take 23 us for 95 MB, 15 at that rate and the level table, the first loads and the reduction at the end
// (arithmetic on two values at once, or 12 and 16 words in flight: 1 %).  Measured against it, fp32 forward / backward: one launch
// that walks the images in batches with a barrier of the grid after each 257 / 287 (each barrier leaves every SM waiting through the
// merge); launches that form the statistics of one batch and the results of the one before 129 to 220 / 241 to 494; tiles of both
// kinds from one queue 146 forward; batches that fit L2, one after the other, 102 / 178; rows one chunk ahead through shared memory
// 107 / 167; merges by the CTAs of the third launch instead of a second one 110 / 170; two to six waves of tiles, bf16 forward 54 to 74.
#include <algorithm>
#include <cfloat>

#include "dfa3d_launch.h"
#include "dfa3d_rowvec.cuh"
#include "dfa3d_segments.h"

namespace dfa3d {
namespace {

enum Act { kNone = 0, kRelu = 1, kSilu = 2 };

// Threads of a CTA: at least as many as a row has words of V channels.
template <int V> constexpr int kThreads = V == 4 ? 256 : 1024 / V;
// CTAs an SM: what the registers of a thread's rows leave.
template <int V> constexpr int kResident = V == 4 ? 3 : V;
// Words of a thread in flight, and of each of two tensors.
constexpr int kAhead = 8, kGradAhead = 4;
// Below it a factor of the gradient has lost some of its 24 bits, or is about to: 2^24 times the smallest normal number.
constexpr float kSmallestFactor = FLT_MIN * 16777216.f;
// ... of the two that are only read: 8-byte words leave registers for more (bf16 backward 84 us; four words and four CTAs an SM 86).
template <typename T, int V> constexpr int kGradStatsAhead = V == 4 && sizeof(T) == 2 ? 8 : kGradAhead;

struct GnArgs {
  const int64_t *shapes, *start;     // level table, or null: one level
  int shape_stride;
  int B, N, C, G, L, act;
  int weight_rows;                   // 1, or L: weights of each level's own
  const float *weight, *bias;
  float eps;
  int cpg, V, nv, RL;                // channels a group, a word; words a row, rows a CTA reads at a time
  int R, tiles, entries;             // rows of a tile; tiles and pieces of an image
  Divisor by_r, by_tiles, by_nv, by_per, by_groups, by_levels;
  bool whole;                        // a word's channels are of one group: by_per divides by its words, else by its channels
  bool wide_params;                  // four weights at a time
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// over eight lanes
__device__ __forceinline__ float sum8(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  v += __shfl_xor_sync(0xffffffffu, v, 2);
  return v + __shfl_xor_sync(0xffffffffu, v, 4);
}

__device__ __forceinline__ float sigmoid(float z) { return __fdividef(1.f, 1.f + __expf(-z)); }
template <bool ACT>
__device__ __forceinline__ float activate(float z, int act) {
  if (!ACT) return z;
  if (act == kRelu) return z <= 0.f ? 0.f : z;                       // a NaN passes, as in torch
  return z * sigmoid(z);
}
// dz of dy
template <bool ACT>
__device__ __forceinline__ float activate_grad(float g, float z, int act) {
  if (!ACT) return g;
  if (act == kRelu) return z <= 0.f ? 0.f : g;
  const float s = sigmoid(z);
  return g * s * fmaf(z, 1.f - s, 1.f);
}

// The launches of a call follow one another closely: each lets the next begin as its CTAs leave, and waits for the one before it
// with launch_wait() before it reads what that wrote.
__device__ __forceinline__ void launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void launch_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Every thread returns with the table complete.
__device__ __forceinline__ void make_table(SegmentTable &seg, const GnArgs &a) {
  if (threadIdx.x < 32) make_segments_warp(seg, a.shapes, a.shape_stride, a.start, a.L, a.N);
  __syncthreads();
}

// A thread's place in a CTA's rows: row lane rl, word cv; `at` elements behind the first word of a row of lane 0.
struct Place {
  int rl, cv;
  unsigned at;
  __device__ __forceinline__ Place(const GnArgs &a) {
    rl = quotient(threadIdx.x, a.by_nv);
    cv = threadIdx.x - rl * a.nv;
    at = (unsigned)(rl * a.C + cv * a.V);
  }
};

// The tile of a CTA: rows [r0, r1) of image b; the segment that its first row belongs to, or its last one.
struct Tile {
  int b, t, r0, r1, i;
  __device__ __forceinline__ Tile(const GnArgs &a, const SegmentTable &seg, bool last) {
    b = quotient(blockIdx.x, a.by_tiles);
    t = blockIdx.x - b * a.tiles;
    r0 = t * a.R;
    r1 = min(a.N, r0 + a.R);
    i = 0;
    while (seg.end[i] <= (last ? r1 - 1 : r0)) ++i;
  }
};

// A thread's next U words, RL rows (`step` elements) apart.  base, the row r of lane 0 and the row `end` are the same for the
// CTA; ALL: no lane's last word lies at or beyond `end`.
template <typename T, int V, int U, bool ONCE, bool ALL>
__device__ __forceinline__ void load_rows(const T *base, unsigned at, int r, int end, int RL, long long step, Word<T, V> (&w)[U]) {
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (ALL || r + u * RL < end) w[u] = ONCE ? load_once<T, V>(base + u * step + at) : load_word<T, V>(base + u * step + at);
}

template <typename T, int V>
__device__ __forceinline__ void zero_rows(T *base, unsigned at, int r, int end, int RL, long long step) {
  const float zero[V] = {};
  for (; r < end; r += RL, base += step) store_word<T, V>(base + at, zero);
}

// The groups of a thread's channels; their weights.
template <int V>
__device__ __forceinline__ void groups_of(const GnArgs &a, int cv, int (&g)[V]) {
#pragma unroll
  for (int c = 0; c < V; ++c) g[c] = a.whole ? (c == 0 ? quotient(cv, a.by_per) : g[0]) : quotient(cv * V + c, a.by_per);
}
template <int V>
__device__ __forceinline__ void params_of(const GnArgs &a, const float *p, float (&f)[V]) {
  if constexpr (V == 4) {
    if (a.wide_params) {
      const float4 t = __ldg(reinterpret_cast<const float4 *>(p));
      f[0] = t.x; f[1] = t.y; f[2] = t.z; f[3] = t.w;
      return;
    }
  }
#pragma unroll
  for (int c = 0; c < V; ++c) f[c] = __ldg(p + c);
}

// ------------------------------------------------------------------------------------------------
// forward
// ------------------------------------------------------------------------------------------------
// m2 and what two parts' means, `delta` apart, add to it, `cross` = na nb / (na + nb).  A part without values (cross = 0) adds
// nothing: its mean is 0 and delta the other's mean, whose square may not fit 32 bits (infinity times 0 is NaN).
__device__ __forceinline__ float squares(float delta, float cross, float m2) {
  return cross > 0.f ? fmaf(delta * delta, cross, m2) : m2;
}

// Number, mean and sum of squares around it, of a thread's values of each of its channels.
template <int V>
struct Moments {
  float n = 0.f, mean[V] = {}, m2[V] = {};
  // U rows more, of which those before `have` count (all of them if ALL)
  template <typename T, int U, bool ALL>
  __device__ __forceinline__ void add(const Word<T, V> (&w)[U], int have) {
    float s[V] = {}, q[V] = {}, f[V];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (ALL || u < have) {
        widen_word<T, V>(w[u], f);
#pragma unroll
        for (int c = 0; c < V; ++c) s[c] += f[c];
      }
    const float nc = ALL ? (float)U : (float)have, inv = ALL ? 1.f / U : __fdividef(1.f, nc);
    const float total = n + nc, part = __fdividef(nc, total), cross = n * part;
#pragma unroll
    for (int c = 0; c < V; ++c) s[c] *= inv;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (ALL || u < have) {
        widen_word<T, V>(w[u], f);
#pragma unroll
        for (int c = 0; c < V; ++c) {
          f[c] -= s[c];
          q[c] = fmaf(f[c], f[c], q[c]);
        }
      }
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const float delta = s[c] - mean[c];
      mean[c] = fmaf(delta, part, mean[c]);
      m2[c] += squares(delta, cross, q[c]);
    }
    n = total;
  }
};

// Mean and sum of squares around it of a group's values in `rows` rows from `base` on (the CTA's): dst (G).  Ends with a barrier.
template <typename T, int V>
__device__ __forceinline__ void moments_of_piece(const T *base, int rows, const GnArgs &a, const Place &at, float2 *chan, float *count,
                                                 float2 *dst) {
  constexpr int U = kAhead;
  const long long step = (long long)a.RL * a.C;
  // a thread's channels are of one group where V divides it: one entry for all of them, or one for each
  const int lane = threadIdx.x & 31, sub = lane & 7, width = a.whole ? a.nv : a.C, per = (int)a.by_per.d;
  if (at.rl < a.RL) {
    Moments<V> k;
    Word<T, V> w[U];
    int r = 0;
    for (; r + U * a.RL <= rows; r += U * a.RL, base += U * step) {
      load_rows<T, V, U, false, true>(base, at.at, r, rows, a.RL, step, w);
      k.template add<T, U, true>(w, U);
    }
    if (r + at.rl < rows) {
      load_rows<T, V, U, false, false>(base, at.at, r + at.rl, rows, a.RL, step, w);
      int have = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) have += r + at.rl + u * a.RL < rows;
      k.template add<T, U, false>(w, have);
    }
    if (a.whole) {
      float m = 0.f, q = 0.f;
#pragma unroll
      for (int c = 0; c < V; ++c) m += k.mean[c];
      m *= 1.f / V;
#pragma unroll
      for (int c = 0; c < V; ++c) q += fmaf((k.mean[c] - m) * (k.mean[c] - m), k.n, k.m2[c]);
      chan[at.rl * width + at.cv] = make_float2(m, q);
    } else {
#pragma unroll
      for (int c = 0; c < V; ++c) chan[at.rl * width + at.cv * V + c] = make_float2(k.mean[c], k.m2[c]);
    }
    if (at.cv == 0) count[at.rl] = a.whole ? k.n * V : k.n;
  }
  __syncthreads();
  // eight lanes have a group
  const float inv_n = __fdividef(1.f, (float)rows * (float)a.cpg);
  const int l0 = quotient(sub, a.by_per), j0 = sub - l0 * per, dl = quotient(8, a.by_per), dj = 8 - dl * per;
  for (int g0 = (threadIdx.x >> 5) * 4; g0 < a.G; g0 += kThreads<V> / 8) {
    const int g = g0 + (lane >> 3), RL = g < a.G ? a.RL : 0;
    const float2 *entries = chan + g * per;
    float s = 0.f, q = 0.f;
#pragma unroll 1
    for (int l = l0, j = j0; l < RL; l += dl) {
      s = fmaf(count[l], entries[l * width + j].x, s);
      j += dj;
      if (j >= per) j -= per, ++l;
    }
    const float m = sum8(s) * inv_n;
#pragma unroll 1
    for (int l = l0, j = j0; l < RL; l += dl) {
      const float2 v = entries[l * width + j];
      q += squares(v.x - m, count[l], v.y);
      j += dj;
      if (j >= per) j -= per, ++l;
    }
    q = sum8(q);
    if (sub == 0 && RL) dst[g] = make_float2(m, q);
  }
  __syncthreads();
}

// A tile's statistics into partial (B, entries, G), of each of its pieces.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads<V>, kResident<V>)
group_stats_kernel(const T *__restrict__ x, const GnArgs a, float2 *__restrict__ partial) {
  extern __shared__ float2 chan[];                       // a thread's channels
  __shared__ float count[kThreads<V>];                   // values that an entry of a row lane stands for
  __shared__ SegmentTable seg;
  launch_next();
  make_table(seg, a);
  Tile tile(a, seg, false);
  const Place at(a);
  for (int lo = tile.r0; lo < tile.r1; ++tile.i) {
    const int hi = min(tile.r1, seg.end[tile.i]), rows = hi - lo, from = lo;
    lo = hi;
    if (rows <= 0 || (tile.i & 1) == 0) continue;
    moments_of_piece<T, V>(x + ((long long)tile.b * a.N + from) * a.C, rows, a, at, chan, count,
                           partial + ((long long)tile.b * a.entries + tile.t + tile.i) * a.G);
  }
}

// A segment of an image, and the tiles that have a piece of it.
struct Span {
  int begin, end, from, to;
  __device__ __forceinline__ Span(const GnArgs &a, const SegmentTable &seg, int i) {
    begin = segment_begin(seg, i);
    end = seg.end[i];
    from = quotient(begin, a.by_r);
    to = end > begin ? quotient(end - 1, a.by_r) : from - 1;
  }
};

constexpr int kMergeThreads = 256;

// The group of a level of an image that a warp merges.
struct MergeTask {
  int b, l, g;
  bool mine;
  __device__ __forceinline__ MergeTask(const GnArgs &a, int task) {
    mine = task < a.B * a.L * a.G;
    const int q = quotient(task, a.by_groups);
    g = task - q * a.G;
    b = quotient(q, a.by_levels);
    l = q - b * a.L;
  }
};

// Merges the tiles' parts: mean, rstd (B, L, G).
__global__ void __launch_bounds__(kMergeThreads)
group_merge_kernel(const GnArgs a, const float2 *partial, float *__restrict__ mean_out, float *__restrict__ rstd_out) {
  constexpr int U = 8;
  __shared__ SegmentTable seg;
  launch_next();
  make_table(seg, a);
  const int task = blockIdx.x * (kMergeThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const MergeTask k(a, task);
  launch_wait();
  if (!k.mine) return;
  const Span s(a, seg, 2 * k.l + 1);
  const float2 *src = partial + ((long long)k.b * a.entries + 2 * k.l + 1) * a.G + k.g;
  float n = 0.f, mean = 0.f, m2 = 0.f;
  for (int t = s.from + lane; t <= s.to; t += 32 * U) {
    float2 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (t + 32 * u <= s.to) v[u] = __ldcg(src + (long long)(t + 32 * u) * a.G);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int tu = t + 32 * u;
      if (tu > s.to) break;
      const float nb = (float)(min(s.end, (tu + 1) * a.R) - max(s.begin, tu * a.R)) * (float)a.cpg, total = n + nb;
      const float part = __fdividef(nb, total), delta = v[u].x - mean;
      mean = fmaf(delta, part, mean);
      m2 += squares(delta, n * part, v[u].y);
      n = total;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float nb = __shfl_down_sync(0xffffffffu, n, o), mb = __shfl_down_sync(0xffffffffu, mean, o);
    const float qb = __shfl_down_sync(0xffffffffu, m2, o), total = n + nb, delta = mb - mean;
    const float part = total > 0.f ? __fdividef(nb, total) : 0.f;
    mean = fmaf(delta, part, mean);
    m2 += squares(delta, n * part, qb);
    n = total;
  }
  if (lane == 0) {
    mean_out[task] = mean;
    rstd_out[task] = n > 0.f ? rsqrtf(__fdividef(m2, n) + a.eps) : 0.f;
  }
}

// y = act((x - mean) * rstd * weight + bias).  A tile is walked from its end: what the statistics read last is still in L2.
template <typename T, int V, bool ACT>
__global__ void __launch_bounds__(kThreads<V>, kResident<V>)
group_apply_kernel(const T *__restrict__ x, const GnArgs a, const float *mean_in, const float *rstd_in, T *__restrict__ y) {
  constexpr int U = kAhead;
  __shared__ SegmentTable seg;
  launch_next();
  make_table(seg, a);
  Tile tile(a, seg, true);
  const Place at(a);
  const long long step = (long long)a.RL * a.C;
  const int chunk = U * a.RL;
  int group[V];
  groups_of<V>(a, at.cv, group);
  bool waited = false;
  for (int hi = tile.r1; hi > tile.r0; --tile.i) {
    const int lo = max(tile.r0, segment_begin(seg, tile.i)), all = hi - lo, rows = at.rl < a.RL ? all : 0, l = tile.i >> 1;
    if (all <= 0) continue;
    hi = lo;
    int r = (all - 1) / chunk * chunk;                   // the last chunk of rows, which may be a short one
    const long long first = ((long long)tile.b * a.N + lo + r) * a.C;
    const T *in = x + first;
    T *out = y + first;
    Word<T, V> w[U];
    // on its way before the statistics are there
    if (tile.i & 1) load_rows<T, V, U, true, false>(in, at.at, r + at.rl, rows, a.RL, step, w);
    if (!waited) launch_wait();
    waited = true;
    if (rows <= 0) continue;
    if ((tile.i & 1) == 0) {
      zero_rows<T, V>(out - (long long)r * a.C, at.at, at.rl, rows, a.RL, step);
      continue;
    }
    float mean[V], scale[V], shift[V];
    const int w0 = (a.weight_rows == 1 ? 0 : l) * a.C + at.cv * V;
    const long long g0 = ((long long)tile.b * a.L + l) * a.G;
    params_of<V>(a, a.weight + w0, scale);
    params_of<V>(a, a.bias + w0, shift);
#pragma unroll
    for (int c = 0; c < V; ++c) {
      mean[c] = __ldcg(mean_in + g0 + group[c]);
      scale[c] *= __ldcg(rstd_in + g0 + group[c]);
    }
    auto store = [&](int u) {
      float f[V];
      widen_word<T, V>(w[u], f);
#pragma unroll
      for (int c = 0; c < V; ++c) f[c] = activate<ACT>(fmaf(f[c] - mean[c], scale[c], shift[c]), a.act);
      store_once<T, V>(out + u * step + at.at, f);
    };
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (r + at.rl + u * a.RL < rows) store(u);
    for (r -= chunk; r >= 0; r -= chunk) {
      in -= U * step;
      out -= U * step;
      load_rows<T, V, U, true, true>(in, at.at, r, rows, a.RL, step, w);
#pragma unroll
      for (int u = 0; u < U; ++u) store(u);
    }
  }
}

// ------------------------------------------------------------------------------------------------
// small images: one launch
// ------------------------------------------------------------------------------------------------
// A cluster of CTAs has a level of an image: each keeps the sums of its own rows in shared memory, reads those of the others behind a
// barrier of the cluster, and goes through its rows, which the L1 still has, once more.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ float2 of_rank(const float2 *p, int rank) {
  unsigned at;
  float2 v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((unsigned)__cvta_generic_to_shared(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
  return v;
}

constexpr int kMaxCluster = 8;

// A CTA's rows [r0, r1) of level l of image b: `per` rows to each of `size` CTAs, as far as the level goes.
struct Share {
  int b, l, rank, size, begin, end, per, r0, r1;
  __device__ __forceinline__ Share(const GnArgs &a, const SegmentTable &seg) {
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(size));
    const int q = ((int)blockIdx.x - rank) / size;
    b = quotient(q, a.by_levels);
    l = q - b * a.L;
    begin = segment_begin(seg, 2 * l + 1);
    end = seg.end[2 * l + 1];
    per = (end - begin + size - 1) / size;
    r0 = min(begin + rank * per, end);
    r1 = min(r0 + per, end);
  }
  __device__ __forceinline__ int rows_of(int j) const { return max(0, min(end - begin - j * per, per)); }
};

// The rows of no level before level l, and behind the last one.
template <typename T, int V>
__device__ __forceinline__ void zero_gaps(const GnArgs &a, const SegmentTable &seg, const Share &k, const Place &at, T *out) {
  if (at.rl >= a.RL) return;
  for (int i = 2 * k.l; i <= 2 * a.L; i += 2 * (a.L - k.l)) {
    const int begin = segment_begin(seg, i), first = k.rank * a.RL;
    zero_rows<T, V>(out + ((long long)k.b * a.N + begin + first) * a.C, at.at, first + at.rl, seg.end[i] - begin, k.size * a.RL,
                    (long long)k.size * a.RL * a.C);
    if (k.l + 1 < a.L) break;
  }
}

template <typename T, int V, bool ACT>
__global__ void __launch_bounds__(kThreads<V>, kResident<V>)
group_image_kernel(const T *__restrict__ x, const GnArgs a, float *__restrict__ mean_out, float *__restrict__ rstd_out,
                   T *__restrict__ y) {
  constexpr int U = kAhead;
  extern __shared__ float2 chan[];
  __shared__ float count[kThreads<V>];
  __shared__ SegmentTable seg;
  float2 *own = chan + kThreads<V> * V, *merged = own + a.G;      // (G) each: of the CTA's rows; mean and rstd of the level
  make_table(seg, a);
  const Share k(a, seg);
  const Place at(a);
  const int rows = k.r1 - k.r0;
  const long long first = ((long long)k.b * a.N + k.r0) * a.C, step = (long long)a.RL * a.C;
  moments_of_piece<T, V>(x + first, rows, a, at, chan, count, own);
  cluster_arrive();
  cluster_wait();
  for (int g = threadIdx.x; g < a.G; g += kThreads<V>) {
    float2 v[kMaxCluster];
#pragma unroll
    for (int j = 0; j < kMaxCluster; ++j)
      if (j < k.size) v[j] = of_rank(own + g, j);
    float n = 0.f, mean = 0.f, m2 = 0.f;
#pragma unroll
    for (int j = 0; j < kMaxCluster; ++j)
      if (j < k.size && k.rows_of(j) > 0) {
        const float nb = (float)k.rows_of(j) * (float)a.cpg, total = n + nb, part = __fdividef(nb, total), delta = v[j].x - mean;
        mean = fmaf(delta, part, mean);
        m2 += squares(delta, n * part, v[j].y);
        n = total;
      }
    const float rstd = n > 0.f ? rsqrtf(__fdividef(m2, n) + a.eps) : 0.f;
    merged[g] = make_float2(mean, rstd);
    if (k.rank == 0 && mean_out) {
      const long long to = ((long long)k.b * a.L + k.l) * a.G + g;
      mean_out[to] = mean;
      rstd_out[to] = rstd;
    }
  }
  cluster_arrive();                                      // done with the others' shared memory
  __syncthreads();
  if (at.rl < a.RL) {
    int group[V];
    float mean[V], scale[V], shift[V];
    groups_of<V>(a, at.cv, group);
    const int w0 = (a.weight_rows == 1 ? 0 : k.l) * a.C + at.cv * V;
    params_of<V>(a, a.weight + w0, scale);
    params_of<V>(a, a.bias + w0, shift);
#pragma unroll
    for (int c = 0; c < V; ++c) {
      mean[c] = merged[group[c]].x;
      scale[c] *= merged[group[c]].y;
    }
    const T *in = x + first;
    T *out = y + first;
    for (int r = at.rl; r < rows; r += U * a.RL, in += U * step, out += U * step) {
      Word<T, V> w[U];
      load_rows<T, V, U, false, false>(in, at.at, r, rows, a.RL, step, w);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (r + u * a.RL >= rows) break;
        float f[V];
        widen_word<T, V>(w[u], f);
#pragma unroll
        for (int c = 0; c < V; ++c) f[c] = activate<ACT>(fmaf(f[c] - mean[c], scale[c], shift[c]), a.act);
        store_word<T, V>(out + u * step + at.at, f);
      }
    }
  }
  zero_gaps<T, V>(a, seg, k, at, y);
  cluster_wait();
}

// ------------------------------------------------------------------------------------------------
// backward
// ------------------------------------------------------------------------------------------------
// Sums of dz and of dz * xhat over a tile's pieces: by_channel (B, entries, C), and times gamma over a group's channels: by_group
// (B, entries, G).
template <typename T, int V, bool ACT>
__global__ void __launch_bounds__(kThreads<V>, kResident<V>)
group_grad_stats_kernel(const T *__restrict__ grad_y, const T *__restrict__ x, const GnArgs a, const float *__restrict__ mean_in,
                        const float *__restrict__ rstd_in, float2 *__restrict__ by_channel, float2 *__restrict__ by_group) {
  constexpr int U = kGradStatsAhead<T, V>;
  extern __shared__ float2 chan[];                       // (RL, C)
  __shared__ SegmentTable seg;
  launch_next();
  make_table(seg, a);
  Tile tile(a, seg, false);
  const Place at(a);
  const long long step = (long long)a.RL * a.C;
  int group[V];
  groups_of<V>(a, at.cv, group);
  for (int lo = tile.r0; lo < tile.r1; ++tile.i) {
    const int hi = min(tile.r1, seg.end[tile.i]), rows = hi - lo, from = lo, l = tile.i >> 1;
    lo = max(lo, hi);
    if (rows <= 0 || (tile.i & 1) == 0) continue;
    const float *gamma = a.weight + (a.weight_rows == 1 ? 0 : l) * a.C, *beta = a.bias + (gamma - a.weight);
    const long long g0 = ((long long)tile.b * a.L + l) * a.G;
    if (at.rl < a.RL) {
      const long long first = ((long long)tile.b * a.N + from) * a.C;
      const T *xin = x + first, *gin = grad_y + first;
      float mean[V], scale[V], shift[V], s1[V] = {}, s2[V] = {};
      if (ACT) {
        params_of<V>(a, gamma + at.cv * V, scale);
        params_of<V>(a, beta + at.cv * V, shift);
      }
#pragma unroll
      for (int c = 0; c < V; ++c) {
        mean[c] = __ldg(mean_in + g0 + group[c]);
        if (ACT) scale[c] *= __ldg(rstd_in + g0 + group[c]);      // as the forward forms it
      }
      Word<T, V> xw[U], gw[U];
      auto add = [&](int u) {
        float xf[V], gf[V];
        widen_word<T, V>(xw[u], xf);
        widen_word<T, V>(gw[u], gf);
#pragma unroll
        for (int c = 0; c < V; ++c) {
          const float centred = xf[c] - mean[c];
          const float dz = ACT ? activate_grad<ACT>(gf[c], fmaf(centred, scale[c], shift[c]), a.act) : gf[c];
          s1[c] += dz;
          s2[c] = fmaf(dz, centred, s2[c]);
        }
      };
      int r = 0;
      for (; r + U * a.RL <= rows; r += U * a.RL, xin += U * step, gin += U * step) {
        load_rows<T, V, U, false, true>(xin, at.at, r, rows, a.RL, step, xw);
        load_rows<T, V, U, false, true>(gin, at.at, r, rows, a.RL, step, gw);
#pragma unroll
        for (int u = 0; u < U; ++u) add(u);
      }
      load_rows<T, V, U, false, false>(xin, at.at, r + at.rl, rows, a.RL, step, xw);
      load_rows<T, V, U, false, false>(gin, at.at, r + at.rl, rows, a.RL, step, gw);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (r + at.rl + u * a.RL < rows) add(u);
#pragma unroll
      for (int c = 0; c < V; ++c) chan[at.rl * a.C + at.cv * V + c] = make_float2(s1[c], s2[c]);
    }
    __syncthreads();
    const long long entry = (long long)tile.b * a.entries + tile.t + tile.i;
    for (int c = threadIdx.x; c < a.C; c += kThreads<V>) {
      float2 s = chan[c];
      for (int j = 1; j < a.RL; ++j) {
        s.x += chan[j * a.C + c].x;
        s.y += chan[j * a.C + c].y;
      }
      s.y *= __ldg(rstd_in + g0 + c / a.cpg);
      by_channel[entry * a.C + c] = s;
      const float w = __ldg(gamma + c);
      chan[c] = make_float2(s.x * w, s.y * w);
    }
    __syncthreads();
    const int lane = threadIdx.x & 31, sub = lane & 7;
    for (int q0 = (threadIdx.x >> 5) * 4; q0 < a.G; q0 += kThreads<V> / 8) {      // eight lanes have a group
      const int g = q0 + (lane >> 3);
      float u = 0.f, v = 0.f;
      if (g < a.G)
        for (int c = g * a.cpg + sub; c < (g + 1) * a.cpg; c += 8) {
          u += chan[c].x;
          v += chan[c].y;
        }
      u = sum8(u);
      v = sum8(v);
      if (sub == 0 && g < a.G) by_group[entry * a.G + g] = make_float2(u, v);
    }
    __syncthreads();
  }
}

// The first `merges` CTAs: means over a group of a level of an image, by a warp: means (B, L, G).  The others: by_channel summed over
// a level's tiles into by_level (B, L, C), 32 channels a CTA, a warp every eighth tile.
__global__ void __launch_bounds__(kMergeThreads)
group_grad_merge_kernel(const GnArgs a, int merges, const float2 *by_group, const float2 *by_channel, float2 *__restrict__ means,
                        float2 *__restrict__ by_level) {
  constexpr int U = 8, kWarps = kMergeThreads / 32;
  __shared__ SegmentTable seg;
  __shared__ float2 part[kMergeThreads];
  launch_next();
  make_table(seg, a);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  launch_wait();
  const bool channels = (int)blockIdx.x >= merges;
  const int chunk = ((int)blockIdx.x - merges) % ((a.C + 31) / 32), c = chunk * 32 + lane;
  const int level = channels ? ((int)blockIdx.x - merges) / ((a.C + 31) / 32) : 0;      // of the B * L
  const MergeTask k(a, channels ? level * a.G : (int)blockIdx.x * kWarps + warp);
  float u = 0.f, v = 0.f;
  if (k.mine) {
    const Span s(a, seg, 2 * k.l + 1);
    const long long entry = (long long)k.b * a.entries + 2 * k.l + 1;
    const float2 *src = channels ? by_channel + entry * a.C + c : by_group + entry * a.G + k.g;
    const int first = channels ? warp : lane, every = channels ? kWarps : 32, width = channels ? a.C : a.G;
    if (!channels || c < a.C)
      for (int t = s.from + first; t <= s.to; t += every * U) {
        float2 p[U];
#pragma unroll
        for (int j = 0; j < U; ++j)
          if (t + every * j <= s.to) p[j] = __ldcg(src + (long long)(t + every * j) * width);
#pragma unroll
        for (int j = 0; j < U; ++j)
          if (t + every * j <= s.to) {
            u += p[j].x;
            v += p[j].y;
          }
      }
    if (!channels) {
      u = warp_sum(u);
      v = warp_sum(v);
      const float n = (float)(s.end - s.begin) * (float)a.cpg;
      if (lane == 0) means[(k.b * a.L + k.l) * a.G + k.g] = n > 0.f ? make_float2(__fdividef(u, n), __fdividef(v, n)) : make_float2(0.f, 0.f);
    }
  }
  if (!channels) return;
  part[threadIdx.x] = make_float2(u, v);
  __syncthreads();
  if (warp == 0 && c < a.C) {
#pragma unroll
    for (int j = 1; j < kWarps; ++j) {
      u += part[j * 32 + lane].x;
      v += part[j * 32 + lane].y;
    }
    by_level[(long long)level * a.C + c] = make_float2(u, v);
  }
}

// grad_weight, grad_bias (weight_rows, C): by_level summed over images, and over levels where they share the weights.  32 columns a
// CTA, whose warps take the (image, level)s in turn.
template <int WARPS>
__device__ __forceinline__ void parameter_sums(const GnArgs &a, const float2 *by_level, int chunk, float *grad_weight,
                                               float *grad_bias) {
  __shared__ float2 part[WARPS][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, column = chunk * 32 + lane;
  const int row = column / a.C, c = column - row * a.C, every = a.weight_rows == 1 ? 1 : a.L, terms = a.B * a.L / every;
  const bool mine = column < a.weight_rows * a.C;
  float2 s = make_float2(0.f, 0.f);
  if (mine)
#pragma unroll 4
    for (int t = warp; t < terms; t += WARPS) {
      const float2 v = __ldcg(by_level + ((long long)t * every + row) * a.C + c);
      s.x += v.x;
      s.y += v.y;
    }
  part[warp][lane] = s;
  __syncthreads();
  if (warp != 0 || !mine) return;
#pragma unroll
  for (int w = 1; w < WARPS; ++w) {
    s.x += part[w][lane].x;
    s.y += part[w][lane].y;
  }
  grad_bias[column] = s.x;
  grad_weight[column] = s.y;
}

// A thread's channels of a piece's rows, one by one, where rstd^2 mean(d * xhat) does not fit a normal number: xhat is formed first.
template <typename T, bool ACT>
__device__ __noinline__ void grad_in_steps(const T *grad_y, const T *x, T *grad_x, const GnArgs &a, long long first, int rl, int rows,
                                           int channel, int count, int w0, long long g0, const float *mean_in, const float *rstd_in,
                                           const float2 *means) {
  for (int c = 0; c < count; ++c) {
    const long long g = g0 + (channel + c) / a.cpg;
    const float mean = __ldg(mean_in + g), rstd = __ldg(rstd_in + g), scale = __ldg(a.weight + w0 + c) * rstd;
    const float shift = ACT ? __ldg(a.bias + w0 + c) : 0.f;
    const float2 m = __ldcg(means + g);
    for (int r = rl; r < rows; r += a.RL) {
      const long long at = first + (long long)r * a.C + channel + c;
      const float centred = wide(x[at]) - mean, dy = wide(grad_y[at]);
      const float dz = ACT ? activate_grad<ACT>(dy, fmaf(centred, scale, shift), a.act) : dy;
      grad_x[at] = narrow<T>(fmaf(dz, scale, -fmaf(centred * rstd, rstd * m.y, rstd * m.x)));
    }
  }
}

// grad_x = rstd * (d - mean(d) - xhat * mean(d * xhat)), d = dz * gamma, means over the group; the CTAs beyond its
// `tiles` form the parameters' gradients.
template <typename T, int V, bool ACT>
__global__ void __launch_bounds__(kThreads<V>, kResident<V>)
group_grad_apply_kernel(const T *__restrict__ grad_y, const T *__restrict__ x, const __grid_constant__ GnArgs a, int tiles,
                        const float *__restrict__ mean_in, const float *__restrict__ rstd_in, const float2 *means,
                        const float2 *by_level, T *__restrict__ grad_x, float *grad_weight, float *grad_bias) {
  constexpr int U = kGradAhead;
  __shared__ SegmentTable seg;
  const int beyond = (int)blockIdx.x - tiles;
  if (beyond >= 0) {
    launch_wait();
    parameter_sums<kThreads<V> / 32>(a, by_level, beyond, grad_weight, grad_bias);
    return;
  }
  make_table(seg, a);
  Tile tile(a, seg, true);
  const Place at(a);
  const long long step = (long long)a.RL * a.C;
  const int chunk = U * a.RL;
  int group[V];
  groups_of<V>(a, at.cv, group);
  bool waited = false;
  for (int hi = tile.r1; hi > tile.r0; --tile.i) {
    const int lo = max(tile.r0, segment_begin(seg, tile.i)), all = hi - lo, rows = at.rl < a.RL ? all : 0, l = tile.i >> 1;
    if (all <= 0) continue;
    hi = lo;
    int r = (all - 1) / chunk * chunk;
    const long long first = ((long long)tile.b * a.N + lo + r) * a.C;
    const T *xin = x + first, *gin = grad_y + first;
    T *out = grad_x + first;
    Word<T, V> xw[U], gw[U];
    if (tile.i & 1) {
      load_rows<T, V, U, true, false>(xin, at.at, r + at.rl, rows, a.RL, step, xw);
      load_rows<T, V, U, true, false>(gin, at.at, r + at.rl, rows, a.RL, step, gw);
    }
    if (!waited) launch_wait();
    waited = true;
    if (rows <= 0) continue;
    if ((tile.i & 1) == 0) {
      zero_rows<T, V>(out - (long long)r * a.C, at.at, at.rl, rows, a.RL, step);
      continue;
    }
    // grad_x = dz * scale - (k1 + (x - mean) * k2).  With eps = 0 and next to no spread, or a wide one and small gradients,
    // k2 = rstd^2 mean(d * xhat) may not fit a normal number.
    bool fits = true;
    float mean[V], scale[V], shift[V], k1[V], k2[V];
    const int w0 = (a.weight_rows == 1 ? 0 : l) * a.C + at.cv * V;
    const long long g0 = ((long long)tile.b * a.L + l) * a.G;
    params_of<V>(a, a.weight + w0, scale);
    if (ACT) params_of<V>(a, a.bias + w0, shift);
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const float rstd = __ldg(rstd_in + g0 + group[c]);
      const float2 m = __ldcg(means + g0 + group[c]);
      mean[c] = __ldg(mean_in + g0 + group[c]);
      scale[c] *= rstd;
      k1[c] = rstd * m.x;
      k2[c] = rstd * rstd * m.y;
      const float y = fabsf(m.y), k = fabsf(k2[c]);
      if (y > 0.f && y <= FLT_MAX && !(k >= kSmallestFactor && k <= FLT_MAX)) fits = false;
    }
    if (!fits) {
      grad_in_steps<T, ACT>(grad_y, x, grad_x, a, ((long long)tile.b * a.N + lo) * a.C, at.rl, rows, at.cv * V, V, w0, g0, mean_in, rstd_in,
                            means);
      continue;
    }
    auto store = [&](int u) {
      float xf[V], gf[V];
      widen_word<T, V>(xw[u], xf);
      widen_word<T, V>(gw[u], gf);
#pragma unroll
      for (int c = 0; c < V; ++c) {
        const float centred = xf[c] - mean[c];
        const float dz = ACT ? activate_grad<ACT>(gf[c], fmaf(centred, scale[c], shift[c]), a.act) : gf[c];
        xf[c] = fmaf(dz, scale[c], -fmaf(centred, k2[c], k1[c]));
      }
      store_once<T, V>(out + u * step + at.at, xf);
    };
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (r + at.rl + u * a.RL < rows) store(u);
    for (r -= chunk; r >= 0; r -= chunk) {
      xin -= U * step;
      gin -= U * step;
      out -= U * step;
      load_rows<T, V, U, true, true>(xin, at.at, r, rows, a.RL, step, xw);
      load_rows<T, V, U, true, true>(gin, at.at, r, rows, a.RL, step, gw);
#pragma unroll
      for (int u = 0; u < U; ++u) store(u);
    }
  }
}

// ------------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------------
int threads_of(int V) { return V == 4 ? kThreads<4> : V == 2 ? kThreads<2> : kThreads<1>; }

int resident_of(int V) { return V == 4 ? kResident<4> : V == 2 ? kResident<2> : kResident<1>; }

// Rows of a tile: as many as make one full wave of CTAs of the whole call, but at least four of a thread, and one tile an image where
// there are more images than CTAs in a wave.  6 x 30 825 x 256 bf16 forward 49 us, at two waves 54, three 59; 40 000 x 256 fp32 32, 42, 49; 6 x 30 825 x 256 fp32 97,
// 97, 100 (backward 158, 155, 159).
int tile_rows(int B, int N, int C, int V) {
  const int RL = threads_of(V) / (C / V);
  const long long slots = 148LL * resident_of(V), tiles = std::max(1LL, slots / B);
  const long long rows = std::max((N + tiles - 1) / tiles, 4LL * RL);
  return (int)std::min<long long>(rows, N);
}

// CTAs of a cluster that has a level of an image in one launch, or 0 for three launches of tiles: up to eight, while a thread would
// have more than eight rows, and none where it would have more than 32 of eight.  us, one launch / three (host 6.4 / 11):
// 2 x 336 x 128 fp32 5.7 / 6.2, 375 x 256 6.7 / 6.2, 200 x 40 x 64 bf16 6.1 / 7.0, 2000 x 16 x 64 fp32 25 / 30, 6 x 920 x 256 10.5 / 10.3; with
// more rows 1600 x 256 bf16 11.0 / 8.3, 5800 x 64 15.4 / 9.1.  The backward stays with three: 23 / 12 at 6 x 920 x 256.
int cluster_size(int N, int C) {
  const int rows = 1024 / C;                             // that a CTA of any word reads at a time
  if (N > kMaxCluster * 32 * rows) return 0;
  int size = 1;
  while (size < kMaxCluster && N > size * 8 * rows) size *= 2;
  return size;
}

void complete(GnArgs &a, int V) {
  a.cpg = a.C / a.G;
  a.V = V;
  a.nv = a.C / V;
  a.RL = threads_of(V) / a.nv;
  a.R = tile_rows(a.B, a.N, a.C, V);
  a.tiles = (a.N + a.R - 1) / a.R;
  a.entries = a.tiles + 2 * a.L + 1;
  a.whole = a.cpg % V == 0;
  a.by_r = make_divisor(a.R);
  a.by_tiles = make_divisor(a.tiles);
  a.by_nv = make_divisor(a.nv);
  a.by_groups = make_divisor(a.G);
  a.by_levels = make_divisor(a.L);
  a.by_per = make_divisor(a.whole ? a.cpg / V : a.cpg);
  a.wide_params = a.C % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.weight) | reinterpret_cast<uintptr_t>(a.bias)) & 15) == 0;
}

template <typename... P, typename... A>
cudaError_t launch_with(void (*kernel)(P...), unsigned grid, int threads, size_t shared, cudaLaunchAttribute *at, int count,
                        cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = shared;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = count;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}
// A launch that may begin while the one before it in the sequence runs (`follows`).
template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), unsigned grid, int threads, size_t shared, bool follows, cudaStream_t st, A... args) {
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  return launch_with(kernel, grid, threads, shared, at, follows ? 1 : 0, st, args...);
}
// ... of clusters of `size` CTAs.
template <typename... P, typename... A>
cudaError_t launch_clusters(void (*kernel)(P...), unsigned grid, int size, int threads, size_t shared, cudaStream_t st, A... args) {
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = size;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  return launch_with(kernel, grid, threads, shared, at, 1, st, args...);
}
#define DFA3D_TRY(call) do { const cudaError_t rc_ = (call); if (rc_ != cudaSuccess) return rc_; } while (0)

unsigned merge_grid(const GnArgs &a) {
  return (unsigned)(((long long)a.B * a.L * a.G + kMergeThreads / 32 - 1) / (kMergeThreads / 32));
}

template <typename T, int V>
cudaError_t forward(const T *x, GnArgs a, T *y, float *mean, float *rstd, void *workspace, cudaStream_t st) {
  complete(a, V);
  if (const int size = cluster_size(a.N, a.C)) {
    auto all = a.act == kNone ? group_image_kernel<T, V, false> : group_image_kernel<T, V, true>;
    return launch_clusters(all, (unsigned)(a.B * a.L * size), size, kThreads<V>, sizeof(float2) * (kThreads<V> * V + 2 * a.G), st, x, a,
                           mean, rstd, y);
  }
  float2 *partial = static_cast<float2 *>(workspace);
  if (!mean) {                                           // nobody keeps them: behind the tiles' parts
    mean = reinterpret_cast<float *>(partial + (long long)a.B * a.entries * a.G);
    rstd = mean + (long long)a.B * a.L * a.G;
  }
  const unsigned grid = (unsigned)(a.B * a.tiles);
  DFA3D_TRY(launch(group_stats_kernel<T, V>, grid, kThreads<V>, sizeof(float2) * kThreads<V> * V, false, st, x, a, partial));
  DFA3D_TRY(launch(group_merge_kernel, merge_grid(a), kMergeThreads, 0, true, st, a, partial, mean, rstd));
  auto apply = a.act == kNone ? group_apply_kernel<T, V, false> : group_apply_kernel<T, V, true>;
  return launch(apply, grid, kThreads<V>, 0, true, st, x, a, mean, rstd, y);
}

template <typename T, int V>
cudaError_t backward(const T *grad_y, const T *x, GnArgs a, const float *mean, const float *rstd, T *grad_x,
                     float *grad_weight, float *grad_bias, void *workspace, cudaStream_t st) {
  complete(a, V);
  const long long pieces = (long long)a.B * a.entries;
  float2 *by_channel = static_cast<float2 *>(workspace), *by_group = by_channel + pieces * a.C, *means = by_group + pieces * a.G,
         *by_level = means + (long long)a.B * a.L * a.G;
  const unsigned grid = (unsigned)(a.B * a.tiles);
  auto stats = a.act == kNone ? group_grad_stats_kernel<T, V, false> : group_grad_stats_kernel<T, V, true>;
  auto apply = a.act == kNone ? group_grad_apply_kernel<T, V, false> : group_grad_apply_kernel<T, V, true>;
  DFA3D_TRY(launch(stats, grid, kThreads<V>, sizeof(float2) * kThreads<V> * V, false, st, grad_y, x, a, mean, rstd, by_channel,
                   by_group));
  const unsigned merges = merge_grid(a), channels = grad_weight ? (unsigned)(a.B * a.L * ((a.C + 31) / 32)) : 0;
  DFA3D_TRY(launch(group_grad_merge_kernel, merges + channels, kMergeThreads, 0, true, st, a, merges, by_group, by_channel, means,
                   by_level));
  const int sums = grad_weight ? (a.C * a.weight_rows + 31) / 32 : 0;
  return launch(apply, sums + (grad_x ? grid : 0), kThreads<V>, 0, true, st, grad_y, x, a, grad_x ? (int)grid : 0, mean, rstd, means, by_level, grad_x,
                grad_weight, grad_bias);
}

// Elements a thread reads at a time: as many as divide the channels and as every address is aligned for, up to four.
int vector_width(int C, size_t size, std::initializer_list<const void *> addresses) {
  int v = 4;
  while (v > 1) {
    bool ok = C % v == 0;
    for (const void *p : addresses) ok = ok && reinterpret_cast<uintptr_t>(p) % (v * size) == 0;
    if (ok) break;
    v /= 2;
  }
  return v;
}

GnArgs arguments(int B, int N, int C, int G, const int64_t *shapes, int shape_stride, const int64_t *start, int L, const float *weight,
                 const float *bias, int weight_rows, float eps, int act) {
  GnArgs a = {};
  a.shapes = shapes; a.start = start; a.shape_stride = shape_stride;
  a.B = B; a.N = N; a.C = C; a.G = G; a.L = L; a.act = act;
  a.weight_rows = weight_rows; a.weight = weight; a.bias = bias; a.eps = eps;
  return a;
}

}  // namespace

// For any word that a launch may read by.
long long group_norm_workspace(int B, int N, int C, int G, int L, bool backward) {
  if (B == 0 || N == 0 || (!backward && cluster_size(N, C))) return 0;
  long long pieces = 0;
  for (int V = 4; V >= 1; V /= 2)
    if (C % V == 0) {
      const int R = tile_rows(B, N, C, V);
      pieces = std::max<long long>(pieces, (long long)B * ((N + R - 1) / R + 2 * L + 1));
    }
  return (pieces * (backward ? C + G : G) + (long long)B * L * (backward ? C + G : G)) * (long long)sizeof(float2);
}

#define DFA3D_GN(fn, v, ...)                                            \
  if (dtype == 0) {                                                     \
    using T = float;                                                    \
    if (v == 4) return fn<T, 4>(__VA_ARGS__);                           \
    if (v == 2) return fn<T, 2>(__VA_ARGS__);                           \
    return fn<T, 1>(__VA_ARGS__);                                       \
  } else if (dtype == 1) {                                              \
    using T = __nv_bfloat16;                                            \
    if (v == 4) return fn<T, 4>(__VA_ARGS__);                           \
    if (v == 2) return fn<T, 2>(__VA_ARGS__);                           \
    return fn<T, 1>(__VA_ARGS__);                                       \
  } else {                                                              \
    using T = __half;                                                   \
    if (v == 4) return fn<T, 4>(__VA_ARGS__);                           \
    if (v == 2) return fn<T, 2>(__VA_ARGS__);                           \
    return fn<T, 1>(__VA_ARGS__);                                       \
  }

cudaError_t launch_group_norm_forward(const void *x, int dtype, int B, int N, int C, int G, const int64_t *shapes,
                                      int shape_stride, const int64_t *start, int L, const float *weight, const float *bias,
                                      int weight_rows, float eps, int act, void *y, float *mean, float *rstd, void *workspace,
                                      cudaStream_t s) {
  const GnArgs a = arguments(B, N, C, G, shapes, shape_stride, start, L, weight, bias, weight_rows, eps, act);
  const int v = vector_width(C, dtype == 0 ? 4 : 2, {x, y});
  DFA3D_GN(forward, v, (const T *)x, a, (T *)y, mean, rstd, workspace, s)
}

cudaError_t launch_group_norm_backward(const void *grad_y, const void *x, int dtype, int B, int N, int C, int G,
                                       const int64_t *shapes, int shape_stride, const int64_t *start, int L, const float *weight,
                                       const float *bias, int weight_rows, const float *mean, const float *rstd, int act,
                                       void *grad_x, float *grad_weight, float *grad_bias, void *workspace, cudaStream_t s) {
  const GnArgs a = arguments(B, N, C, G, shapes, shape_stride, start, L, weight, bias, weight_rows, 0.f, act);
  const int v = vector_width(C, dtype == 0 ? 4 : 2, {x, grad_y, grad_x ? grad_x : x});
  DFA3D_GN(backward, v, (const T *)grad_y, (const T *)x, a, mean, rstd, (T *)grad_x, grad_weight, grad_bias, workspace, s)
}

}  // namespace dfa3d
