// How the rows of a feature pyramid are cut up for the group norm: which rows belong to which level, and which rows a CTA takes.
// Plain arithmetic, the same on the device and in the CPU tests.
//
// The N rows of an image are a sequence of 2L + 1 segments: before every level a gap (segment 2l, empty in an ordinary table),
// the level (2l + 1), and what is left behind the last one (2L).  A table that points outside of the N rows, overlaps or goes
// backwards is cut to what is left: segments are disjoint, ascending and cover [0, N) whatever the table says.
//
// The rows are also split into tiles of R consecutive rows.  A piece is what a tile and a segment share; going along the rows every
// new piece advances the tile or the segment, so tile + segment is different for every piece of an image.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define DFA3D_BOTH __host__ __device__ __forceinline__
#else
#define DFA3D_BOTH inline
#endif

namespace dfa3d {

constexpr int kMaxLevels = 32;
constexpr int kMaxSegments = 2 * kMaxLevels + 1;

struct SegmentTable {
  int end[kMaxSegments];      // first row behind segment i; segment i begins at end[i - 1]
  int count;
};

DFA3D_BOTH int segment_begin(const SegmentTable &t, int i) { return i == 0 ? 0 : t.end[i - 1]; }

// What a level's entry in the table says, cut to [0, N].  Level l is then [max(first, e), max(first, last, e)) where e is the end of
// the levels before it: the largest of their `last` (and `first`).
struct LevelSpan {
  int first, last;
};
DFA3D_BOTH LevelSpan level_span(int64_t h, int64_t w, int64_t start, int N) {
  const int64_t limit = (int64_t)N + 1;
  h = h < 0 ? 0 : h > limit ? limit : h;
  w = w < 0 ? 0 : w > limit ? limit : w;
  const int64_t rows = h * w, first = start < 0 ? 0 : start > N ? N : start;
  // a start before row 0 does not make the level shorter
  const int64_t last = start < 0 ? rows : start > N ? N : start + rows;
  return {(int)first, (int)(last > N ? N : last)};
}

// shapes (L, stride): height and width first; without a table (shapes null) the N rows are one level.
inline void make_segments(SegmentTable &t, const int64_t *shapes, int stride, const int64_t *start, int L, int N) {
  int end = 0;
  for (int l = 0; l < L; ++l) {
    const LevelSpan s = shapes ? level_span(shapes[(int64_t)l * stride], shapes[(int64_t)l * stride + 1], start[l], N)
                               : LevelSpan{0, N};
    t.end[2 * l] = s.first > end ? s.first : end;
    end = s.last > t.end[2 * l] ? s.last : t.end[2 * l];
    t.end[2 * l + 1] = end;
  }
  t.end[2 * L] = N;
  t.count = 2 * L + 1;
}

#ifdef __CUDACC__
// The same by one warp, lane l with level l (kMaxLevels = 32).
__device__ __forceinline__ void make_segments_warp(SegmentTable &t, const int64_t *shapes, int stride, const int64_t *start, int L,
                                                   int N) {
  const int l = threadIdx.x & 31;
  LevelSpan s = {0, shapes ? 0 : N};
  if (shapes && l < L) s = level_span(shapes[(int64_t)l * stride], shapes[(int64_t)l * stride + 1], start[l], N);
  int end = s.last > s.first ? s.last : s.first;      // the largest one up to this level
  if (l >= L) end = 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int e = __shfl_up_sync(0xffffffffu, end, o);
    if (l >= o && e > end) end = e;
  }
  int before = __shfl_up_sync(0xffffffffu, end, 1);
  if (l == 0) before = 0;
  if (l < L) {
    t.end[2 * l] = s.first > before ? s.first : before;
    t.end[2 * l + 1] = end;
  }
  if (l == 0) {
    t.end[2 * L] = N;
    t.count = 2 * L + 1;
  }
}
#endif

// Division of 0 <= n < 2^31 by a number that the host knows: (hi(n m) + n) >> s with m = 2^32 (2^s - d) / d + 1, s = ceil(log2 d)
// (Granlund and Montgomery, "Division by invariant integers using multiplication", PLDI 1994).
struct Divisor {
  uint32_t d, m;
  int s;
};
inline Divisor make_divisor(uint32_t d) {
  Divisor v = {d, 0, 0};
  while ((1ull << v.s) < d) ++v.s;
  v.m = (uint32_t)((((1ull << v.s) - d) << 32) / d + 1);
  return v;
}
DFA3D_BOTH int quotient(int n, const Divisor &v) {
#ifdef __CUDA_ARCH__
  const uint32_t hi = __umulhi((uint32_t)n, v.m);
#else
  const uint32_t hi = (uint32_t)(((uint64_t)(uint32_t)n * v.m) >> 32);
#endif
  return (int)((hi + (uint32_t)n) >> v.s);
}

}  // namespace dfa3d
