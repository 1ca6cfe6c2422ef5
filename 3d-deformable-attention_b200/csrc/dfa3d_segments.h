// How the rows of a feature pyramid are cut up for the group norm: which rows belong to which level, and which rows a CTA takes.
// Plain arithmetic, the same on the device and in the CPU tests.
//
// The N rows of an image are a sequence of 2L + 1 segments: before every level a gap (segment 2l, empty in an ordinary table),
// the level (2l + 1), and what is left behind the last one (2L).  A table that points outside of the N rows, overlaps or goes
// backwards is cut to what is left: segments are disjoint, ascending and cover [0, N) whatever the table says.
//
// The rows are also split into S runs of consecutive rows, one for a CTA.  A piece is what a run and a segment share; going along
// the rows every new piece advances the run or the segment, so run + segment is different for every piece of an image and below
// S + 2L + 1.
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

// shapes (L, stride): height and width first; without a table (shapes null) the N rows are one level.
DFA3D_BOTH void make_segments(SegmentTable &t, const int64_t *shapes, int stride, const int64_t *start, int L, int N) {
  int at = 0;
  for (int l = 0; l < L; ++l) {
    int64_t first = 0, rows = N;
    if (shapes) {
      const int64_t limit = (int64_t)N + 1;
      int64_t h = shapes[(int64_t)l * stride], w = shapes[(int64_t)l * stride + 1];
      h = h < 0 ? 0 : h > limit ? limit : h;
      w = w < 0 ? 0 : w > limit ? limit : w;
      first = start[l];
      rows = h * w;
    }
    const int64_t begin = first < at ? at : first > N ? N : first;
    // a start before `at` shortens the level by what others have
    int64_t last = first < 0 ? rows : first > N ? N : first + rows;
    last = last < begin ? begin : last > N ? N : last;
    t.end[2 * l] = (int)begin;
    t.end[2 * l + 1] = at = (int)last;
  }
  t.end[2 * L] = N;
  t.count = 2 * L + 1;
}

// Run s of S: rows [run_begin(s), run_begin(s + 1)).
DFA3D_BOTH int run_begin(int s, int S, int N) { return (int)((int64_t)N * s / S); }

// The run that row r (0 <= r < N) belongs to.
DFA3D_BOTH int run_of(int r, int S, int N) { return (int)((((int64_t)r + 1) * S - 1) / N); }

}  // namespace dfa3d
