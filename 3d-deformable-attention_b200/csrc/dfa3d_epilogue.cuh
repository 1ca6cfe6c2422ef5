// What the epilogues of the feed-forward products do with a row of sums in registers.
#pragma once
#include "dfa3d_act.cuh"
#include "dfa3d_lost.h"
#include "dfa3d_rowvec.cuh"
#include "dfa3d_tcgen05.cuh"

namespace dfa3d {

// The 16-byte piece `piece` of row `row` of a slab as tiled copies lay it out.
template <int ROW_BYTES> __device__ __forceinline__ uint32_t piece_of(uint32_t slab, int row, int piece) {
  const int mix = ROW_BYTES == 128 ? row & 7 : (row >> 1) & 3;
  return slab + row * ROW_BYTES + ((piece ^ mix) << 4);
}

// Row `row` of a slab that a wait was for which has run out.
template <int ROW_BYTES> __device__ __forceinline__ void lose_row(uint32_t slab, int row) {
  for (int piece = 0; piece < ROW_BYTES / 16; ++piece)
    tc::write16(slab + row * ROW_BYTES + piece * 16, make_uint4(kLost, kLost, kLost, kLost));
}

template <int ACT, int N> __device__ __forceinline__ void activate_each(float (&z)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const Two a = activate<ACT>(Two{z[i], z[i + 1]});
    z[i] = a.x;
    z[i + 1] = a.y;
  }
}
template <int N> __device__ __forceinline__ void activate_all(float (&z)[N], int act) {
  switch (act) {
    case DFA3D_ROW_RELU: return activate_each<DFA3D_ROW_RELU>(z);
    case DFA3D_ROW_SILU: return activate_each<DFA3D_ROW_SILU>(z);
    case DFA3D_ROW_GELU: return activate_each<DFA3D_ROW_GELU>(z);
    default: return;
  }
}
template <int ACT, int N> __device__ __forceinline__ void slope_each(float (&z)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    Two a, s;
    activate_both<ACT>(Two{z[i], z[i + 1]}, a, s);
    z[i] = s.x;
    z[i + 1] = s.y;
  }
}
template <int N> __device__ __forceinline__ void slope_all(float (&z)[N], int act) {
  switch (act) {
    case DFA3D_ROW_RELU: return slope_each<DFA3D_ROW_RELU>(z);
    case DFA3D_ROW_SILU: return slope_each<DFA3D_ROW_SILU>(z);
    case DFA3D_ROW_GELU: return slope_each<DFA3D_ROW_GELU>(z);
    default: return slope_each<DFA3D_ROW_NONE>(z);
  }
}
// gate, up, d -> d up act'(gate), d act(gate), act(gate) up
template <int ACT, int N> __device__ __forceinline__ void gate_each(float (&g)[N], float (&u)[N], float (&d)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const Two up{u[i], u[i + 1]}, through{d[i], d[i + 1]};
    Two a, s;
    activate_both<ACT>(Two{g[i], g[i + 1]}, a, s);
    const Two grad_gate = through * up * s, grad_up = through * a, h = a * up;
    g[i] = grad_gate.x;
    g[i + 1] = grad_gate.y;
    d[i] = grad_up.x;
    d[i + 1] = grad_up.y;
    u[i] = h.x;
    u[i + 1] = h.y;
  }
}
template <int N> __device__ __forceinline__ void gate_all(float (&g)[N], float (&u)[N], float (&d)[N], int act) {
  switch (act) {
    case DFA3D_ROW_RELU: return gate_each<DFA3D_ROW_RELU>(g, u, d);
    case DFA3D_ROW_SILU: return gate_each<DFA3D_ROW_SILU>(g, u, d);
    case DFA3D_ROW_GELU: return gate_each<DFA3D_ROW_GELU>(g, u, d);
    default: return gate_each<DFA3D_ROW_NONE>(g, u, d);
  }
}

template <int N> __device__ __forceinline__ void add_bias(float (&z)[N], uint32_t bias) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const float4 b = tc::read_four(bias + i * 4);
    const Two lo = Two{z[i], z[i + 1]} + Two{b.x, b.y}, hi = Two{z[i + 2], z[i + 3]} + Two{b.z, b.w};
    z[i] = lo.x; z[i + 1] = lo.y; z[i + 2] = hi.x; z[i + 3] = hi.y;
  }
}

// columns of this lane's row into a slab, from piece `first` on
template <typename O, int ROW_BYTES, int N> __device__ __forceinline__ void put(const float (&z)[N], uint32_t slab, int row, int first) {
  constexpr int V = 16 / (int)sizeof(O);
#pragma unroll
  for (int i = 0; i < N; i += V) {
    float f[V];
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = z[i + k];
    const uint4 w = narrow_word<O, V>(f);
    tc::write16(piece_of<ROW_BYTES>(slab, row, first + i / V), w);
  }
}
// z = z + slab, or z * slab
template <typename O, int ROW_BYTES, bool TIMES, int N>
__device__ __forceinline__ void combine(float (&z)[N], uint32_t slab, int row, int first) {
  constexpr int V = 16 / (int)sizeof(O);
#pragma unroll
  for (int i = 0; i < N; i += V) {
    const uint4 w = tc::read16(piece_of<ROW_BYTES>(slab, row, first + i / V));
    float f[V];
    widen_word<O, V>(w, f);
#pragma unroll
    for (int k = 0; k < V; ++k) z[i + k] = TIMES ? z[i + k] * f[k] : z[i + k] + f[k];
  }
}

}  // namespace dfa3d
