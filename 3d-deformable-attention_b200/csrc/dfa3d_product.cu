// Matrix products of a feed-forward block with everything that follows them in their epilogue.
//
// Two CTAs on neighbouring SMs make a pair that walks over tiles of 256 rows; each holds 128 rows of A and half of B's columns, and the
// tensor cores of both read both halves: what bounds these products (a few hundred columns, summed over a few hundred) is the way
// from L2 into shared memory, and B crosses it half as often.  Where A's rows fit (256 summed elements: 64 KB) they stay for all tiles
// of their rows, and a pair's tiles are neighbours, so that A crosses it once.  In each CTA a warp asks for operand tiles of 64
// along the summed axis (tiled copies into rings), one thread of the pair issues the products, whose 32-bit sums stay in tensor
// memory, two to four tiles at a time, so that the next tile is summed while the other warps read the last one, apply bias,
// activation, residual or derivatives in 32 bits, round once and hand rows to tiled stores.
#include <type_traits>

#include "dfa3d_act.cuh"
#include "dfa3d_common.cuh"
#include "dfa3d_product.h"
#include "dfa3d_rowvec.cuh"
#include "dfa3d_tcgen05.cuh"
#include "dfa3d_tensor_map.h"

namespace dfa3d {
namespace {

constexpr int kRows = 128, kDepth = 64;          // of a CTA's tile; along the summed axis, 128 bytes
constexpr int kOperandA = kRows * kDepth * 2;

struct Maps {
  CUtensorMap a0, a1, b0, b1, b2, in, out[3];
};
struct Extents {
  int rows, n, steps0, steps1;      // steps of kDepth
  int tiles, tiles_n;
  int act, has_in, direct;          // direct: `in` and `out` do not lie as tiled copies need it
  const void *bias0, *bias1, *in;
  void *out;
  long long in_pitch, out_pitch;
};

// RESIDENT: A's rows stay for all tiles of their rows.
template <ProductKind KIND, typename I, typename O, int BN, bool RESIDENT> struct Tile {
  static constexpr bool gated = KIND == kGated || KIND == kGatedGrad;
  static constexpr int outs = KIND == kGatedGrad ? 3 : 1;
  static constexpr int columns = gated ? BN / 2 : BN;                            // of a result
  static constexpr int sums = KIND == kGatedGrad ? BN + BN / 2 : BN;             // accumulator columns
  static constexpr int depth = 512 / sums < 4 ? 512 / sums : 4;                  // accumulators
  static constexpr int memory = depth * sums <= 256 ? 256 : 512;
  // Epilogue warps: sixteen where a tile is summed quickly; eight, and more operands on their way, where it takes longer; eight
  // for the three results of kGatedGrad, which need 96 columns in registers and three slabs a warp.
  static constexpr int groups = KIND == kGatedGrad || !RESIDENT ? 2 : 4, warps = 4 * groups, threads = (4 + warps) * 32;
  static constexpr bool apart = sizeof(I) != sizeof(O);                          // `in` has a slab of its own
  static constexpr int chunk = KIND == kGatedGrad ? 32 : 128 / (int)sizeof(I);   // columns that a warp takes at a time
  static constexpr int chunks = columns / chunk;
  static constexpr int turns = chunks < groups ? groups / chunks : 1;            // a warp has a chunk of every so many tiles
  static constexpr int sub = 16;                                                // columns in registers, twice
  static constexpr int in_bytes = chunk * (int)sizeof(I), row_bytes = chunk * (int)sizeof(O);
  static constexpr int slab = 32 * row_bytes, slab_in = apart ? 32 * in_bytes : 0;
  static constexpr int slabs = warps * (outs * slab + slab_in);
  static constexpr int bias = warps * chunk * (gated ? 2 : 1) * 4;
  static constexpr int b_rows = BN / 2, b_bytes = b_rows * kDepth * 2;           // of each CTA
  static constexpr int b_ones = KIND == kInputGrad ? b_rows : BN / 4;            // columns of an mn-major B (kGatedGrad: the second)
  // About 2400 cycles pass from a product that frees a slot to the one that reads what was loaded into it, and a step of BN = 256 is
  // summed in 512: the rings have to hold that much.
  static constexpr int room = 227 * 1024 - 2048 - slabs - bias;
  static constexpr int both = room / (kOperandA + b_bytes) < 8 ? room / (kOperandA + b_bytes) : 8;
  static constexpr int slots_a = !RESIDENT ? both : KIND == kGatedGrad ? 8 : 4;
  static constexpr int most_b = (room - slots_a * kOperandA) / b_bytes;
  static constexpr int slots_b = most_b < 12 ? most_b : 12;
  static constexpr int barriers = 2 * slots_a + 2 * slots_b + 2 * depth + warps + 1;
  static constexpr int bytes = 1024 + slots_a * kOperandA + slots_b * b_bytes + slabs + bias + barriers * 8 + 16;
  // whoever reads an accumulator reads it every time, or it would take one phase of its barrier for another
  static_assert(depth % turns == 0 && (chunks <= groups ? groups % chunks : chunks % groups) == 0, "turns");
  static_assert(bytes <= 227 * 1024 && slots_b >= 4 && (row_bytes == 64 || row_bytes == 128) && chunks >= 1, "layout");
};

// The 16-byte piece `piece` of row `row` of a slab as tiled copies lay it out.
template <int ROW_BYTES> __device__ __forceinline__ uint32_t piece_of(uint32_t slab, int row, int piece) {
  const int mix = ROW_BYTES == 128 ? row & 7 : (row >> 1) & 3;
  return slab + row * ROW_BYTES + ((piece ^ mix) << 4);
}

template <int ACT, int N> __device__ __forceinline__ void activate_each(float (&z)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) z[i] = activate<ACT>(z[i]);
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
  for (int i = 0; i < N; ++i) {
    float a;
    activate_both<ACT>(z[i], a, z[i]);
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
  for (int i = 0; i < N; ++i) {
    float a, s;
    activate_both<ACT>(g[i], a, s);
    g[i] = d[i] * u[i] * s;
    d[i] = d[i] * a;
    u[i] = a * u[i];
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

// one instruction for two sums
__device__ __forceinline__ void add_two(float &a, float &b, float c, float d) {
  asm("{\n.reg .b64 x, y;\nmov.b64 x, {%0, %1};\nmov.b64 y, {%2, %3};\nadd.rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}"
      : "+f"(a), "+f"(b)
      : "f"(c), "f"(d));
}
template <int N> __device__ __forceinline__ void add_bias(float (&z)[N], uint32_t bias) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const float4 b = tc::read_four(bias + i * 4);
    add_two(z[i], z[i + 1], b.x, b.y);
    add_two(z[i + 2], z[i + 3], b.z, b.w);
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

// What a warp of a direct product does instead of tiled copies: rows between a slab and memory, element by element, neighbours by
// neighbouring lanes.
template <typename E, int ROW_BYTES, bool OUT, typename P>
__device__ __forceinline__ void copy_direct(P *memory, long long pitch, int rows, int columns, uint32_t slab, int lane) {
  constexpr int size = (int)sizeof(E);
  for (int r = 0; r < rows; ++r) {
    for (int c = lane; c < columns; c += 32) {
      const uint32_t at = piece_of<ROW_BYTES>(slab, r, c * size / 16) + c * size % 16;
      if constexpr (OUT) memory[r * pitch + c] = tc::read_one<E>(at);
      else tc::write_one<E>(at, memory[r * pitch + c]);
    }
  }
}

// A tile by its row and column among the tiles: divided once, then counted, since a division takes a warp a few hundred cycles.  Rows
// begin with different columns: if all pairs read the same weights at a time, they queue for the few places that hold them.
struct Place {
  int m, n, turn;
  __device__ __forceinline__ Place(int tile, int across) : m(tile / across), n(tile - tile / across * across), turn(m % across) {}
  __device__ __forceinline__ void on(int tiles, int across) {
    n += tiles;
    while (n >= across) {
      n -= across;
      ++m;
      if (++turn == across) turn = 0;
    }
  }
  __device__ __forceinline__ int column(int across) const { return n + turn < across ? n + turn : n + turn - across; }
};

template <ProductKind KIND, typename T, typename I, typename O, int BN, bool RESIDENT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Tile<KIND, I, O, BN, RESIDENT>::threads, 1)
    product_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Extents p) {
  using L = Tile<KIND, I, O, BN, RESIDENT>;
  extern __shared__ uint8_t raw[];
  const uint32_t base_a = (tc::shared_address(raw) + 1023) & ~1023u, base_b = base_a + L::slots_a * kOperandA;
  const uint32_t slabs = base_b + L::slots_b * L::b_bytes, bias_at = slabs + L::slabs;
  const uint32_t full_a = bias_at + L::bias, empty_a = full_a + L::slots_a * 8;
  const uint32_t full_b = empty_a + L::slots_a * 8, empty_b = full_b + L::slots_b * 8;
  const uint32_t summed = empty_b + L::slots_b * 8, drained = summed + L::depth * 8;
  const uint32_t in_there = drained + L::depth * 8, quiet = in_there + L::warps * 8, where = quiet + 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = tc::rank_in_pair();
  // neighbouring tiles, which share their rows, for each pair
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int first_tile = (int)((long long)p.tiles * pair / pairs), last_tile = (int)((long long)p.tiles * (pair + 1) / pairs);

  if (warp == 1) {
    for (int i = lane; i < L::barriers; i += 32) {      // all of them lie side by side; only the drained ones have many arrivals
      const int from = (int)(drained - full_a) / 8;
      tc::barrier_init(full_a + i * 8, i >= from && i < from + L::depth ? 2 * 4 * L::chunks : 1);
    }
    tc::barriers_visible();
  }
  if (warp == 2) tc::tensor_memory_take<L::memory, true>(where);
  const Place first(first_tile, p.tiles_n);
  if (warp == 0) {      // the first rows and columns come from far away: they are asked for while the CTAs find together
    const int m0 = (first.m * 2 + (int)rank) * kRows;
    if (lane < p.steps0 && lane < 8) tc::tile_to_l2(&maps.a0, lane * kDepth, m0);
    else if (lane < p.steps0 + p.steps1 && lane < 8) tc::tile_to_l2(&maps.a1, (lane - p.steps0) * kDepth, m0);
  }
  tc::order_before();
  __syncwarp();
  tc::pair_sync();
  tc::order_after();
  uint32_t memory;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(memory) : "r"(where));

  const int steps = p.steps0 + p.steps1, slots_a = RESIDENT ? steps : L::slots_a;
  if (warp == 0 || warp == 3) {
    // ---- operand tiles: this CTA's, into its shared memory; the first CTA's barriers count those of both.  One warp for each
    // operand: a step of a narrow tile is summed as fast as one thread asks for its operands. ----
    if (tc::one_lane()) {
      const bool is_a = warp == 3;
      const uint32_t ring = is_a ? base_a : base_b, full = is_a ? full_a : full_b, empty = is_a ? empty_a : empty_b;
      const uint32_t first_full = tc::address_in(full, 0), bytes = is_a ? kOperandA : L::b_bytes;
      const int slots = is_a ? slots_a : L::slots_b;
      int slot = 0, asked = 0;      // asked: no more than it takes to go round once
      uint32_t phase = 0;
      bool ok = true;
      auto take = [&] {             // the next slot, once it is free
        ok = tc::wait(empty + slot * 8, phase ^ 1);
        if (ok && rank == 0) tc::arrive_expect(full + slot * 8, 2 * bytes);
        return ok;
      };
      auto next = [&] {
        if (asked < slots) ++asked;
        if (++slot == slots) {
          slot = 0;
          phase ^= 1;
        }
      };
      Place at_tile = first;
      for (int tile = first_tile; tile < last_tile && ok; ++tile, at_tile.on(1, p.tiles_n)) {
        const int m0 = (at_tile.m * 2 + (int)rank) * kRows, n0 = at_tile.column(p.tiles_n) * L::columns;
        if (is_a) {
          const bool fresh = tile == first_tile || at_tile.n == 0, look = fresh && tile + p.tiles_n - at_tile.n < last_tile;
          if (RESIDENT && !fresh) continue;
          for (int k = 0; k < steps; ++k, next()) {
            const bool second = k >= p.steps0;
            const CUtensorMap *map = second ? &maps.a1 : &maps.a0;
            const int at = (second ? k - p.steps0 : k) * kDepth;
            if (!take()) break;
            tc::tile_load_pair(ring + slot * kOperandA, map, at, m0, first_full + slot * 8);
            if (look) tc::tile_to_l2(map, at, m0 + 2 * kRows);
          }
        } else if constexpr (KIND == kInputGrad) {
          constexpr int box = L::b_rows < 64 ? L::b_rows : 64;
          for (int k = 0; k < steps; ++k, next()) {
            const bool second = k >= p.steps0;
            const CUtensorMap *map = second ? &maps.b1 : &maps.b0;
            const int at = (second ? k - p.steps0 : k) * kDepth;
            if (!take()) break;
#pragma unroll
            for (int i = 0; i < L::b_rows / box; ++i)
              tc::tile_load_pair(ring + slot * L::b_bytes + i * kDepth * 128, map, n0 + (int)rank * L::b_rows + i * box, at,
                                 first_full + slot * 8);
          }
        } else {
          const CUtensorMap *map = L::gated && rank ? &maps.b1 : &maps.b0;
          const int y = L::gated ? n0 : n0 + (int)rank * L::b_rows;
          for (int k = 0; k < p.steps0; ++k, next()) {
            if (!take()) break;
            tc::tile_load_pair(ring + slot * L::b_bytes, map, k * kDepth, y, first_full + slot * 8);
          }
          if constexpr (KIND == kGatedGrad) {      // half as wide: two steps fill a slot
            for (int k = 0; k < p.steps1 && ok; k += 2, next()) {
              if (!take()) break;
              tc::tile_load_pair(ring + slot * L::b_bytes, &maps.b2, n0 + (int)rank * L::b_ones, k * kDepth, first_full + slot * 8);
              tc::tile_load_pair(ring + slot * L::b_bytes + L::b_bytes / 2, &maps.b2, n0 + (int)rank * L::b_ones, (k + 1) * kDepth,
                                 first_full + slot * 8);
            }
          }
        }
      }
      // nothing may be on its way into shared memory when the CTAs end
      if (rank == 0) {
        for (int i = 0; i < asked; ++i) {
          if (--slot < 0) {
            slot = slots - 1;
            phase ^= 1;
          }
          tc::wait(full + slot * 8, phase);
        }
      }
      if (!ok) __nanosleep(1000000);
    }
  } else if (warp == 1) {
    // ---- products of both CTAs ----
    // The whole warp walks, so that addresses and descriptors stay uniform; one lane issues.
    if (rank == 0) {
      constexpr uint32_t shape = tc::product_shape<T>(2 * kRows, BN, false, KIND == kInputGrad);
      constexpr uint32_t shape_d = tc::product_shape<T>(2 * kRows, BN / 2, false, true);
      int sa = 0, sb = 0, slot = 0;
      uint32_t phase_a = 0, phase_b = 0, round = 0;
      bool ok = true;
      Place at_tile = first;
      for (int tile = first_tile; tile < last_tile && ok; ++tile, at_tile.on(1, p.tiles_n)) {
        const uint32_t acc = memory + slot * L::sums;
        const bool fresh = tile == first_tile || at_tile.n == 0, last = tile + 1 == last_tile || at_tile.n + 1 == p.tiles_n;
        if (!(ok = tc::wait_warp(drained + slot * 8, round ^ 1))) break;
        tc::order_after();
        // Steps of one of the two sums of a tile; everything that can be known before is, since a step of a narrow tile is issued
        // no faster than it is summed.
        auto sum = [&](auto second, int from, int to, uint32_t d) {
          constexpr bool SECOND = decltype(second)::value;      // kGatedGrad: grad_y Wd
          constexpr uint32_t form = SECOND ? shape_d : shape;
          for (int k = from; k < to; ++k) {
            const int use = RESIDENT ? k : sa;
            if (fresh || !RESIDENT) {
              if (!(ok = tc::wait_warp(full_a + use * 8, phase_a))) return;
              if (++sa == slots_a) {
                sa = 0;
                phase_a ^= 1;
              }
            }
            const bool odd = SECOND && (k - from) % 2 != 0;      // the second half of a slot
            if (!odd && !(ok = tc::wait_warp(full_b + sb * 8, phase_b))) return;
            tc::order_after();
            const uint64_t a = tc::k_major(base_a + use * kOperandA);
            const uint32_t at_b = base_b + sb * L::b_bytes + (odd ? L::b_bytes / 2 : 0);
            constexpr bool mn = SECOND || KIND == kInputGrad, narrow_b = mn && L::b_ones < 64;
            const uint64_t b = narrow_b ? tc::mn_major_narrow(at_b) : mn ? tc::mn_major(at_b, kDepth * 128) : tc::k_major(at_b);
            constexpr int step_b = (narrow_b ? 1024 : mn ? 2048 : 32) / 16;
            const bool give_b = !SECOND || odd || k + 1 == to;
            if (tc::one_lane()) {
              tc::product<true>(d, a, b, form, k > from);
#pragma unroll
              for (int j = 1; j < kDepth / 16; ++j) tc::product<true>(d, a + j * 2, b + j * step_b, form, true);
              if (last || !RESIDENT) tc::products_arrive<true>(empty_a + use * 8);
              if (give_b) tc::products_arrive<true>(empty_b + sb * 8);
            }
            __syncwarp();
            if (give_b && ++sb == L::slots_b) {
              sb = 0;
              phase_b ^= 1;
            }
          }
        };
        if constexpr (KIND == kGatedGrad) {
          sum(std::false_type(), 0, p.steps0, acc);
          if (ok) sum(std::true_type(), p.steps0, steps, acc + BN);
        } else {
          sum(std::false_type(), 0, steps, acc);
        }
        if (ok && tc::one_lane()) tc::products_arrive<true>(summed + slot * 8);
        __syncwarp();
        if (++slot == L::depth) {
          slot = 0;
          round ^= 1;
        }
      }
      if (tc::one_lane()) tc::products_arrive<true>(quiet);
      __syncwarp();
    }
    tc::wait_warp(quiet, 0);
  } else if (warp >= 4) {
    // ---- epilogue: a warp has 32 rows; the groups of four warps take a tile's chunks of columns in turn ----
    const int e = warp - 4, quarter = warp & 3, group = e >> 2;
    const uint32_t slab_in = slabs + e * (L::outs * L::slab + L::slab_in), slab = slab_in + L::slab_in;
    const uint32_t bias = bias_at + e * (L::bias / L::warps), there = in_there + e * 8, first_drained = tc::address_in(drained, 0);
    const bool loads = p.has_in && !p.direct;
    const T *bias0 = static_cast<const T *>(p.bias0), *bias1 = static_cast<const T *>(p.bias1);
    uint32_t in_phase = 0;
    bool ok = true;

    // Chunk number c of this pair: tile first_tile + c / chunks; this warp has c = group, group + groups, ...
    const int all = (last_tile - first_tile) * L::chunks;
    struct Chunk {
      int c, row, column;
      Place place;
    };
    auto locate = [&](Chunk &h) {
      h.row = (h.place.m * 2 + (int)rank) * kRows + quarter * 32;
      h.column = h.place.column(p.tiles_n) * L::columns + h.c % L::chunks * L::chunk;
    };
    auto go_on = [&](Chunk &h) {
      h.place.on((h.c + L::groups) / L::chunks - h.c / L::chunks, p.tiles_n);
      h.c += L::groups;
      locate(h);
    };
    auto inside = [&](const Chunk &h) { return h.row < p.rows && h.column < p.n; };
    Chunk now{group, 0, 0, first};
    now.place.on(group / L::chunks, p.tiles_n);
    locate(now);
    Chunk then = now;            // of what is added to a chunk or multiplied by it, the one to ask for next
    auto ask = [&] {
      while (then.c < all && !inside(then)) go_on(then);
      if (then.c >= all) return;
      tc::arrive_expect(there, 32 * L::in_bytes);
      tc::tile_load(slab_in, &maps.in, then.column, then.row, there);
      go_on(then);
      if (then.c < all) tc::tile_to_l2(&maps.in, then.column, then.row);
    };
    if (loads && lane == 0) ask();
    // biases of the next chunk are on their way while this one is worked on
    constexpr int ahead = L::chunk / 32;
    float next0[ahead], next1[ahead];
    auto ask_bias = [&](int c, int col) {
#pragma unroll
      for (int i = 0; i < ahead; ++i) {
        const bool in = c < all && col + i * 32 + lane < p.n;
        next0[i] = in && bias0 ? wide(bias0[col + i * 32 + lane]) : 0.f;
        if constexpr (L::gated) next1[i] = in && bias1 ? wide(bias1[col + i * 32 + lane]) : 0.f;
      }
    };
    if constexpr (KIND != kInputGrad) ask_bias(now.c, now.column);

    while (now.c < all) {
      const int it = now.c / L::chunks, slot = it % L::depth, m0 = now.row, col = now.column;
      const uint32_t acc = memory + ((uint32_t)quarter << 21) + slot * L::sums + now.c % L::chunks * L::chunk;
      const bool some = inside(now);
      const int rows_in = min(32, p.rows - m0), cols_in = min(L::chunk, p.n - col);
      if constexpr (KIND != kInputGrad) {
#pragma unroll
        for (int i = 0; i < ahead; ++i) {
          tc::write_one<float>(bias + (i * 32 + lane) * 4, next0[i]);
          if constexpr (L::gated) tc::write_one<float>(bias + (L::chunk + i * 32 + lane) * 4, next1[i]);
        }
        go_on(now);
        ask_bias(now.c, now.column);
      } else {
        go_on(now);
      }
      __syncwarp();
      if (some) {
        if (p.direct && p.has_in) {
          __syncwarp();
          copy_direct<I, L::in_bytes, false>(static_cast<const I *>(p.in) + m0 * p.in_pitch + col, p.in_pitch, rows_in, cols_in, slab_in,
                                             lane);
        } else if ((!loads || L::apart) && lane == 0) {
          tc::stores_read<0>();
        }
        __syncwarp();
      }
      if (ok) ok = __all_sync(0xffffffffu, tc::wait(summed + slot * 8, (uint32_t)(it / L::depth) & 1));
      tc::order_after();
      if (some) {
        if (loads) {
          if (ok) ok = __all_sync(0xffffffffu, tc::wait(there, in_phase));
          in_phase ^= 1;
        }
        // columns of the accumulators, the next ones on their way while these are worked on
        constexpr int sums = KIND == kGatedGrad ? 3 : L::gated ? 2 : 1, turns = L::chunk / L::sub;
        float v[2][sums][L::sub];
        auto fetch = [&](int t) {
#pragma unroll
          for (int i = 0; i < sums; ++i) tc::tensor_load(v[t & 1][i], acc + i * (BN / 2) + t * L::sub);
        };
        fetch(0);
#pragma unroll
        for (int t = 0; t < turns; ++t) {
          const int off = t * L::sub, first = off * (int)sizeof(O) / 16;
          float(&z)[L::sub] = v[t & 1][0];
#pragma unroll
          for (int i = 0; i < sums; ++i) tc::tensor_loads_done(v[t & 1][i]);
          if (t + 1 < turns) fetch(t + 1);
          if constexpr (KIND != kInputGrad) add_bias(z, bias + off * 4);
          if constexpr (L::gated) add_bias(v[t & 1][1], bias + (L::chunk + off) * 4);
          if constexpr (KIND == kGatedGrad) {
            float(&u)[L::sub] = v[t & 1][1], (&d)[L::sub] = v[t & 1][2];
            gate_all(z, u, d, p.act);
            if (!ok) z[0] = u[0] = d[0] = __int_as_float(0x7fffffff);
            put<O, L::row_bytes>(d, slab + L::slab, lane, first);
            put<O, L::row_bytes>(u, slab + 2 * L::slab, lane, first);
          } else if constexpr (KIND == kGated) {
            activate_all(z, p.act);
#pragma unroll
            for (int i = 0; i < L::sub; ++i) z[i] *= v[t & 1][1][i];
          } else {
            if constexpr (KIND == kLinear) activate_all(z, p.act);
            if constexpr (KIND == kSlope) slope_all(z, p.act);
            if (p.has_in) combine<I, L::in_bytes, KIND == kSlope>(z, slab_in, lane, off * (int)sizeof(I) / 16);
          }
          if (!ok) z[0] = __int_as_float(0x7fffffff);
          put<O, L::row_bytes>(z, slab, lane, first);
        }
      }
      tc::order_before();
      if (!p.direct) tc::shared_to_async();
      __syncwarp();
      if (lane == 0) tc::arrive_in(first_drained + slot * 8);
      if (!some) continue;
      if (p.direct) {
        copy_direct<O, L::row_bytes, true>(static_cast<O *>(p.out) + m0 * p.out_pitch + col, p.out_pitch, rows_in, cols_in, slab, lane);
      } else if (lane == 0) {
#pragma unroll
        for (int o = 0; o < L::outs; ++o) tc::tile_store(&maps.out[o], col, m0, slab + o * L::slab);
        tc::stores_asked();
        if (loads) {
          if (!L::apart) tc::stores_read<0>();
          if (ok) ask();
        }
      }
    }
    if (lane == 0) tc::stores_done();
  }
  tc::order_before();
  __syncwarp();
  tc::pair_sync();      // the other CTA's products read this one's shared memory, its warps arrive at this one's barriers
  if (warp == 2) {
    tc::order_after();
    tc::tensor_memory_give<L::memory, true>(memory);
  }
}

template <ProductKind KIND, typename T, typename I, typename O, int BN, bool RESIDENT>
cudaError_t launch_as(const ProductArgs &a, cudaStream_t s) {
  using L = Tile<KIND, I, O, BN, RESIDENT>;
  auto code = [&](size_t size) { return size == 4 ? DFA3D_DTYPE_F32 : a.dtype; };
  auto fits = [](const void *q, long long pitch, size_t size) {
    return (reinterpret_cast<uintptr_t>(q) & 15u) == 0 && pitch * size % 16 == 0;
  };
  Maps m{};
  Extents p{};
  p.direct = !fits(a.out[0], a.out_pitch, sizeof(O)) || (a.in.data && !fits(a.in.data, a.in.pitch, sizeof(I)));
  if (p.direct && KIND != kLinear && KIND != kInputGrad) return cudaErrorInvalidValue;      // their results are workspaces
  constexpr int b_box = KIND == kInputGrad ? (L::b_rows < 64 ? L::b_rows : 64) : L::b_rows;
  bool ok = describe_matrix(m.a0, a.dtype, a.a0.data, a.rows, a.k0, a.a0.pitch, kDepth, kRows);
  if (a.k1 > 0) ok = ok && describe_matrix(m.a1, a.dtype, a.a1.data, a.rows, a.k1, a.a1.pitch, kDepth, kRows);
  if constexpr (KIND == kInputGrad) {
    ok = ok && describe_matrix(m.b0, a.dtype, a.b0.data, a.k0, a.n, a.b0.pitch, b_box, kDepth);
    if (a.k1 > 0) ok = ok && describe_matrix(m.b1, a.dtype, a.b1.data, a.k1, a.n, a.b1.pitch, b_box, kDepth);
  } else {
    ok = ok && describe_matrix(m.b0, a.dtype, a.b0.data, a.n, a.k0, a.b0.pitch, kDepth, b_box);
    if constexpr (L::gated) ok = ok && describe_matrix(m.b1, a.dtype, a.b1.data, a.n, a.k0, a.b1.pitch, kDepth, b_box);
    if constexpr (KIND == kGatedGrad) ok = ok && describe_matrix(m.b2, a.dtype, a.b2.data, a.k1, a.n, a.b2.pitch, L::b_ones, kDepth);
  }
  if (!p.direct) {
    if (a.in.data) ok = ok && describe_matrix(m.in, code(sizeof(I)), a.in.data, a.rows, a.n, a.in.pitch, L::chunk, 32);
    for (int o = 0; o < L::outs; ++o)
      ok = ok && describe_matrix(m.out[o], code(sizeof(O)), a.out[o], a.rows, a.n, a.out_pitch, L::chunk, 32);
  }
  if (!ok) return cudaErrorInvalidValue;
  p.rows = (int)a.rows;
  p.n = a.n;
  p.steps0 = (a.k0 + kDepth - 1) / kDepth;
  p.steps1 = (a.k1 + kDepth - 1) / kDepth;
  p.tiles_n = (a.n + L::columns - 1) / L::columns;
  p.tiles = (int)((a.rows + 2 * kRows - 1) / (2 * kRows)) * p.tiles_n;
  p.act = a.act;
  p.has_in = a.in.data != nullptr;
  p.bias0 = a.bias0;
  p.bias1 = a.bias1;
  p.in = a.in.data;
  p.in_pitch = a.in.pitch;
  p.out = a.out[0];
  p.out_pitch = a.out_pitch;
  constexpr auto kernel = &product_kernel<KIND, T, I, O, BN, RESIDENT>;
  cudaError_t rc = allow_shared<kernel>(L::bytes);
  if (rc != cudaSuccess) return rc;
  const int pairs = sm_count() / 2, grid = 2 * (p.tiles < pairs ? p.tiles : pairs);
  kernel<<<grid, L::threads, L::bytes, s>>>(m, p);
  return cudaGetLastError();
}

template <ProductKind KIND, typename T, typename I, typename O, int BN> cudaError_t launch_tiles(const ProductArgs &a, cudaStream_t s) {
  const int steps = (a.k0 + kDepth - 1) / kDepth + (a.k1 + kDepth - 1) / kDepth;
  return steps <= Tile<KIND, I, O, BN, true>::slots_a ? launch_as<KIND, T, I, O, BN, true>(a, s)
                                                      : launch_as<KIND, T, I, O, BN, false>(a, s);
}

// The width of tile whose slowest pair has the least to do: a tile costs its columns and, for operands and epilogue, about as much as
// 32 more.  Wide tiles read A fewer times, narrow ones spread a small or an unevenly divided product over more SMs.
int tile_width(long long rows, int n, int widest) {
  const long long pairs = sm_count() / 2, rows_of = (rows + 2 * kRows - 1) / (2 * kRows);
  int best = 64;
  long long least = -1;
  for (int w = 64; w <= widest; w *= 2) {
    const long long tiles = rows_of * ((n + w - 1) / w), cost = (tiles + pairs - 1) / pairs * (w + 32);
    if (least < 0 || cost <= least) {
      least = cost;
      best = w;
    }
  }
  return best;
}

template <typename T> cudaError_t launch_typed(const ProductArgs &a, cudaStream_t s) {
  switch (a.kind) {
    case kLinear: {
      const int w = tile_width(a.rows, a.n, 256);
      if (a.wide)
        return w == 256   ? launch_tiles<kLinear, T, float, float, 256>(a, s)
               : w == 128 ? launch_tiles<kLinear, T, float, float, 128>(a, s)
                          : launch_tiles<kLinear, T, float, float, 64>(a, s);
      return w == 256   ? launch_tiles<kLinear, T, T, T, 256>(a, s)
             : w == 128 ? launch_tiles<kLinear, T, T, T, 128>(a, s)
                        : launch_tiles<kLinear, T, T, T, 64>(a, s);
    }
    case kSlope: {
      const bool narrow = tile_width(a.rows, a.n, 128) == 64;
      if (a.wide) return narrow ? launch_tiles<kSlope, T, float, T, 64>(a, s) : launch_tiles<kSlope, T, float, T, 128>(a, s);
      return narrow ? launch_tiles<kSlope, T, T, T, 64>(a, s) : launch_tiles<kSlope, T, T, T, 128>(a, s);
    }
    case kGated:
      return tile_width(a.rows, a.n, 128) == 128 ? launch_tiles<kGated, T, T, T, 256>(a, s) : launch_tiles<kGated, T, T, T, 128>(a, s);
    case kGatedGrad: return launch_tiles<kGatedGrad, T, T, T, 128>(a, s);
    case kInputGrad: {
      const int w = tile_width(a.rows, a.n, 256);
      return w == 256   ? launch_tiles<kInputGrad, T, T, T, 256>(a, s)
             : w == 128 ? launch_tiles<kInputGrad, T, T, T, 128>(a, s)
                        : launch_tiles<kInputGrad, T, T, T, 64>(a, s);
    }
  }
  return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_product(const ProductArgs &a, cudaStream_t s) {
  if (const cudaError_t rc = bind_context()) return rc;
  return a.dtype == DFA3D_DTYPE_F16 ? launch_typed<__half>(a, s) : launch_typed<__nv_bfloat16>(a, s);
}

}  // namespace dfa3d
