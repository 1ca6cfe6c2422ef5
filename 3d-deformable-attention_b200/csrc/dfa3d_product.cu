// Matrix products of a feed-forward block with everything that follows them in their epilogue.
//
// Two CTAs on neighbouring SMs make a pair that walks over tiles of 256 rows; each holds 128 rows of A and half of B's columns, and the
// tensor cores of both read both halves: what bounds these products (a few hundred columns, summed over a few hundred) is the way
// from L2 into shared memory, and B crosses it half as often.  Where A's rows fit (256 summed elements: 64 KB) they stay for all tiles
// of their rows, and a pair's tiles are neighbours, so that A crosses it once.  In each CTA a warp asks for operand tiles of 64
// along the summed axis (tiled copies into rings), one thread of the pair issues the products, whose 32-bit sums stay in tensor
// memory, two to four tiles at a time, so that the next tile is summed while the other warps read the last one, apply bias,
// activation, residual or derivatives in 32 bits, round once and hand rows to tiled stores.
//
// Measured on calls that follow one another, bf16, 40 000 rows between 256 and 512 columns (10.5 GFLOP a product, 7 us at 1.6 PFLOP/s;
// 61 MB, 9.4 us at 6.5 TB/s):
//   256 -> 512: 15.8 us; with SiLU 20.2, with GELU 25.4; GELU's derivative times a gradient 32.3.   512 -> 256: 14.8; with a residual
//   of 16 bits 17.5, of 32 bits 28.   Input gradients: 14.8, of two products at once 30.2.   Gated hidden rows with SiLU 24.5, with GELU
//   28.5; their three backward results, 123 MB, 45.7 and 48.3.
// An activation's instructions (GELU 19.6 cycles of a scheduler for a warp's 32 elements, SiLU 13.4: 11 and 7.5 us of these calls) come
// almost whole on top of the rest: where a tile has as many chunks as there are takers, all epilogue warps read the same sums, compute
// and store at the same time, and issue on 37 to 42 of 100 cycles.  Without one neither HBM (results of this size stay in L2, 0 to 2 MB
// are written out while a kernel runs) nor the tensor cores (15 to 30 % of the cycles) are near their rates; what is left is the way from L2 into
// shared memory, uneven last rounds of tiles and about 4 us of setting up and ending.
//
// Gradients are rounded to 16 bits behind an activation's derivative, once: they are operands of the next products, and the bias
// gradient is the sum of what those read.
#include <type_traits>

#include "dfa3d_common.cuh"
#include "dfa3d_epilogue.cuh"
#include "dfa3d_product.h"
#include "dfa3d_tensor_map.h"

namespace dfa3d {
namespace {

constexpr int kRows = 128, kDepth = 64;          // of a CTA's tile; along the summed axis, 128 bytes
constexpr int kOperandA = kRows * kDepth * 2;
constexpr int kAhead = 10;                        // steps between asking for operands into L2 and into shared memory

struct Maps {
  CUtensorMap a0, a1, b0, b1, b2, in, out[3];
};
struct Extents {
  int rows, n, steps0, steps1;      // steps of kDepth
  int tiles, tiles_n;
  int act, has_in;
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
  // Epilogue warps: sixteen where a tile is summed quickly; eight, and more operands on their way, where it takes longer.  Two mates
  // share the chunk of three results of kGatedGrad, whose slabs leave no room for sixteen.
  static constexpr int groups = KIND == kGatedGrad || RESIDENT ? 4 : 2, warps = 4 * groups, threads = (4 + warps) * 32;
  static constexpr int mates = KIND == kGatedGrad ? 2 : 1, takers = groups / mates;
  static constexpr bool apart = sizeof(I) != sizeof(O);                          // `in` has a slab of its own
  static constexpr int chunk = KIND == kGatedGrad ? 32 : 128 / (int)sizeof(I);   // columns that a warp takes at a time
  static constexpr int chunks = columns / chunk;
  static constexpr int part = chunk / mates;                                     // of a chunk, columns of a warp
  static constexpr int turns = chunks < takers ? takers / chunks : 1;            // a warp has a chunk of every so many tiles
  static constexpr int sub = 16;                                                // columns in registers, twice
  static constexpr int in_bytes = chunk * (int)sizeof(I), row_bytes = chunk * (int)sizeof(O);
  static constexpr int slab = 32 * row_bytes, slab_in = apart ? 32 * in_bytes : 0;
  static constexpr int slabs = warps / mates * (outs * slab + slab_in);
  static constexpr int bias = warps * part * (gated ? 2 : 1) * 4;
  static constexpr int b_rows = BN / 2, b_bytes = b_rows * kDepth * 2;           // of each CTA
  static constexpr int b_ones = KIND == kInputGrad ? b_rows : BN / 4;            // columns of an mn-major B (kGatedGrad: the second)
  // Steps whose operands share a slot of the ring: waiting for a slot, giving it back and asking for the next cost the one thread that
  // does each about 400 cycles, and a step of BN = 256 is summed in 512, of 128 in 256.  Without RESIDENT a slot holds A's too.
  static constexpr int per = BN == 256 ? 1 : RESIDENT && BN == 64 ? 4 : 2;
  static constexpr int per_second = RESIDENT ? 2 * per : per;                    // of the second sum of kGatedGrad, half as wide
  static constexpr int in_slot_b = per * b_bytes, slot = in_slot_b + (RESIDENT ? 0 : per * kOperandA);
  static constexpr int slots_a = !RESIDENT ? 0 : KIND == kGatedGrad ? 8 : 4;
  static constexpr int room = 227 * 1024 - 512 - slots_a * kOperandA - slabs - bias;
  static constexpr int slots = room / slot < 8 ? room / slot : 8;
  static constexpr int barriers = 2 * slots_a + 2 * slots + 2 * depth + warps + 1;
  static constexpr int bytes = slots_a * kOperandA + slots * slot + slabs + bias + barriers * 8 + 16;
  // whoever reads an accumulator reads it every time, or it would take one phase of its barrier for another
  static_assert(depth % turns == 0 && (chunks <= takers ? takers % chunks : chunks % takers) == 0 && part % sub == 0, "turns");
  static_assert(one_an_sm(bytes) && bytes <= 227 * 1024 && slots >= 3 && (row_bytes == 64 || row_bytes == 128) && chunks >= 1, "layout");
};

// What a warp of a direct product does instead of tiled copies: rows between a slab and memory, neighbours by neighbouring lanes, a
// batch of rows at a time so that their loads are on their way together.
template <typename E, int SIZE, int ROW_BYTES, bool OUT, typename P>
__device__ __forceinline__ void copy_direct(P *memory, long long pitch, int rows, int columns, uint32_t slab, int lane) {
  constexpr int batch = 8;
  for (int c = lane; c < columns; c += 32) {
    const int piece = c * SIZE / 16, rest = c * SIZE % 16;
    for (int r = 0; r < rows; r += batch) {
      E v[batch];
#pragma unroll
      for (int i = 0; i < batch; ++i) {
        if (r + i >= rows) continue;
        if constexpr (OUT) v[i] = tc::read_one<E>(piece_of<ROW_BYTES>(slab, r + i, piece) + rest);
        else v[i] = memory[(r + i) * pitch + c];
      }
#pragma unroll
      for (int i = 0; i < batch; ++i) {
        if (r + i >= rows) continue;
        if constexpr (OUT) memory[(r + i) * pitch + c] = v[i];
        else tc::write_one<E>(piece_of<ROW_BYTES>(slab, r + i, piece) + rest, v[i]);
      }
    }
  }
}
// 16-bit rows that lie on the 4-byte grid go two elements at a time.
template <typename E, int ROW_BYTES, bool OUT, typename P>
__device__ __forceinline__ void copy_rows_direct(P *memory, long long pitch, int rows, int columns, uint32_t slab, int lane) {
  if constexpr (sizeof(E) == 2) {
    if (((reinterpret_cast<uintptr_t>(memory) | (uintptr_t)(pitch * 2)) & 3) == 0) {
      using Word = std::conditional_t<OUT, float, const float>;      // two elements; nothing is computed with it
      copy_direct<float, 4, ROW_BYTES, OUT>(reinterpret_cast<Word *>(memory), pitch / 2, rows, columns / 2, slab, lane);
      if (columns % 2 == 0) return;
      const int c = columns - 1;
      if (lane < rows) {
        const uint32_t at = piece_of<ROW_BYTES>(slab, lane, c * 2 / 16) + c * 2 % 16;
        if constexpr (OUT) memory[lane * pitch + c] = tc::read_one<E>(at);
        else tc::write_one<E>(at, memory[lane * pitch + c]);
      }
      return;
    }
  }
  copy_direct<E, (int)sizeof(E), ROW_BYTES, OUT>(memory, pitch, rows, columns, slab, lane);
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

// DIRECT: `in` and `out` do not lie as tiled copies need it.  A kernel of its own: that code's registers cost the others a third.
template <ProductKind KIND, typename T, typename I, typename O, int BN, bool RESIDENT, bool DIRECT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Tile<KIND, I, O, BN, RESIDENT>::threads, 1)
    product_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Extents p) {
  using L = Tile<KIND, I, O, BN, RESIDENT>;
  extern __shared__ __align__(1024) uint8_t raw[];      // operand tiles and slabs begin on its grid
  const uint32_t base_a = tc::shared_address(raw), ring = base_a + L::slots_a * kOperandA;
  const uint32_t slabs = ring + L::slots * L::slot, bias_at = slabs + L::slabs;
  const uint32_t full_a = bias_at + L::bias, empty_a = full_a + L::slots_a * 8;
  const uint32_t full = empty_a + L::slots_a * 8, empty = full + L::slots * 8;
  const uint32_t summed = empty + L::slots * 8, drained = summed + L::depth * 8;
  const uint32_t in_there = drained + L::depth * 8, quiet = in_there + L::warps * 8, where = quiet + 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = tc::rank_in_pair();
  // neighbouring tiles, which share their rows, for each pair
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int first_tile = (int)((long long)p.tiles * pair / pairs), last_tile = (int)((long long)p.tiles * (pair + 1) / pairs);

  if (warp == 1) {
    for (int i = lane; i < L::barriers; i += 32) {      // all of them lie side by side
      const uint32_t at = full_a + i * 8;
      tc::barrier_init(at, at >= drained && at < in_there       ? 2 * 4 * L::chunks * L::mates
                           : at >= full && at < empty && !RESIDENT ? 2
                                                                   : 1);
    }
    tc::barriers_visible();
  }
  if (warp == 2) tc::tensor_memory_take<L::memory>(where);
  const Place first(first_tile, p.tiles_n);
  tc::let_next_kernel_begin();
  tc::wait_for_last_kernel();
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

  const int steps = p.steps0 + p.steps1;
  if (warp == 0 || warp == 3) {
    // ---- operand tiles: this CTA's, into its shared memory; the first CTA's barriers count those of both.  One warp for each
    // operand: a step of a narrow tile is summed as fast as one thread asks for its operands. ----
    if (tc::one_lane()) {
      const bool own = RESIDENT && warp == 3;                    // A's slots have barriers of their own
      const uint32_t there = own ? full_a : full, gone = own ? empty_a : empty, first_there = tc::address_in(there, 0);
      const int slots = own ? steps : L::slots;
      int slot = 0, asked = 0;      // asked: no more than it takes to go round once
      uint32_t phase = 0;
      bool ok = true;
      auto take = [&](uint32_t bytes) {      // the next slot, once it is free
        ok = tc::wait(gone + slot * 8, phase ^ 1);
        if (ok && rank == 0) tc::arrive_expect(there + slot * 8, 2 * bytes);
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
        if (warp == 3) {
          const bool fresh = tile == first_tile || at_tile.n == 0, look = fresh && tile + p.tiles_n - at_tile.n < last_tile;
          if (RESIDENT && !fresh) continue;
          constexpr int PER = RESIDENT ? 1 : L::per;
          // the two sums of kGatedGrad share no slot
          for (int k = 0, count; k < steps; k += count, next()) {
            count = min(PER, (KIND == kGatedGrad && k < p.steps0 ? p.steps0 : steps) - k);
            if (!take(count * kOperandA)) break;
            uint32_t to = RESIDENT ? base_a + slot * kOperandA : ring + slot * L::slot + L::in_slot_b;
            for (int j = k; j < k + count; ++j, to += kOperandA) {
              const bool second = j >= p.steps0;
              const CUtensorMap *map = second ? &maps.a1 : &maps.a0;
              const int at = (second ? j - p.steps0 : j) * kDepth;
              tc::tile_load_pair(to, map, at, m0, first_there + slot * 8);
              if constexpr (RESIDENT) {
                if (look) tc::tile_to_l2(map, at, m0 + 2 * kRows);
              } else if (fresh) {
                // a few steps further, of these rows or of the next: all of a long sum's would push one another out of L2
                const int then = j + kAhead < steps ? j + kAhead : j + kAhead - steps;
                const bool here = j + kAhead < steps;
                if (here || (look && then < steps)) {
                  const bool other = then >= p.steps0;
                  tc::tile_to_l2(other ? &maps.a1 : &maps.a0, (other ? then - p.steps0 : then) * kDepth, here ? m0 : m0 + 2 * kRows);
                }
              }
            }
          }
        } else {
          const int first_steps = KIND == kGatedGrad ? p.steps0 : steps;
          for (int k = 0; k < first_steps; k += L::per, next()) {
            const int count = min(L::per, first_steps - k);
            if (!take(count * L::b_bytes)) break;
            uint32_t to = ring + slot * L::slot;
            for (int j = k; j < k + count; ++j, to += L::b_bytes) {
              if constexpr (KIND == kInputGrad) {
                const bool second = j >= p.steps0;
                const CUtensorMap *map = second ? &maps.b1 : &maps.b0;
                const int at = (second ? j - p.steps0 : j) * kDepth;
                constexpr int box = L::b_rows < 64 ? L::b_rows : 64;
#pragma unroll
                for (int i = 0; i < L::b_rows / box; ++i)
                  tc::tile_load_pair(to + i * kDepth * 128, map, n0 + (int)rank * L::b_rows + i * box, at, first_there + slot * 8);
              } else {
                tc::tile_load_pair(to, L::gated && rank ? &maps.b1 : &maps.b0, j * kDepth, L::gated ? n0 : n0 + (int)rank * L::b_rows,
                                   first_there + slot * 8);
              }
            }
          }
          if constexpr (KIND == kGatedGrad) {
            for (int k = 0; k < p.steps1 && ok; k += L::per_second, next()) {
              const int count = min(L::per_second, p.steps1 - k);
              if (!take(count * (L::b_bytes / 2))) break;
              uint32_t to = ring + slot * L::slot;
              for (int j = k; j < k + count; ++j, to += L::b_bytes / 2)
                tc::tile_load_pair(to, &maps.b2, n0 + (int)rank * L::b_ones, j * kDepth, first_there + slot * 8);
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
          tc::wait(there + slot * 8, phase);
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
      int at_ring = 0, slot = 0;
      uint32_t phase_a = 0, phase = 0, round = 0;
      bool ok = true;
      Place at_tile = first;
      for (int tile = first_tile; tile < last_tile && ok; ++tile, at_tile.on(1, p.tiles_n)) {
        const uint32_t acc = memory + slot * L::sums;
        const bool fresh = tile == first_tile || at_tile.n == 0, last = tile + 1 == last_tile || at_tile.n + 1 == p.tiles_n;
        if (!(ok = tc::wait_warp(drained + slot * 8, round ^ 1))) break;
        tc::order_after();
        auto sum = [&](auto second, int from, int to, uint32_t d) {
          constexpr bool SECOND = decltype(second)::value;      // kGatedGrad: grad_y Wd
          constexpr uint32_t form = SECOND ? shape_d : shape;
          constexpr int PER = SECOND ? L::per_second : L::per, bytes_b = SECOND ? L::b_bytes / 2 : L::b_bytes;
          constexpr bool mn = SECOND || KIND == kInputGrad, narrow_b = mn && L::b_ones < 64;
          constexpr int step_b = (narrow_b ? 1024 : mn ? 2048 : 32) / 16;
          for (int k = from; k < to; k += PER) {
            const int count = min(PER, to - k);
            if (RESIDENT && fresh)
              for (int j = 0; j < count; ++j)
                if (!(ok = tc::wait_warp(full_a + (k + j) * 8, phase_a))) return;
            if (!(ok = tc::wait_warp(full + at_ring * 8, phase))) return;
            tc::order_after();
            const uint32_t at_b = ring + at_ring * L::slot, at_a = RESIDENT ? base_a + k * kOperandA : at_b + L::in_slot_b;
            const uint64_t a = tc::k_major(at_a);
            const uint64_t b = narrow_b ? tc::mn_major_narrow(at_b) : mn ? tc::mn_major(at_b, kDepth * 128) : tc::k_major(at_b);
            if (tc::one_lane()) {
              tc::product(d, a, b, form, k > from);
#pragma unroll
              for (int j = 1; j < PER * (kDepth / 16); ++j) {
                const int step = j / (kDepth / 16), part = j % (kDepth / 16);
                if (step < count)
                  tc::product(d, a + step * (kOperandA / 16) + part * 2, b + step * (bytes_b / 16) + part * step_b, form, true);
              }
              if (RESIDENT && last)
                for (int j = 0; j < count; ++j) tc::products_arrive(empty_a + (k + j) * 8);
              tc::products_arrive(empty + at_ring * 8);
            }
            __syncwarp();
            if (++at_ring == L::slots) {
              at_ring = 0;
              phase ^= 1;
            }
          }
        };
        if constexpr (KIND == kGatedGrad) {
          sum(std::false_type(), 0, p.steps0, acc);
          if (ok) sum(std::true_type(), p.steps0, steps, acc + BN);
        } else {
          sum(std::false_type(), 0, steps, acc);
        }
        if (last) phase_a ^= 1;
        if (ok && tc::one_lane()) tc::products_arrive(summed + slot * 8);
        __syncwarp();
        if (++slot == L::depth) {
          slot = 0;
          round ^= 1;
        }
      }
      if (tc::one_lane()) tc::products_arrive(quiet);
      __syncwarp();
    }
    tc::wait_warp(quiet, 0);
  } else if (warp >= 4) {
    // ---- epilogue: a warp has 32 rows; the groups of four warps take a tile's chunks of columns in turn ----
    const int e = warp - 4, quarter = warp & 3, taker = (e >> 2) / L::mates, mate = (e >> 2) % L::mates;
    const uint32_t slab_in = slabs + (taker * 4 + quarter) * (L::outs * L::slab + L::slab_in), slab = slab_in + L::slab_in;
    auto meet = [&] {      // with the mate
      if constexpr (L::mates == 1) __syncwarp();
      else asm volatile("bar.sync %0, %1;" ::"r"(1 + taker * 4 + quarter), "n"(32 * L::mates) : "memory");
    };
    const uint32_t bias = bias_at + e * (L::bias / L::warps), there = in_there + e * 8, first_drained = tc::address_in(drained, 0);
    const bool loads = p.has_in && !DIRECT;
    const T *bias0 = static_cast<const T *>(p.bias0), *bias1 = static_cast<const T *>(p.bias1);
    uint32_t in_phase = 0;
    bool ok = true, comes = true;      // sums; what is added to them or multiplied by them

    // Chunk number c of this pair: tile first_tile + c / chunks; this warp has c = taker, taker + takers, ...
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
      h.place.on((h.c + L::takers) / L::chunks - h.c / L::chunks, p.tiles_n);
      h.c += L::takers;
      locate(h);
    };
    auto inside = [&](const Chunk &h) { return h.row < p.rows && h.column < p.n; };
    Chunk now{taker, 0, 0, first};
    now.place.on(taker / L::chunks, p.tiles_n);
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
    constexpr int ahead = (L::part + 31) / 32;
    float next0[ahead], next1[ahead];
    auto ask_bias = [&] {
#pragma unroll
      for (int i = 0; i < ahead; ++i) {
        const int k = i * 32 + lane, col = now.column + mate * L::part + k;
        const bool in = now.c < all && k < L::part && col < p.n;
        next0[i] = in && bias0 ? wide(bias0[col]) : 0.f;
        if constexpr (L::gated) next1[i] = in && bias1 ? wide(bias1[col]) : 0.f;
      }
    };
    if constexpr (KIND != kInputGrad) ask_bias();

    while (now.c < all) {
      const int it = now.c / L::chunks, slot = it % L::depth, m0 = now.row, col = now.column;
      const uint32_t acc = memory + ((uint32_t)quarter << 21) + slot * L::sums + now.c % L::chunks * L::chunk + mate * L::part;
      const bool some = inside(now);
      const int rows_in = min(32, p.rows - m0), cols_in = min(L::chunk, p.n - col);
      if constexpr (KIND != kInputGrad) {
#pragma unroll
        for (int i = 0; i < ahead; ++i) {
          const int k = i * 32 + lane;
          if (k >= L::part) continue;
          tc::write_one<float>(bias + k * 4, next0[i]);
          if constexpr (L::gated) tc::write_one<float>(bias + (L::part + k) * 4, next1[i]);
        }
        go_on(now);
        ask_bias();
      } else {
        go_on(now);
      }
      __syncwarp();
      if (some) {
        if (DIRECT && p.has_in) {
          __syncwarp();
          copy_rows_direct<I, L::in_bytes, false>(static_cast<const I *>(p.in) + m0 * p.in_pitch + col, p.in_pitch, rows_in, cols_in,
                                                  slab_in, lane);
        } else if ((!loads || L::apart) && lane == 0 && mate == 0) {
          tc::stores_read<0>();
        }
        meet();
      }
      if (ok) ok = __all_sync(0xffffffffu, tc::wait(summed + slot * 8, (uint32_t)(it / L::depth) & 1));
      tc::order_after();
      if (some) {
        if (loads && comes) {
          comes = __all_sync(0xffffffffu, tc::wait(there, in_phase));
          in_phase ^= 1;
          ok = ok && comes;
        }
        // columns of the accumulators, the next ones on their way while these are worked on
        constexpr int sums = KIND == kGatedGrad ? 3 : L::gated ? 2 : 1, turns = L::part / L::sub;
        float v[2][sums][L::sub];
        auto fetch = [&](int t) {
#pragma unroll
          for (int i = 0; i < sums; ++i) tc::tensor_load(v[t & 1][i], acc + i * (BN / 2) + t * L::sub);
        };
        fetch(0);
#pragma unroll
        for (int t = 0; t < turns; ++t) {
          const int off = t * L::sub, first = (mate * L::part + off) * (int)sizeof(O) / 16;
          float(&z)[L::sub] = v[t & 1][0];
#pragma unroll
          for (int i = 0; i < sums; ++i) tc::tensor_loads_done(v[t & 1][i]);
          if (t + 1 < turns) {
            fetch(t + 1);
          } else {      // the accumulator may be summed into again
            tc::order_before();
            __syncwarp();
            if (ok && lane == 0) tc::arrive_in(first_drained + slot * 8);
          }
          if constexpr (KIND != kInputGrad) add_bias(z, bias + off * 4);
          if constexpr (L::gated) add_bias(v[t & 1][1], bias + (L::part + off) * 4);
          if constexpr (KIND == kGatedGrad) {
            float(&u)[L::sub] = v[t & 1][1], (&d)[L::sub] = v[t & 1][2];
            gate_all(z, u, d, p.act);
            put<O, L::row_bytes>(d, slab + L::slab, lane, first);
            put<O, L::row_bytes>(u, slab + 2 * L::slab, lane, first);
          } else if constexpr (KIND == kGated) {
            activate_all(z, p.act);
#pragma unroll
            for (int i = 0; i < L::sub; i += 2) {
              const Two h = Two{z[i], z[i + 1]} * Two{v[t & 1][1][i], v[t & 1][1][i + 1]};
              z[i] = h.x;
              z[i + 1] = h.y;
            }
          } else {
            if constexpr (KIND == kLinear) activate_all(z, p.act);
            if constexpr (KIND == kSlope) slope_all(z, p.act);
            if (p.has_in) combine<I, L::in_bytes, KIND == kSlope>(z, slab_in, lane, off * (int)sizeof(I) / 16);
          }
          put<O, L::row_bytes>(z, slab, lane, first);
        }
      }
      if (!some) {
        __syncwarp();
        if (ok && lane == 0) tc::arrive_in(first_drained + slot * 8);
        continue;
      }
      if (!ok)
        for (int o = 0; o < L::outs; ++o) lose_row<L::row_bytes>(slab + o * L::slab, lane);
      if (!DIRECT) tc::shared_to_async();
      meet();
      if constexpr (DIRECT) {
        copy_rows_direct<O, L::row_bytes, true>(static_cast<O *>(p.out) + m0 * p.out_pitch + col, p.out_pitch, rows_in, cols_in, slab, lane);
      } else if (lane == 0 && mate == 0) {
#pragma unroll
        for (int o = 0; o < L::outs; ++o) tc::tile_store(&maps.out[o], col, m0, slab + o * L::slab);
        tc::stores_asked();
        if (loads) {
          if (!L::apart) tc::stores_read<0>();
          if (comes) ask();
        }
      }
    }
    if (!comes) tc::wait(there, in_phase ^ 1);      // what is late may still be on its way
    if (lane == 0) tc::stores_done();
  }
  tc::order_before();
  __syncwarp();
  tc::pair_sync();      // the other CTA's products read this one's shared memory, its warps arrive at this one's barriers
  if (warp == 2) {
    tc::order_after();
    tc::tensor_memory_give<L::memory>(memory);
  }
}

template <typename I, typename O> bool lies_direct(const ProductArgs &a) {
  auto fits = [](const void *q, long long pitch, size_t size) {
    return (reinterpret_cast<uintptr_t>(q) & 15u) == 0 && pitch * size % 16 == 0;
  };
  return !fits(a.out[0], a.out_pitch, sizeof(O)) || (a.in.data && !fits(a.in.data, a.in.pitch, sizeof(I)));
}

template <ProductKind KIND, typename T, typename I, typename O, int BN, bool RESIDENT, bool DIRECT>
cudaError_t launch_as(const ProductArgs &a, cudaStream_t s) {
  using L = Tile<KIND, I, O, BN, RESIDENT>;
  auto code = [&](size_t size) { return size == 4 ? DFA3D_DTYPE_F32 : a.dtype; };
  Maps m{};
  Extents p{};
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
  if constexpr (!DIRECT) {
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
  constexpr auto kernel = &product_kernel<KIND, T, I, O, BN, RESIDENT, DIRECT>;
  cudaError_t rc = allow_shared<kernel>(L::bytes);
  if (rc != cudaSuccess) return rc;
  const int pairs = sm_count() / 2, grid = 2 * (p.tiles < pairs ? p.tiles : pairs);
  return launch_after(kernel, grid, L::threads, L::bytes, s, m, p);
}

template <ProductKind KIND, typename T, typename I, typename O, int BN, bool DIRECT = false>
cudaError_t launch_tiles(const ProductArgs &a, cudaStream_t s) {
  const int steps = (a.k0 + kDepth - 1) / kDepth + (a.k1 + kDepth - 1) / kDepth;
  return steps <= Tile<KIND, I, O, BN, true>::slots_a ? launch_as<KIND, T, I, O, BN, true, DIRECT>(a, s)
                                                      : launch_as<KIND, T, I, O, BN, false, DIRECT>(a, s);
}

// Any width for results of the caller, narrow tiles where they lie off the 16-byte grid.
template <ProductKind KIND, typename T, typename O> cudaError_t launch_widths(const ProductArgs &a, int width, cudaStream_t s) {
  if (lies_direct<O, O>(a)) return launch_tiles<KIND, T, O, O, 64, true>(a, s);
  return width == 256   ? launch_tiles<KIND, T, O, O, 256>(a, s)
         : width == 128 ? launch_tiles<KIND, T, O, O, 128>(a, s)
                        : launch_tiles<KIND, T, O, O, 64>(a, s);
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
  // the results of the other kinds are workspaces
  if (a.kind != kLinear && a.kind != kInputGrad && lies_direct<T, T>(a) && !a.wide) return cudaErrorInvalidValue;
  switch (a.kind) {
    case kLinear: {
      const int w = tile_width(a.rows, a.n, 256);
      return a.wide ? launch_widths<kLinear, T, float>(a, w, s) : launch_widths<kLinear, T, T>(a, w, s);
    }
    case kSlope: {
      const bool narrow = tile_width(a.rows, a.n, 128) == 64;
      if (a.wide) return narrow ? launch_tiles<kSlope, T, float, T, 64>(a, s) : launch_tiles<kSlope, T, float, T, 128>(a, s);
      return narrow ? launch_tiles<kSlope, T, T, T, 64>(a, s) : launch_tiles<kSlope, T, T, T, 128>(a, s);
    }
    case kGated:
      return tile_width(a.rows, a.n, 128) == 128 ? launch_tiles<kGated, T, T, T, 256>(a, s) : launch_tiles<kGated, T, T, T, 128>(a, s);
    case kGatedGrad: return launch_tiles<kGatedGrad, T, T, T, 128>(a, s);
    case kInputGrad: return launch_widths<kInputGrad, T, T>(a, tile_width(a.rows, a.n, 256), s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_product(const ProductArgs &a, cudaStream_t s) {
  if (const cudaError_t rc = bind_context()) return rc;
  return a.dtype == DFA3D_DTYPE_F16 ? launch_typed<__half>(a, s) : launch_typed<__nv_bfloat16>(a, s);
}

}  // namespace dfa3d
