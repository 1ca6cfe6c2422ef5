// The gated feed-forward block with one kernel: y = (act(x Wg^T + bg) * (x Wu^T + bu)) Wd^T + bd + residual, whose hidden rows never leave
// the SMs.  Written to memory and read again they are most of what the two kernels of dfa3d_product.cu move (82 of 123 MB for 40 000 rows
// 256 -> 512 -> 256 with a 16-bit residual that is x).
//
// A pair of CTAs takes 256 rows, which stay (64 KB each), and walks over 128 hidden columns at a time: gate and up are summed in half of
// tensor memory, sixteen warps read them at once, so that the next ones may be summed, and turn them into hidden rows in shared memory,
// which are the operand of the next product, summed in the other half over all hidden columns.  The products of one item and the sums of
// the next are issued in turn, so that the tensor cores sum while the warps work; a result is read while the next rows begin.
//
// Measured against the two kernels, us, bf16, SiLU, behind a flush of L2 / on calls that follow one another:
//   16-bit residual: 256 -> 512 -> 256, 30 000 rows 36.9 to 42.0 / 28.2 to 35.1, 40 000 rows 47.1 to 48.2 / 39.3 to 43.0, 80 000 rows 69.6
//   to 78.8 / 61.9 to 74.1; 256 -> 1024 -> 256, 80 000 rows 115 to 136 / 107 to 133.
//   32-bit residual: 45.1 to 48.1 / 33.2 to 43.9, 59.4 to 56.4 / 50.2 to 51.0, 90.1 to 93.2 / 81.6 to 89.2; 144 to 161 / 135 to 155.  The
//   result's chunks, twice as many, take most of what the hidden rows save; at 40 000 rows all of it.
// The floor of 40 000 rows is 31.5 GFLOP, 20 us at 1.6 PFLOP/s.  What binds is the chain of an item -- products, 32 columns of math a warp,
// hand-over -- of about 3900 cycles, and 5200 between the rows of two tiles, where a warp's chunks of the result go through one slab
// one after the other: two slabs a warp leave three slots of the ring instead of five, which cost wide blocks 10 %.  157 tiles of rows
// over 74 pairs are three rounds for 2.1 rounds of work.
#include "dfa3d_common.cuh"
#include "dfa3d_epilogue.cuh"
#include "dfa3d_product.h"
#include "dfa3d_tensor_map.h"

namespace dfa3d {
namespace {

constexpr int kRows = 128, kDepth = 64, kHidden = 128;      // of a CTA's tile; along a summed axis; hidden columns of an item
constexpr int kOperandA = kRows * kDepth * 2, kStepsA = 4;
constexpr int kWarps = 16, kThreads = (4 + kWarps) * 32;

struct Maps {
  CUtensorMap x, gate, up, down, in, out;
};
struct Extents {
  int rows, n, hidden, steps, across, tiles;      // steps of kDepth of x, steps of kHidden, pairs of row tiles
  int act, has_in;
  const void *bias_gate, *bias_up, *bias_down;
};

template <typename O, int BN> struct Block {
  static constexpr int slot = kHidden * kDepth * 2, slots = 5;                 // a step of gate or up, or of down
  static constexpr int down_rows = BN / 2, down_bytes = down_rows * kDepth * 2;
  static constexpr int hidden = kRows * kHidden * 2;
  static constexpr int chunk = 64 / (int)sizeof(O), part = BN / 4, chunks = part / chunk;      // columns of the result: at a time, of a warp
  static constexpr int slab = 32 * 64;
  static constexpr int bias = (64 + 32) * 4;
  static constexpr int sums_y = 2 * kHidden;                                   // tensor memory: gate and up, then the result
  static constexpr int barriers = 2 * kStepsA + 2 * slots + 4 + 2 + kWarps + 1;
  static constexpr int bytes = kStepsA * kOperandA + hidden + slots * slot + kWarps * (slab + bias) + barriers * 8 + 16;
  static_assert(one_an_sm(bytes) && bytes <= 227 * 1024 && down_bytes <= slot && chunks >= 1, "layout");
};

template <typename T, typename O, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    gated_block_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Extents p) {
  using L = Block<O, BN>;
  extern __shared__ __align__(1024) uint8_t raw[];
  const uint32_t base_a = tc::shared_address(raw), base_h = base_a + kStepsA * kOperandA, ring = base_h + L::hidden;
  const uint32_t slabs = ring + L::slots * L::slot, bias_at = slabs + kWarps * L::slab;
  const uint32_t full_a = bias_at + kWarps * L::bias, empty_a = full_a + kStepsA * 8, full = empty_a + kStepsA * 8, empty = full + L::slots * 8;
  const uint32_t summed = empty + L::slots * 8, drained = summed + 8, h_full = drained + 8, h_empty = h_full + 8;
  const uint32_t y_full = h_empty + 8, y_empty = y_full + 8, in_there = y_empty + 8, quiet = in_there + kWarps * 8, where = quiet + 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = tc::rank_in_pair();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int first_tile = (int)((long long)p.tiles * pair / pairs), last_tile = (int)((long long)p.tiles * (pair + 1) / pairs);

  if (warp == 1) {
    for (int i = lane; i < L::barriers; i += 32) {      // all of them lie side by side
      const uint32_t at = full_a + i * 8;
      tc::barrier_init(at, at == drained || at == h_full || at == y_empty ? 2 * kWarps : 1);      // the warps of both CTAs
    }
    tc::barriers_visible();
  }
  if (warp == 2) tc::tensor_memory_take<512>(where);
  tc::let_next_kernel_begin();
  tc::wait_for_last_kernel();
  tc::order_before();
  __syncwarp();
  tc::pair_sync();
  tc::order_after();
  uint32_t memory;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(memory) : "r"(where));
  const int items = (last_tile - first_tile) * p.across;      // (rows, hidden columns), hidden columns first

  if (warp == 0 || warp == 3) {
    // ---- operands: this CTA's; the first CTA's barriers count those of both ----
    if (tc::one_lane()) {
      const bool is_x = warp == 3;
      const uint32_t there = is_x ? full_a : full, gone = is_x ? empty_a : empty, first_there = tc::address_in(there, 0);
      const int slots = is_x ? p.steps : L::slots;
      int slot = 0, asked = 0;
      uint32_t phase = 0;
      bool ok = true;
      auto take = [&](uint32_t bytes) {
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
      if (is_x) {
        for (int tile = first_tile; tile < last_tile && ok; ++tile) {
          const int m0 = (tile * 2 + (int)rank) * kRows;
          for (int k = 0; k < p.steps; ++k, next()) {
            if (!take(kOperandA)) break;
            tc::tile_load_pair(base_a + k * kOperandA, &maps.x, k * kDepth, m0, first_there + slot * 8);
            if (tile + 1 < last_tile) tc::tile_to_l2(&maps.x, k * kDepth, m0 + 2 * kRows);
          }
        }
      } else {
        int j = 0, last = 0;
        for (int item = 0; item <= items && ok; ++item) {
          if (item < items) {
            for (int k = 0; k < p.steps; ++k, next()) {
              if (!take(L::slot)) break;
              tc::tile_load_pair(ring + slot * L::slot, rank ? &maps.up : &maps.gate, k * kDepth, j * kHidden, first_there + slot * 8);
            }
          }
          if (item > 0 && ok) {
            for (int k = 0; k < kHidden / kDepth; ++k, next()) {
              if (!take(L::down_bytes)) break;
              tc::tile_load_pair(ring + slot * L::slot, &maps.down, last * kHidden + k * kDepth, (int)rank * L::down_rows,
                                 first_there + slot * 8);
            }
          }
          last = j;
          if (++j == p.across) j = 0;
        }
      }
      if (rank == 0) {      // nothing may be on its way into shared memory when the CTAs end
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
    if (rank == 0) {
      constexpr uint32_t shape = tc::product_shape<T>(2 * kRows, 2 * kHidden, false, false), shape_y = tc::product_shape<T>(2 * kRows, BN, false, false);
      int slot = 0, j = 0, last = 0, rows_done = 0;
      uint32_t phase = 0, phase_a = 0;
      bool ok = true;
      auto next = [&] {
        if (++slot == L::slots) {
          slot = 0;
          phase ^= 1;
        }
      };
      for (int item = 0; item <= items && ok; ++item) {
        if (item < items) {      // gate and up of this item
          if (!(ok = tc::wait_warp(drained, (uint32_t)(item + 1) & 1))) break;
          tc::order_after();
          for (int k = 0; k < p.steps; ++k) {
            if (j == 0 && !(ok = tc::wait_warp(full_a + k * 8, phase_a))) break;
            if (!(ok = tc::wait_warp(full + slot * 8, phase))) break;
            tc::order_after();
            const uint64_t a = tc::k_major(base_a + k * kOperandA), b = tc::k_major(ring + slot * L::slot);
            if (tc::one_lane()) {
              tc::product(memory, a, b, shape, k > 0);
#pragma unroll
              for (int i = 1; i < 4; ++i) tc::product(memory, a + i * 2, b + i * 2, shape, true);
              if (j + 1 == p.across) tc::products_arrive(empty_a + k * 8);
              tc::products_arrive(empty + slot * 8);
              if (k + 1 == p.steps) tc::products_arrive(summed);
            }
            __syncwarp();
            next();
          }
          if (j + 1 == p.across) phase_a ^= 1;
        }
        if (item > 0 && ok) {      // the result's share of the last one
          const int of = item - 1;
          if (last == 0 && !(ok = tc::wait_warp(y_empty, (uint32_t)(rows_done + 1) & 1))) break;
          if (!(ok = tc::wait_warp(h_full, (uint32_t)of & 1))) break;
          for (int k = 0; k < kHidden / kDepth; ++k) {
            if (!(ok = tc::wait_warp(full + slot * 8, phase))) break;
            tc::order_after();
            const uint64_t a = tc::k_major(base_h + k * kOperandA), b = tc::k_major(ring + slot * L::slot);
            if (tc::one_lane()) {
              tc::product(memory + L::sums_y, a, b, shape_y, last > 0 || k > 0);
#pragma unroll
              for (int i = 1; i < 4; ++i) tc::product(memory + L::sums_y, a + i * 2, b + i * 2, shape_y, true);
              tc::products_arrive(empty + slot * 8);
              if (k + 1 == kHidden / kDepth) {
                tc::products_arrive(h_empty);
                if (last + 1 == p.across) tc::products_arrive(y_full);
              }
            }
            __syncwarp();
            next();
          }
          if (last + 1 == p.across) ++rows_done;
        }
        last = j;
        if (++j == p.across) j = 0;
      }
      if (tc::one_lane()) tc::products_arrive(quiet);
      __syncwarp();
    }
    tc::wait_warp(quiet, 0);
  } else if (warp >= 4) {
    // ---- hidden rows and results: a warp has 32 rows, a quarter of the columns ----
    const int e = warp - 4, quarter = warp & 3, group = e >> 2;
    const uint32_t slab = slabs + e * L::slab, bias = bias_at + e * L::bias, there = in_there + e * 8;
    const uint32_t first_drained = tc::address_in(drained, 0), first_h_full = tc::address_in(h_full, 0), first_y_empty = tc::address_in(y_empty, 0);
    const uint32_t lanes = memory + ((uint32_t)quarter << 21);
    const T *bias_gate = static_cast<const T *>(p.bias_gate), *bias_up = static_cast<const T *>(p.bias_up);
    const T *bias_down = static_cast<const T *>(p.bias_down);
    const int y_column = group * L::part;
    uint32_t in_phase = 0;
    bool ok = true, comes = true;      // sums and hidden rows; residuals

    auto row_of = [&](int tile) { return (tile * 2 + (int)rank) * kRows + quarter * 32; };
    auto inside = [&](int tile, int c) { return row_of(tile) < p.rows && y_column + c * L::chunk < p.n; };
    int ask_tile = first_tile, ask_c = -1;
    auto ask = [&] {      // of the next chunk with something inside, the residual
      do {
        if (++ask_c == L::chunks) {
          ask_c = 0;
          ++ask_tile;
        }
      } while (ask_tile < last_tile && !inside(ask_tile, ask_c));
      if (ask_tile >= last_tile) return;
      tc::arrive_expect(there, L::slab);
      tc::tile_load(slab, &maps.in, y_column + ask_c * L::chunk, row_of(ask_tile), there);
    };
    if (p.has_in && lane == 0) ask();

    auto result = [&](int tile, int done) {      // of the rows of `tile`, the done-th of this pair
      if (ok) ok = __all_sync(0xffffffffu, tc::wait(y_full, (uint32_t)done & 1));
      tc::order_after();
#pragma unroll
      for (int c = 0; c < L::chunks; ++c) {
        const int col = y_column + c * L::chunk;
        if (inside(tile, c)) {
          if (lane < L::chunk) {
            const bool in = bias_down && col + lane < p.n;
            tc::write_one<float>(bias + (64 + lane) * 4, in ? wide(bias_down[col + lane]) : 0.f);
          }
          if (!p.has_in && lane == 0) tc::stores_read<0>();
          __syncwarp();
          if (p.has_in && comes) {
            comes = __all_sync(0xffffffffu, tc::wait(there, in_phase));
            in_phase ^= 1;
            ok = ok && comes;
          }
#pragma unroll
          for (int off = 0; off < L::chunk; off += 16) {
            float z[16];
            tc::tensor_load(z, lanes + L::sums_y + col + off);
            tc::tensor_loads_done(z);
            add_bias(z, bias + (64 + off) * 4);
            if (p.has_in) combine<O, 64, false>(z, slab, lane, off * (int)sizeof(O) / 16);
            put<O, 64>(z, slab, lane, off * (int)sizeof(O) / 16);
          }
        }
        if (c + 1 == L::chunks) {
          tc::order_before();
          __syncwarp();
          if (ok && lane == 0) tc::arrive_in(first_y_empty);
        }
        if (!inside(tile, c)) continue;
        if (!ok) lose_row<64>(slab, lane);
        tc::shared_to_async();
        __syncwarp();
        if (lane == 0) {
          tc::tile_store(&maps.out, col, row_of(tile), slab);
          tc::stores_asked();
          if (p.has_in) {
            tc::stores_read<0>();
            if (comes) ask();
          }
        }
        __syncwarp();
      }
    };

    int j = 0, tile = first_tile;
    float next_gate = 0.f, next_up = 0.f;
    auto ask_bias = [&] {
      const int col = j * kHidden + group * 32 + lane;
      next_gate = bias_gate && col < p.hidden ? wide(bias_gate[col]) : 0.f;
      next_up = bias_up && col < p.hidden ? wide(bias_up[col]) : 0.f;
    };
    ask_bias();
    for (int item = 0; item < items; ++item) {
      const bool begin = j == 0 && tile > first_tile;
      const int before = tile - 1;
      tc::write_one<float>(bias + lane * 4, next_gate);
      tc::write_one<float>(bias + (32 + lane) * 4, next_up);
      if (++j == p.across) {
        j = 0;
        ++tile;
      }
      ask_bias();
      __syncwarp();
      if (ok) ok = __all_sync(0xffffffffu, tc::wait(summed, (uint32_t)item & 1));
      tc::order_after();
      const uint32_t acc = lanes + group * 32;
      float g[2][16], u[2][16];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        tc::tensor_load(g[t], acc + t * 16);
        tc::tensor_load(u[t], acc + kHidden + t * 16);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        tc::tensor_loads_done(g[t]);
        tc::tensor_loads_done(u[t]);
      }
      tc::order_before();
      __syncwarp();
      if (ok && lane == 0) tc::arrive_in(first_drained);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        add_bias(g[t], bias + t * 64);
        add_bias(u[t], bias + 128 + t * 64);
        activate_all(g[t], p.act);
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const Two h = Two{g[t][i], g[t][i + 1]} * Two{u[t][i], u[t][i + 1]};
          g[t][i] = h.x;
          g[t][i + 1] = h.y;
        }
        if (t == 0 && ok) ok = __all_sync(0xffffffffu, tc::wait(h_empty, (uint32_t)(item + 1) & 1));
        if (ok) put<T, 128>(g[t], base_h + (group >> 1) * kOperandA + quarter * 32 * 128, lane, (group & 1) * 4 + t * 2);
      }
      tc::shared_to_async();
      __syncwarp();
      if (ok && lane == 0) tc::hand_over_in(first_h_full);
      // the result of the rows before these is there when the first hidden columns of these have been made
      if (begin) result(before, before - first_tile);
    }
    if (items > 0) result(last_tile - 1, last_tile - 1 - first_tile);
    if (!comes) tc::wait(there, in_phase ^ 1);      // a residual that is late may still be on its way
    if (lane == 0) tc::stores_done();
  }
  tc::order_before();
  __syncwarp();
  tc::pair_sync();      // the other CTA's products read this one's shared memory, its warps arrive at this one's barriers
  if (warp == 2) {
    tc::order_after();
    tc::tensor_memory_give<512>(memory);
  }
}

template <typename T, typename O, int BN> cudaError_t launch_block(const ProductArgs &a, int hidden, const void *bias2, cudaStream_t s) {
  using L = Block<O, BN>;
  const int out_type = sizeof(O) == 4 ? DFA3D_DTYPE_F32 : a.dtype;
  Maps m{};
  if (!describe_matrix(m.x, a.dtype, a.a0.data, a.rows, a.k0, a.a0.pitch, kDepth, kRows) ||
      !describe_matrix(m.gate, a.dtype, a.b0.data, hidden, a.k0, a.b0.pitch, kDepth, kHidden) ||
      !describe_matrix(m.up, a.dtype, a.b1.data, hidden, a.k0, a.b1.pitch, kDepth, kHidden) ||
      !describe_matrix(m.down, a.dtype, a.b2.data, a.n, hidden, a.b2.pitch, kDepth, L::down_rows) ||
      !describe_matrix(m.out, out_type, a.out[0], a.rows, a.n, a.out_pitch, L::chunk, 32) ||
      (a.in.data && !describe_matrix(m.in, out_type, a.in.data, a.rows, a.n, a.in.pitch, L::chunk, 32)))
    return cudaErrorInvalidValue;
  Extents p{};
  p.rows = (int)a.rows;
  p.n = a.n;
  p.hidden = hidden;
  p.steps = (a.k0 + kDepth - 1) / kDepth;
  p.across = (hidden + kHidden - 1) / kHidden;
  p.tiles = (int)((a.rows + 2 * kRows - 1) / (2 * kRows));
  p.act = a.act;
  p.has_in = a.in.data != nullptr;
  p.bias_gate = a.bias0;
  p.bias_up = a.bias1;
  p.bias_down = bias2;
  constexpr auto kernel = &gated_block_kernel<T, O, BN>;
  cudaError_t rc = allow_shared<kernel>(L::bytes);
  if (rc != cudaSuccess) return rc;
  const int pairs = sm_count() / 2;
  return launch_after(kernel, 2 * (p.tiles < pairs ? p.tiles : pairs), kThreads, L::bytes, s, m, p);
}

template <typename T, typename O> cudaError_t launch_typed(const ProductArgs &a, int hidden, const void *bias2, cudaStream_t s) {
  return a.n > 128 ? launch_block<T, O, 256>(a, hidden, bias2, s) : launch_block<T, O, 128>(a, hidden, bias2, s);
}

}  // namespace

bool gated_block_covers(const ProductArgs &a, int hidden) {
  const int size = a.wide ? 4 : 2;
  auto fits = [&](const void *q, long long pitch) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0 && pitch * size % 16 == 0; };
  if (a.k0 > kStepsA * kDepth || a.n > 256 || !fits(a.out[0], a.out_pitch) || (a.in.data && !fits(a.in.data, a.in.pitch))) return false;
  // What of the time of the busiest pair of SMs the average one has work for: the two kernels' tiles are narrower and divide more evenly.
  // At 38 row tiles for 74 pairs one kernel takes 0.75 to 0.87 of the two kernels' time up to 512 hidden columns, 0.86 to 0.9 with 1024
  // and 0.95 to 1.05 with 2048; at 75 tiles 0.93 to 1.0, but with 1024 and 2048, where a tile takes longer, 1.04 to 1.17, at 86 tiles
  // then 0.9 to 1.1, at 118 0.8 to 0.95.  Measured with 16-bit residuals; with 32-bit ones 0.75 to 1.02, and behind a flush of L2
  // 1.05 at 157 tiles of 512 hidden columns.
  const long long tiles = (a.rows + 2 * kRows - 1) / (2 * kRows), pairs = sm_count() / 2, rounds = (tiles + pairs - 1) / pairs;
  return tiles * 10 >= rounds * pairs * (rounds > 1 && hidden > 512 ? 6 : 5);
}

cudaError_t launch_gated_block(const ProductArgs &a, int hidden, const void *bias2, cudaStream_t s) {
  if (const cudaError_t rc = bind_context()) return rc;
  if (a.dtype == DFA3D_DTYPE_F16)
    return a.wide ? launch_typed<__half, float>(a, hidden, bias2, s) : launch_typed<__half, __half>(a, hidden, bias2, s);
  return a.wide ? launch_typed<__nv_bfloat16, float>(a, hidden, bias2, s) : launch_typed<__nv_bfloat16, __nv_bfloat16>(a, hidden, bias2, s);
}

}  // namespace dfa3d
