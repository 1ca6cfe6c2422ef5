// Matrix products of a feed-forward block with everything that follows them in their epilogue.  One CTA an SM walks over tiles of 128
// rows: a warp asks for operand tiles of 64 along the summed axis (tiled copies into a ring), one thread issues the products, whose
// 32-bit sums stay in tensor memory, twice over, so that the next tile is summed while eight warps read this one, apply bias,
// activation, residual or derivatives in 32 bits, round once and hand rows to tiled stores.
#include "dfa3d_act.cuh"
#include "dfa3d_common.cuh"
#include "dfa3d_product.h"
#include "dfa3d_rowvec.cuh"
#include "dfa3d_tcgen05.cuh"
#include "dfa3d_tensor_map.h"

namespace dfa3d {
namespace {

constexpr int kRows = 128, kDepth = 64;          // of a tile; along the summed axis, 128 bytes
constexpr int kEpilogueWarps = 8, kProductThreads = (4 + kEpilogueWarps) * 32;
constexpr int kOperandA = kRows * kDepth * 2;

struct Maps {
  CUtensorMap a0, a1, b0, b1, b2, in, out[3];
};
struct Extents {
  int rows, n, steps0, steps1;      // steps of kDepth
  int tiles, tiles_n;
  int act, has_in, direct;          // direct: `in` and `out` are read and written element by element
  const void *bias0, *bias1, *in;
  void *out;
  long long in_pitch, out_pitch;
};

template <ProductKind KIND, typename O, int BN> struct Tile {
  static constexpr bool gated = KIND == kGated || KIND == kGatedGrad;
  static constexpr int outs = KIND == kGatedGrad ? 3 : 1;
  static constexpr int columns = gated ? BN / 2 : BN;                            // of a result
  static constexpr int sums = KIND == kGatedGrad ? BN + BN / 2 : BN;             // accumulator columns
  static constexpr int memory = 2 * sums <= 128 ? 128 : 2 * sums <= 256 ? 256 : 512;
  static constexpr int operand_b = BN * kDepth * 2, stage = kOperandA + operand_b;
  static constexpr int stages = BN == 256 || KIND == kGatedGrad ? 3 : 4;
  static constexpr int half = columns / 2;                                       // of an epilogue warp
  static constexpr int chunk = half < 128 / (int)sizeof(O) ? half : 128 / (int)sizeof(O), chunks = half / chunk;
  static constexpr int row_bytes = chunk * (int)sizeof(O), slab = 32 * row_bytes;
  static constexpr int slabs = 2 * outs * kEpilogueWarps * slab;
  static constexpr int bias = half * (gated ? 2 : 1) * 4;
  static constexpr int barriers = 2 * stages + 4 + 2 * kEpilogueWarps + 1;
  static constexpr int bytes = 1024 + stages * stage + slabs + kEpilogueWarps * bias + barriers * 8 + 16;
  static_assert(bytes <= 227 * 1024 && (row_bytes == 64 || row_bytes == 128) && chunk % 32 == 0, "layout");
};

// The 16-byte piece `piece` of row `row` of a slab as tiled copies lay it out.
template <int ROW_BYTES> __device__ __forceinline__ uint32_t piece_of(uint32_t slab, int row, int piece) {
  const int mix = ROW_BYTES == 128 ? row & 7 : (row >> 1) & 3;
  return slab + row * ROW_BYTES + ((piece ^ mix) << 4);
}

template <int ACT> __device__ __forceinline__ void activate_each(float (&z)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i) z[i] = activate<ACT>(z[i]);
}
__device__ __forceinline__ void activate_all(float (&z)[32], int act) {
  switch (act) {
    case DFA3D_ROW_RELU: return activate_each<DFA3D_ROW_RELU>(z);
    case DFA3D_ROW_SILU: return activate_each<DFA3D_ROW_SILU>(z);
    case DFA3D_ROW_GELU: return activate_each<DFA3D_ROW_GELU>(z);
    default: return;
  }
}
template <int ACT> __device__ __forceinline__ void slope_each(float (&z)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    float a;
    activate_both<ACT>(z[i], a, z[i]);
  }
}
__device__ __forceinline__ void slope_all(float (&z)[32], int act) {
  switch (act) {
    case DFA3D_ROW_RELU: return slope_each<DFA3D_ROW_RELU>(z);
    case DFA3D_ROW_SILU: return slope_each<DFA3D_ROW_SILU>(z);
    case DFA3D_ROW_GELU: return slope_each<DFA3D_ROW_GELU>(z);
    default: return slope_each<DFA3D_ROW_NONE>(z);
  }
}
// gate, up, d -> d up act'(gate), d act(gate), act(gate) up
template <int ACT> __device__ __forceinline__ void gate_each(float (&g)[32], float (&u)[32], float (&d)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    float a, s;
    activate_both<ACT>(g[i], a, s);
    g[i] = d[i] * u[i] * s;
    d[i] = d[i] * a;
    u[i] = a * u[i];
  }
}
__device__ __forceinline__ void gate_all(float (&g)[32], float (&u)[32], float (&d)[32], int act) {
  switch (act) {
    case DFA3D_ROW_RELU: return gate_each<DFA3D_ROW_RELU>(g, u, d);
    case DFA3D_ROW_SILU: return gate_each<DFA3D_ROW_SILU>(g, u, d);
    case DFA3D_ROW_GELU: return gate_each<DFA3D_ROW_GELU>(g, u, d);
    default: return gate_each<DFA3D_ROW_NONE>(g, u, d);
  }
}

__device__ __forceinline__ void add_bias(float (&z)[32], uint32_t bias) {
#pragma unroll
  for (int i = 0; i < 32; i += 4) {
    const float4 b = tc::read_four(bias + i * 4);
    z[i] += b.x; z[i + 1] += b.y; z[i + 2] += b.z; z[i + 3] += b.w;
  }
}

// 32 columns of this lane's row into a slab, from piece `first` on
template <typename O, int ROW_BYTES> __device__ __forceinline__ void put(const float (&z)[32], uint32_t slab, int row, int first) {
  constexpr int V = 16 / (int)sizeof(O);
#pragma unroll
  for (int i = 0; i < 32; i += V) {
    float f[V];
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = z[i + k];
    const uint4 w = narrow_word<O, V>(f);
    tc::write16(piece_of<ROW_BYTES>(slab, row, first + i / V), w);
  }
}
// z = z + slab, or z * slab
template <typename O, int ROW_BYTES, bool TIMES>
__device__ __forceinline__ void combine(float (&z)[32], uint32_t slab, int row, int first) {
  constexpr int V = 16 / (int)sizeof(O);
#pragma unroll
  for (int i = 0; i < 32; i += V) {
    const uint4 w = tc::read16(piece_of<ROW_BYTES>(slab, row, first + i / V));
    float f[V];
    widen_word<O, V>(w, f);
#pragma unroll
    for (int k = 0; k < V; ++k) z[i + k] = TIMES ? z[i + k] * f[k] : z[i + k] + f[k];
  }
}

template <ProductKind KIND, typename T, typename O, int BN>
__global__ void __launch_bounds__(kProductThreads, 1) product_kernel(const __grid_constant__ Maps maps,
                                                                     const __grid_constant__ Extents p) {
  using L = Tile<KIND, O, BN>;
  extern __shared__ uint8_t raw[];
  const uint32_t base = (tc::shared_address(raw) + 1023) & ~1023u;
  const uint32_t slabs = base + L::stages * L::stage, bias_at = slabs + L::slabs;
  const uint32_t full = bias_at + kEpilogueWarps * L::bias, empty = full + L::stages * 8;
  const uint32_t summed = empty + L::stages * 8, drained = summed + 16;
  const uint32_t in_there = drained + 16, quiet = in_there + 2 * kEpilogueWarps * 8, where = quiet + 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::stages; ++i) {
      tc::barrier_init(full + i * 8, 1);
      tc::barrier_init(empty + i * 8, 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc::barrier_init(summed + i * 8, 1);
      tc::barrier_init(drained + i * 8, kEpilogueWarps);
    }
    for (int i = 0; i < 2 * kEpilogueWarps; ++i) tc::barrier_init(in_there + i * 8, 1);
    tc::barrier_init(quiet, 1);
    tc::barriers_visible();
  }
  if (warp == 2) tc::tensor_memory_take<L::memory>(where);
  tc::order_before();
  __syncthreads();
  tc::order_after();
  uint32_t memory;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(memory) : "r"(where));

  const int steps = p.steps0 + p.steps1;
  if (warp == 0) {
    if (tc::one_lane()) {
      // ---- operand tiles ----
      int s = 0, issued = 0;       // issued: no more than it takes to go round once
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < p.tiles && ok; tile += gridDim.x) {
        const int m0 = tile / p.tiles_n * kRows, n0 = tile % p.tiles_n * L::columns;
        for (int k = 0; k < steps; ++k) {
          if (!(ok = tc::wait(empty + s * 8, phase ^ 1))) break;
          const uint32_t a = base + s * L::stage, b = a + kOperandA, bar = full + s * 8;
          const bool second = k >= p.steps0;
          const int at = (second ? k - p.steps0 : k) * kDepth;
          if constexpr (KIND == kGatedGrad) tc::arrive_expect(bar, kOperandA + (second ? L::operand_b / 2 : L::operand_b));
          else tc::arrive_expect(bar, L::stage);
          tc::tile_load(a, second ? &maps.a1 : &maps.a0, at, m0, bar);
          if constexpr (KIND == kInputGrad) {
#pragma unroll
            for (int i = 0; i < BN / 64; ++i) tc::tile_load(b + i * kDepth * 128, second ? &maps.b1 : &maps.b0, n0 + i * 64, at, bar);
          } else if constexpr (L::gated) {
            if (KIND == kGatedGrad && second) {
#pragma unroll
              for (int i = 0; i < L::columns / 64; ++i) tc::tile_load(b + i * kDepth * 128, &maps.b2, n0 + i * 64, at, bar);
            } else {
              tc::tile_load(b, &maps.b0, at, n0, bar);
              tc::tile_load(b + L::operand_b / 2, &maps.b1, at, n0, bar);
            }
          } else {
            tc::tile_load(b, &maps.b0, at, n0, bar);
          }
          if (issued < L::stages) ++issued;
          if (++s == L::stages) {
            s = 0;
            phase ^= 1;
          }
        }
      }
      // nothing may be on its way into shared memory when the CTA ends
      for (int i = 0; i < issued; ++i) {
        if (--s < 0) {
          s = L::stages - 1;
          phase ^= 1;
        }
        tc::wait(full + s * 8, phase);
      }
    }
  } else if (warp == 1) {
    if (tc::one_lane()) {
      // ---- products ----
      constexpr uint32_t shape = tc::product_shape<T>(BN, false, KIND == kInputGrad);
      constexpr uint32_t shape_d = tc::product_shape<T>(BN / 2, false, true);
      int s = 0;
      uint32_t phase = 0;
      bool ok = true;
      int it = 0;
      for (int tile = blockIdx.x; tile < p.tiles && ok; tile += gridDim.x, ++it) {
        const uint32_t acc = memory + (it & 1) * L::sums;
        if (!(ok = tc::wait(drained + (it & 1) * 8, (uint32_t)((it >> 1) + 1) & 1))) break;
        tc::order_after();
        for (int k = 0; k < steps; ++k) {
          if (!(ok = tc::wait(full + s * 8, phase))) break;
          tc::order_after();
          const uint32_t a = base + s * L::stage, b = a + kOperandA;
          if (KIND == kGatedGrad && k >= p.steps0) {
#pragma unroll
            for (int j = 0; j < kDepth / 16; ++j)
              tc::product(acc + BN, tc::k_major(a + j * 32), tc::mn_major(b + j * 2048, kDepth * 128), shape_d, k > p.steps0 || j > 0);
          } else {
#pragma unroll
            for (int j = 0; j < kDepth / 16; ++j)
              tc::product(acc, tc::k_major(a + j * 32),
                          KIND == kInputGrad ? tc::mn_major(b + j * 2048, kDepth * 128) : tc::k_major(b + j * 32), shape,
                          k > 0 || j > 0);
          }
          tc::products_arrive(empty + s * 8);
          if (++s == L::stages) {
            s = 0;
            phase ^= 1;
          }
        }
        if (ok) tc::products_arrive(summed + (it & 1) * 8);
      }
      tc::products_arrive(quiet);
      tc::wait(quiet, 0);
    }
  } else if (warp >= 4) {
    // ---- epilogue: a warp has 32 rows and half of the columns ----
    const int e = warp - 4, quarter = warp & 3, half = e >> 2;
    const uint32_t mine = slabs + e * 2 * L::outs * L::slab, bias = bias_at + e * L::bias, there = in_there + e * 16;
    const bool loads = p.has_in && !p.direct;
    const T *bias0 = static_cast<const T *>(p.bias0), *bias1 = static_cast<const T *>(p.bias1);
    int bias_of = -1, set = 0;
    uint32_t in_phase = 0;
    bool ok = true;

    auto row_of = [&](int tile) { return tile / p.tiles_n * kRows + quarter * 32; };
    auto column_of = [&](int tile) { return tile % p.tiles_n * L::columns + half * L::half; };
    // the next (tile, chunk) of this warp that has something inside of the result; tile >= p.tiles: none
    auto next = [&](int &tile, int &c) {
      do {
        if (++c == L::chunks) {
          c = 0;
          tile += gridDim.x;
        }
      } while (tile < p.tiles && (row_of(tile) >= p.rows || column_of(tile) + c * L::chunk >= p.n));
    };
    auto ask = [&](int tile, int c, int into) {
      if (tile >= p.tiles) return;
      tc::arrive_expect(there + into * 8, L::slab);
      tc::tile_load(mine + into * L::outs * L::slab, &maps.in, column_of(tile) + c * L::chunk, row_of(tile), there + into * 8);
    };
    int ask_tile = blockIdx.x, ask_c = -1;
    if (loads) {
      next(ask_tile, ask_c);
      if (lane == 0) ask(ask_tile, ask_c, 0);
    }

    int it = 0;
    for (int tile = blockIdx.x; tile < p.tiles; tile += gridDim.x, ++it) {
      const int m0 = row_of(tile), n0 = column_of(tile);
      if (n0 != bias_of) {
        __syncwarp();
        for (int i = lane; i < L::half; i += 32) {
          const bool in = n0 + i < p.n;
          const float v = in && bias0 ? wide(bias0[n0 + i]) : 0.f;
          asm volatile("st.shared.f32 [%0], %1;" ::"r"(bias + i * 4), "f"(v) : "memory");
          if constexpr (L::gated) {
            const float w = in && bias1 ? wide(bias1[n0 + i]) : 0.f;
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(bias + (L::half + i) * 4), "f"(w) : "memory");
          }
        }
        __syncwarp();
        bias_of = n0;
      }
      if (ok) ok = __all_sync(0xffffffffu, tc::wait(summed + (it & 1) * 8, (uint32_t)(it >> 1) & 1));
      tc::order_after();
      const uint32_t acc = memory + ((uint32_t)quarter << 21) + (it & 1) * L::sums + half * L::half;
      for (int c = 0; c < L::chunks; ++c) {
        const int col = n0 + c * L::chunk;
        if (m0 >= p.rows || col >= p.n) continue;
        const uint32_t slab = mine + set * L::outs * L::slab;
        if (loads) {
          if (ok) ok = __all_sync(0xffffffffu, tc::wait(there + set * 8, (in_phase >> set) & 1));
          in_phase ^= 1u << set;
          next(ask_tile, ask_c);
          if (lane == 0) {
            tc::stores_read<0>();
            if (ok) ask(ask_tile, ask_c, set ^ 1);
          }
        } else if (!p.direct) {
          if (lane == 0) tc::stores_read<1>();
          __syncwarp();
        }
        const bool row_in = m0 + lane < p.rows;
#pragma unroll
        for (int sub = 0; sub < L::chunk; sub += 32) {
          const int first = sub * (int)sizeof(O) / 16, off = c * L::chunk + sub;
          float z[32];
          if constexpr (L::gated) {
            float u[32];
            tc::tensor_load(z, acc + off);
            tc::tensor_load(u, acc + BN / 2 + off);
            if constexpr (KIND == kGatedGrad) {
              float d[32];
              tc::tensor_load(d, acc + BN + off);
              tc::tensor_loads_done(z);
              tc::tensor_loads_done(u);
              tc::tensor_loads_done(d);
              add_bias(z, bias + off * 4);
              add_bias(u, bias + (L::half + off) * 4);
              gate_all(z, u, d, p.act);
              if (!ok) z[0] = u[0] = d[0] = __int_as_float(0x7fffffff);
              put<O, L::row_bytes>(z, slab, lane, first);
              put<O, L::row_bytes>(d, slab + L::slab, lane, first);
              put<O, L::row_bytes>(u, slab + 2 * L::slab, lane, first);
              continue;
            }
            tc::tensor_loads_done(z);
            tc::tensor_loads_done(u);
            add_bias(z, bias + off * 4);
            add_bias(u, bias + (L::half + off) * 4);
            activate_all(z, p.act);
#pragma unroll
            for (int i = 0; i < 32; ++i) z[i] *= u[i];
          } else {
            tc::tensor_load(z, acc + off);
            tc::tensor_loads_done(z);
            if constexpr (KIND != kInputGrad) add_bias(z, bias + off * 4);
            if constexpr (KIND == kLinear) activate_all(z, p.act);
            if constexpr (KIND == kSlope) slope_all(z, p.act);
            if (loads) combine<O, L::row_bytes, KIND == kSlope>(z, slab, lane, first);
          }
          if (!ok) z[0] = __int_as_float(0x7fffffff);
          if (!p.direct) {
            put<O, L::row_bytes>(z, slab, lane, first);
          } else if (row_in) {
            const O *in = static_cast<const O *>(p.in) + (m0 + lane) * p.in_pitch + col + sub;
            O *out = static_cast<O *>(p.out) + (m0 + lane) * p.out_pitch + col + sub;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (col + sub + i < p.n) out[i] = narrow<O>(p.has_in ? z[i] + wide(in[i]) : z[i]);
          }
        }
        if (!p.direct) {
          tc::shared_to_async();
          __syncwarp();
          if (lane == 0) {
#pragma unroll
            for (int o = 0; o < L::outs; ++o) tc::tile_store(&maps.out[o], col, m0, slab + o * L::slab);
            tc::stores_asked();
          }
          set ^= 1;
        }
      }
      tc::order_before();
      __syncwarp();
      if (lane == 0) tc::arrive(drained + (it & 1) * 8);
    }
    if (lane == 0) tc::stores_done();
  }
  tc::order_before();
  __syncthreads();
  if (warp == 2) {
    tc::order_after();
    tc::tensor_memory_give<L::memory>(memory);
  }
}

template <ProductKind KIND, typename T, typename O, int BN> cudaError_t launch_tiles(const ProductArgs &a, cudaStream_t s) {
  using L = Tile<KIND, O, BN>;
  const int in_type = sizeof(O) == 4 ? DFA3D_DTYPE_F32 : a.dtype;
  Maps m{};
  Extents p{};
  const int per16 = 16 / (int)sizeof(O);
  auto fits = [&](const void *q, long long pitch) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0 && pitch % per16 == 0; };
  p.direct = !fits(a.out[0], a.out_pitch) || (a.in.data && !fits(a.in.data, a.in.pitch));
  if (p.direct && KIND != kLinear && KIND != kInputGrad) return cudaErrorInvalidValue;      // their results are workspaces
  bool ok = describe_matrix(m.a0, a.dtype, a.a0.data, a.rows, a.k0, a.a0.pitch, kDepth, kRows);
  if constexpr (KIND == kInputGrad) {
    ok = ok && describe_matrix(m.b0, a.dtype, a.b0.data, a.k0, a.n, a.b0.pitch, 64, kDepth);
    if (a.k1 > 0)
      ok = ok && describe_matrix(m.a1, a.dtype, a.a1.data, a.rows, a.k1, a.a1.pitch, kDepth, kRows) &&
           describe_matrix(m.b1, a.dtype, a.b1.data, a.k1, a.n, a.b1.pitch, 64, kDepth);
  } else {
    ok = ok && describe_matrix(m.b0, a.dtype, a.b0.data, a.n, a.k0, a.b0.pitch, kDepth, L::gated ? BN / 2 : BN);
    if constexpr (L::gated) ok = ok && describe_matrix(m.b1, a.dtype, a.b1.data, a.n, a.k0, a.b1.pitch, kDepth, BN / 2);
    if constexpr (KIND == kGatedGrad)
      ok = ok && describe_matrix(m.a1, a.dtype, a.a1.data, a.rows, a.k1, a.a1.pitch, kDepth, kRows) &&
           describe_matrix(m.b2, a.dtype, a.b2.data, a.k1, a.n, a.b2.pitch, 64, kDepth);
  }
  if (!p.direct) {
    if (a.in.data) ok = ok && describe_matrix(m.in, in_type, a.in.data, a.rows, a.n, a.in.pitch, L::chunk, 32);
    for (int o = 0; o < L::outs; ++o) ok = ok && describe_matrix(m.out[o], in_type, a.out[o], a.rows, a.n, a.out_pitch, L::chunk, 32);
  }
  if (!ok) return cudaErrorInvalidValue;
  p.rows = (int)a.rows;
  p.n = a.n;
  p.steps0 = (a.k0 + kDepth - 1) / kDepth;
  p.steps1 = (a.k1 + kDepth - 1) / kDepth;
  p.tiles_n = (a.n + L::columns - 1) / L::columns;
  p.tiles = (int)((a.rows + kRows - 1) / kRows) * p.tiles_n;
  p.act = a.act;
  p.has_in = a.in.data != nullptr;
  p.bias0 = a.bias0;
  p.bias1 = a.bias1;
  p.in = a.in.data;
  p.in_pitch = a.in.pitch;
  p.out = a.out[0];
  p.out_pitch = a.out_pitch;
  constexpr auto kernel = &product_kernel<KIND, T, O, BN>;
  cudaError_t rc = allow_shared<kernel>(L::bytes);
  if (rc != cudaSuccess) return rc;
  const int grid = p.tiles < sm_count() ? p.tiles : sm_count();
  kernel<<<grid, kProductThreads, L::bytes, s>>>(m, p);
  return cudaGetLastError();
}

// Wide tiles read each operand fewer times; narrow ones give a small product to more SMs.
int tile_width(long long rows, int n, int widest, int narrowest) {
  for (int w = widest; w > narrowest; w /= 2)
    if (n > w / 2 && (rows + kRows - 1) / kRows * ((n + w - 1) / w) >= sm_count()) return w;
  return narrowest;
}

template <typename T> cudaError_t launch_typed(const ProductArgs &a, cudaStream_t s) {
  switch (a.kind) {
    case kLinear: {
      const int w = tile_width(a.rows, a.n, 256, 64);
      if (a.wide_out)
        return w == 256   ? launch_tiles<kLinear, T, float, 256>(a, s)
               : w == 128 ? launch_tiles<kLinear, T, float, 128>(a, s)
                          : launch_tiles<kLinear, T, float, 64>(a, s);
      return w == 256   ? launch_tiles<kLinear, T, T, 256>(a, s)
             : w == 128 ? launch_tiles<kLinear, T, T, 128>(a, s)
                        : launch_tiles<kLinear, T, T, 64>(a, s);
    }
    case kSlope:
      return tile_width(a.rows, a.n, 256, 64) == 64 ? launch_tiles<kSlope, T, T, 64>(a, s) : launch_tiles<kSlope, T, T, 128>(a, s);
    case kGated:
      return tile_width(a.rows, a.n, 128, 64) == 128 ? launch_tiles<kGated, T, T, 256>(a, s) : launch_tiles<kGated, T, T, 128>(a, s);
    case kGatedGrad: return launch_tiles<kGatedGrad, T, T, 128>(a, s);
    case kInputGrad: {
      const int w = tile_width(a.rows, a.n, 256, 64);
      return w == 256   ? launch_tiles<kInputGrad, T, T, 256>(a, s)
             : w == 128 ? launch_tiles<kInputGrad, T, T, 128>(a, s)
                        : launch_tiles<kInputGrad, T, T, 64>(a, s);
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
