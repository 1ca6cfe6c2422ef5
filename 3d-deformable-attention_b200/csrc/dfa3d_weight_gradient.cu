// Weight and bias gradients of a matrix product: out = g^T x, summed over tens of thousands of rows into a result of a few hundred
// squared.  Each CTA sums one tile of 128 x BN over its share of the rows on the tensor cores -- both operands as they lie, the summed
// axis running over their rows -- and leaves 32-bit partial sums; a second kernel adds the shares up in a fixed order and rounds once.
// The bias gradient is one more operand of the product, a column of ones.
#include "dfa3d_common.cuh"
#include "dfa3d_product.h"
#include "dfa3d_rowvec.cuh"
#include "dfa3d_tcgen05.cuh"
#include "dfa3d_tensor_map.h"

namespace dfa3d {
namespace {

constexpr int kTileP = 128, kDepth = 64, kOnes = 16;          // columns of ones: the narrowest product
constexpr int kThreads8 = 384, kOperandA = kTileP * kDepth * 2;

struct Problem {
  CUtensorMap g, x;
  void *out, *bias;
  int p, q, tiles_q, first;      // first: its first tile among those of all problems
};
struct Problems {
  Problem of[kMaxWeightProblems];
  int count, tiles, shares, steps;      // steps of kDepth rows
  float *partial;                       // [share][tile][BN columns and the bias][128 rows]
};

template <int BN> struct Grad {
  static constexpr int operand_b = BN * kDepth * 2, stage = kOperandA + operand_b, stages = 4;
  static constexpr int ones = kOnes * kDepth * 2;
  static constexpr int memory = BN == 256 ? 512 : BN == 128 ? 256 : 128;
  static constexpr int bytes = 1024 + stages * stage + ones + (2 * stages + 2) * 8 + 16;
  static constexpr int columns = BN + 1;
};

__device__ __forceinline__ int problem_of(const Problems &w, int tile) {
  int i = 0;
  while (i + 1 < w.count && tile >= w.of[i + 1].first) ++i;
  return i;
}

template <typename T, int BN>
__global__ void __launch_bounds__(kThreads8, 1) weight_gradient_kernel(const __grid_constant__ Problems w) {
  using L = Grad<BN>;
  extern __shared__ uint8_t raw[];
  const uint32_t base = (tc::shared_address(raw) + 1023) & ~1023u;
  const uint32_t ones = base + L::stages * L::stage, full = ones + L::ones, empty = full + L::stages * 8, done = empty + L::stages * 8,
                 quiet = done + 8, where = quiet + 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = blockIdx.x % w.tiles, share = blockIdx.x / w.tiles;
  const Problem &pr = w.of[problem_of(w, tile)];
  const int p0 = (tile - pr.first) / pr.tiles_q * kTileP, q0 = (tile - pr.first) % pr.tiles_q * BN;
  const bool bias = pr.bias && q0 == 0;
  const int begin = (int)((long long)share * w.steps / w.shares), end = (int)((long long)(share + 1) * w.steps / w.shares);

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::stages; ++i) {
      tc::barrier_init(full + i * 8, 1);
      tc::barrier_init(empty + i * 8, 1);
    }
    tc::barrier_init(done, 1);
    tc::barrier_init(quiet, 1);
    tc::barriers_visible();
  }
  if (warp == 2) tc::tensor_memory_take<L::memory, false>(where);
  if (warp >= 4) {      // the same whatever the layout
    const T one = narrow<T>(1.f);
    const uint32_t two = (uint32_t)reinterpret_cast<const uint16_t &>(one) * 0x10001u;
    for (int i = threadIdx.x - 128; i < L::ones / 16; i += 256) tc::write16(ones + i * 16, make_uint4(two, two, two, two));
    tc::shared_to_async();
  }
  tc::let_next_kernel_begin();
  tc::wait_for_last_kernel();
  tc::order_before();
  __syncthreads();
  tc::order_after();
  uint32_t memory;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(memory) : "r"(where));

  if (warp == 0) {
    if (tc::one_lane()) {
      int s = 0, issued = 0;
      uint32_t phase = 0;
      for (int k = begin; k < end; ++k) {
        if (!tc::wait(empty + s * 8, phase ^ 1)) break;
        const uint32_t a = base + s * L::stage, b = a + kOperandA, bar = full + s * 8;
        tc::arrive_expect(bar, L::stage);
#pragma unroll
        for (int i = 0; i < kTileP / 64; ++i) tc::tile_load(a + i * kDepth * 128, &pr.g, p0 + i * 64, k * kDepth, bar);
#pragma unroll
        for (int i = 0; i < BN / 64; ++i) tc::tile_load(b + i * kDepth * 128, &pr.x, q0 + i * 64, k * kDepth, bar);
        if (issued < L::stages) ++issued;
        if (++s == L::stages) {
          s = 0;
          phase ^= 1;
        }
      }
      for (int i = 0; i < issued; ++i) {      // nothing may be on its way into shared memory when the CTA ends
        if (--s < 0) {
          s = L::stages - 1;
          phase ^= 1;
        }
        tc::wait(full + s * 8, phase);
      }
    }
  } else if (warp == 1) {
    if (tc::one_lane()) {
      constexpr uint32_t shape = tc::product_shape<T>(kTileP, BN, true, true), shape_ones = tc::product_shape<T>(kTileP, kOnes, true, false);
      int s = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int k = begin; k < end; ++k) {
        if (!(ok = tc::wait(full + s * 8, phase))) break;
        tc::order_after();
        const uint32_t a = base + s * L::stage, b = a + kOperandA;
#pragma unroll
        for (int j = 0; j < kDepth / 16; ++j) {
          const uint64_t da = tc::mn_major(a + j * 2048, kDepth * 128);
          tc::product<false>(memory, da, tc::mn_major(b + j * 2048, kDepth * 128), shape, k > begin || j > 0);
          if (bias) tc::product<false>(memory + BN, da, tc::k_major(ones), shape_ones, k > begin || j > 0);
        }
        tc::products_arrive<false>(empty + s * 8);
        if (++s == L::stages) {
          s = 0;
          phase ^= 1;
        }
      }
      if (ok) tc::products_arrive<false>(done);
      tc::products_arrive<false>(quiet);
      tc::wait(quiet, 0);
    }
  } else if (warp >= 4) {
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const bool ok = __all_sync(0xffffffffu, tc::wait(done, 0));
    tc::order_after();
    const uint32_t acc = memory + ((uint32_t)quarter << 21);
    float *out = w.partial + ((long long)share * w.tiles + tile) * L::columns * kTileP + quarter * 32 + lane;
    const float lost = __int_as_float(0x7fffffff);
    for (int c = half * (BN / 2); c < (half + 1) * (BN / 2); c += 32) {
      if (q0 + c >= pr.q) break;
      float v[32];
      tc::tensor_load(v, acc + c);
      tc::tensor_loads_done(v);
#pragma unroll
      for (int i = 0; i < 32; ++i) out[(c + i) * kTileP] = ok ? v[i] : lost;
    }
    if (bias && half == 0) {
      float v[32];
      tc::tensor_load(v, acc + BN);      // 16 columns of it are the bias gradient
      tc::tensor_loads_done(v);
      out[BN * kTileP] = ok ? v[0] : lost;
    }
  }
  tc::order_before();
  __syncthreads();
  if (warp == 2) {
    tc::order_after();
    tc::tensor_memory_give<L::memory, false>(memory);
  }
}

// A CTA adds up the shares of eight columns of a tile (a thread four rows of one), turns them around in shared memory and writes rows
// of the result.  Few columns, so that even one tile has many CTAs: the shares are read one after the other, and what there is to
// read is little (20 MB at most) but far away.
constexpr int kSumColumns = 8;
template <typename T, int BN> __global__ void __launch_bounds__(256) weight_gradient_sum_kernel(const __grid_constant__ Problems w) {
  __shared__ float turned[kSumColumns][kTileP + 1];
  tc::let_next_kernel_begin();
  tc::wait_for_last_kernel();
  const int tile = blockIdx.x / (BN / kSumColumns), c0 = blockIdx.x % (BN / kSumColumns) * kSumColumns;
  const Problem &pr = w.of[problem_of(w, tile)];
  const int p0 = (tile - pr.first) / pr.tiles_q * kTileP, q0 = (tile - pr.first) % pr.tiles_q * BN + c0;
  if (q0 >= pr.q) return;
  const long long step = (long long)w.tiles * Grad<BN>::columns * kTileP;
  const float *src = w.partial + (long long)tile * Grad<BN>::columns * kTileP;
  const int at = threadIdx.x * 4;      // of 8 x 128
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int s = 0; s < w.shares; ++s) {
    const float4 v = __ldcs(reinterpret_cast<const float4 *>(src + s * step + c0 * kTileP + at));
    sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
  }
  float *to = &turned[at / kTileP][at % kTileP];
  to[0] = sum.x; to[1] = sum.y; to[2] = sum.z; to[3] = sum.w;
  if (pr.bias && q0 == 0 && threadIdx.x < kTileP && p0 + threadIdx.x < pr.p) {
    float total = 0.f;
#pragma unroll 8
    for (int s = 0; s < w.shares; ++s) total += src[s * step + BN * kTileP + threadIdx.x];
    static_cast<T *>(pr.bias)[p0 + threadIdx.x] = narrow<T>(total);
  }
  __syncthreads();
  const int c = threadIdx.x % kSumColumns;
  for (int r = threadIdx.x / kSumColumns; r < kTileP; r += 256 / kSumColumns)
    if (p0 + r < pr.p && q0 + c < pr.q) static_cast<T *>(pr.out)[(long long)(p0 + r) * pr.q + q0 + c] = narrow<T>(turned[c][r]);
}

int width_for(const WeightProblem *w, int count) {
  int q = 0;
  for (int i = 0; i < count; ++i) q = w[i].q > q ? w[i].q : q;
  return q > 128 ? 256 : q > 64 ? 128 : 64;
}
int tiles_for(const WeightProblem *w, int count, int width) {
  int n = 0;
  for (int i = 0; i < count; ++i) n += (w[i].p + kTileP - 1) / kTileP * ((w[i].q + width - 1) / width);
  return n;
}
// As many shares of the rows as SMs allow in one wave, none without rows.
int shares_for(long long rows, int tiles) {
  const long long steps = (rows + kDepth - 1) / kDepth, s = tiles < sm_count() ? sm_count() / tiles : 1;
  return (int)(s < steps ? s : steps);
}

template <typename T, int BN>
cudaError_t launch_shares(int dtype, long long rows, const WeightProblem *w, int count, void *workspace, cudaStream_t s) {
  using L = Grad<BN>;
  Problems q{};
  q.count = count;
  for (int i = 0; i < count; ++i) {
    Problem &o = q.of[i];
    o.out = w[i].out;
    o.bias = w[i].bias;
    o.p = w[i].p;
    o.q = w[i].q;
    o.tiles_q = (w[i].q + BN - 1) / BN;
    o.first = q.tiles;
    q.tiles += (w[i].p + kTileP - 1) / kTileP * o.tiles_q;
    if (!describe_matrix(o.g, dtype, w[i].g.data, rows, w[i].p, w[i].g.pitch, 64, kDepth) ||
        !describe_matrix(o.x, dtype, w[i].x.data, rows, w[i].q, w[i].x.pitch, 64, kDepth))
      return cudaErrorInvalidValue;
  }
  q.shares = shares_for(rows, q.tiles);
  q.steps = (int)((rows + kDepth - 1) / kDepth);
  q.partial = static_cast<float *>(workspace);
  constexpr auto kernel = &weight_gradient_kernel<T, BN>;
  cudaError_t rc = allow_shared<kernel>(L::bytes);
  if (rc != cudaSuccess) return rc;
  rc = launch_after(kernel, q.tiles * q.shares, kThreads8, L::bytes, s, q);
  if (rc != cudaSuccess) return rc;
  return launch_after(&weight_gradient_sum_kernel<T, BN>, q.tiles * (BN / kSumColumns), 256, 0, s, q);
}

template <typename T>
cudaError_t launch_typed(int dtype, long long rows, const WeightProblem *w, int count, void *workspace, cudaStream_t s) {
  const int width = width_for(w, count);
  return width == 256   ? launch_shares<T, 256>(dtype, rows, w, count, workspace, s)
         : width == 128 ? launch_shares<T, 128>(dtype, rows, w, count, workspace, s)
                        : launch_shares<T, 64>(dtype, rows, w, count, workspace, s);
}

}  // namespace

long long weight_gradient_workspace(long long rows, const WeightProblem *w, int count) {
  const int width = width_for(w, count), tiles = tiles_for(w, count, width);
  return (long long)shares_for(rows, tiles) * tiles * (width + 1) * kTileP * 4;
}

cudaError_t launch_weight_gradient(int dtype, long long rows, const WeightProblem *w, int count, void *workspace, cudaStream_t s) {
  if (const cudaError_t rc = bind_context()) return rc;
  return dtype == DFA3D_DTYPE_F16 ? launch_typed<__half>(dtype, rows, w, count, workspace, s)
                                  : launch_typed<__nv_bfloat16>(dtype, rows, w, count, workspace, s);
}

}  // namespace dfa3d
