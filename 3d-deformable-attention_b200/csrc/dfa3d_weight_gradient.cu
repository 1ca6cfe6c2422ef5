// Weight and bias gradients of a matrix product: out = g^T x, summed over tens of thousands of rows into a result of a few hundred
// squared.  Each pair of CTAs sums one tile of 256 x BN over its share of the rows on the tensor cores -- both operands as they lie, the
// summed axis running over their rows -- and leaves 32-bit partial sums; a second kernel adds the shares up in a fixed order and rounds
// once.  The bias gradient is one more operand of the product, columns of ones.  A step of 64 rows is summed in 512 cycles and brings
// 32 KB into each SM: the way from L2 (about 45 bytes a cycle and SM while all read) binds, and without pairs it would be 48 KB.
//
// Measured with the sum kernel on calls that follow one another, bf16: 40 000 x 512 by 256 22.4 us (61 MB, 9.4 us at 6.5 TB/s; the
// partial sums, 19 MB written and read again, are most of the rest), the three gradients of a gated block 256 -> 512 -> 256 40, of 80 000
// rows 256 -> 1024 -> 256 112.  One launch for all gradients of a block: a product of its own has too few tiles for 74 pairs, and
// more shares instead would leave more partial sums behind.
#include "dfa3d_common.cuh"
#include "dfa3d_product.h"
#include "dfa3d_rowvec.cuh"
#include "dfa3d_tcgen05.cuh"
#include "dfa3d_tensor_map.h"

namespace dfa3d {
namespace {

constexpr int kTileP = 128, kDepth = 64;          // of a CTA; a pair has twice as many
constexpr int kOnes = 16;                         // columns of ones of a pair: the narrowest product
constexpr int kThreads8 = 384, kOperandA = kTileP * kDepth * 2;

struct Problem {
  CUtensorMap g, x;
  void *out, *bias;
  int p, q, tiles_q, first;      // first: its first tile (of a pair) among those of all problems
};
struct Problems {
  Problem of[kMaxWeightProblems];
  int count, tiles, shares, steps;      // steps of kDepth rows
  float *partial;                       // [share][tile][CTA of the pair][BN columns and the bias][128 rows]
};

template <int BN> struct Grad {
  static constexpr int half = BN / 2, box = half < 64 ? half : 64;               // columns of x of a CTA, of a tiled copy
  static constexpr int operand_b = half * kDepth * 2, stage = kOperandA + operand_b;
  static constexpr int stages = 6;
  static constexpr int ones = kOnes / 2 * kDepth * 2;
  static constexpr int memory = BN == 256 ? 512 : BN == 128 ? 256 : 128;
  static constexpr int bytes = stages * stage + ones + (2 * stages + 2) * 8 + 16;
  static constexpr int columns = BN + 1;
  static_assert(one_an_sm(bytes) && bytes <= 227 * 1024, "layout");
};

__device__ __forceinline__ int problem_of(const Problems &w, int tile) {
  int i = 0;
  while (i + 1 < w.count && tile >= w.of[i + 1].first) ++i;
  return i;
}

template <typename T, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads8, 1) weight_gradient_kernel(const __grid_constant__ Problems w) {
  using L = Grad<BN>;
  extern __shared__ __align__(1024) uint8_t raw[];
  const uint32_t base = tc::shared_address(raw);
  const uint32_t ones = base + L::stages * L::stage, full = ones + L::ones, empty = full + L::stages * 8, done = empty + L::stages * 8,
                 quiet = done + 8, where = quiet + 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = tc::rank_in_pair();
  const int tile = (int)(blockIdx.x >> 1) % w.tiles, share = (int)(blockIdx.x >> 1) / w.tiles;
  const Problem &pr = w.of[problem_of(w, tile)];
  const int p0 = ((tile - pr.first) / pr.tiles_q * 2 + (int)rank) * kTileP, q0 = (tile - pr.first) % pr.tiles_q * BN;
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
  if (warp == 2) tc::tensor_memory_take<L::memory>(where);
  if (warp >= 4) {      // the same whatever the layout
    const T one = narrow<T>(1.f);
    const uint32_t two = (uint32_t)reinterpret_cast<const uint16_t &>(one) * 0x10001u;
    for (int i = threadIdx.x - 128; i < L::ones / 16; i += 256) tc::write16(ones + i * 16, make_uint4(two, two, two, two));
    tc::shared_to_async();
  }
  tc::let_next_kernel_begin();
  tc::wait_for_last_kernel();
  tc::order_before();
  __syncwarp();
  tc::pair_sync();
  tc::order_after();
  uint32_t memory;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(memory) : "r"(where));

  if (warp == 0) {
    if (tc::one_lane()) {      // this CTA's operands; the first one's barriers count those of both
      const uint32_t first_full = tc::address_in(full, 0);
      int s = 0, issued = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int k = begin; k < end; ++k) {
        if (!(ok = tc::wait(empty + s * 8, phase ^ 1))) break;
        const uint32_t a = base + s * L::stage, b = a + kOperandA, bar = first_full + s * 8;
        if (rank == 0) tc::arrive_expect(full + s * 8, 2 * L::stage);
#pragma unroll
        for (int i = 0; i < kTileP / 64; ++i) tc::tile_load_pair(a + i * kDepth * 128, &pr.g, p0 + i * 64, k * kDepth, bar);
#pragma unroll
        for (int i = 0; i < L::half / L::box; ++i)
          tc::tile_load_pair(b + i * kDepth * 128, &pr.x, q0 + (int)rank * L::half + i * L::box, k * kDepth, bar);
        if (issued < L::stages) ++issued;
        if (++s == L::stages) {
          s = 0;
          phase ^= 1;
        }
      }
      for (int i = 0; i < issued && rank == 0; ++i) {      // nothing may be on its way into shared memory when the CTAs end
        if (--s < 0) {
          s = L::stages - 1;
          phase ^= 1;
        }
        tc::wait(full + s * 8, phase);
      }
      if (!ok) __nanosleep(1000000);
    }
  } else if (warp == 1) {
    if (rank == 0) {
      constexpr uint32_t shape = tc::product_shape<T>(2 * kTileP, BN, true, true), shape_ones = tc::product_shape<T>(2 * kTileP, kOnes, true, false);
      int s = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int k = begin; k < end; ++k) {
        if (!(ok = tc::wait_warp(full + s * 8, phase))) break;
        tc::order_after();
        const uint64_t a = tc::mn_major(base + s * L::stage, kDepth * 128);
        const uint32_t at_b = base + s * L::stage + kOperandA;
        const uint64_t b = L::half < 64 ? tc::mn_major_narrow(at_b) : tc::mn_major(at_b, kDepth * 128);
        constexpr int step_b = (L::half < 64 ? 1024 : 2048) / 16;
        if (tc::one_lane()) {
#pragma unroll
          for (int j = 0; j < kDepth / 16; ++j) {
            tc::product(memory, a + j * (2048 / 16), b + j * step_b, shape, k > begin || j > 0);
            if (bias) tc::product(memory + BN, a + j * (2048 / 16), tc::k_major(ones), shape_ones, k > begin || j > 0);
          }
          tc::products_arrive(empty + s * 8);
        }
        __syncwarp();
        if (++s == L::stages) {
          s = 0;
          phase ^= 1;
        }
      }
      if (tc::one_lane()) {
        if (ok) tc::products_arrive(done);
        tc::products_arrive(quiet);
      }
      __syncwarp();
    }
    tc::wait_warp(quiet, 0);
  } else if (warp >= 4) {
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const bool ok = __all_sync(0xffffffffu, tc::wait(done, 0));
    tc::order_after();
    const uint32_t acc = memory + ((uint32_t)quarter << 21);
    float *out = w.partial + (((long long)share * w.tiles + tile) * 2 + rank) * L::columns * kTileP + quarter * 32 + lane;
    const float lost = __int_as_float(0x7fffffff);
    if (p0 < pr.p) {
      for (int c = half * (BN / 2); c < (half + 1) * (BN / 2); c += 32) {
        if (q0 + c >= pr.q) break;
        float v[32];
        tc::tensor_load(v, acc + c);
        tc::tensor_loads_done(v);
#pragma unroll
        for (int i = 0; i < 32; ++i) out[(c + i) * kTileP] = ok ? v[i] : lost;
      }
      if (bias && half == 0) {
        float v[16];
        tc::tensor_load(v, acc + BN);      // any of them is the bias gradient
        tc::tensor_loads_done(v);
        out[BN * kTileP] = ok ? v[0] : lost;
      }
    }
  }
  tc::order_before();
  __syncwarp();
  tc::pair_sync();
  if (warp == 2) {
    tc::order_after();
    tc::tensor_memory_give<L::memory>(memory);
  }
}

// A CTA adds up the shares of four columns of a CTA's tile -- a thread four rows of one column of every other share --, turns them
// around in shared memory and writes rows of the result.  So few, that even one tile has many CTAs and a thread few loads one after
// the other: what there is to read is little (20 MB where the shares fill one wave of pairs; of a result with more tiles
// than pairs one share, 32 bits an element, 67 MB for 4096 x 4096) but far away.
constexpr int kSumColumns = 4;
template <typename T, int BN> __global__ void __launch_bounds__(256) weight_gradient_sum_kernel(const __grid_constant__ Problems w) {
  __shared__ float4 other[kSumColumns * kTileP / 4];
  __shared__ float other_bias[kTileP];
  __shared__ float turned[kSumColumns][kTileP + 1];
  tc::let_next_kernel_begin();
  tc::wait_for_last_kernel();
  const int half_tile = blockIdx.x / (BN / kSumColumns), tile = half_tile >> 1, c0 = blockIdx.x % (BN / kSumColumns) * kSumColumns;
  const Problem &pr = w.of[problem_of(w, tile)];
  const int p0 = ((tile - pr.first) / pr.tiles_q * 2 + (half_tile & 1)) * kTileP, q0 = (tile - pr.first) % pr.tiles_q * BN + c0;
  if (q0 >= pr.q || p0 >= pr.p) return;
  const long long step = 2LL * w.tiles * Grad<BN>::columns * kTileP;
  const float *src = w.partial + (long long)half_tile * Grad<BN>::columns * kTileP;
  const int odd = threadIdx.x >> 7, at = (threadIdx.x & 127) * 4;      // of 4 x 128
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int s = odd; s < w.shares; s += 2) {
    const float4 v = __ldcs(reinterpret_cast<const float4 *>(src + s * step + c0 * kTileP + at));
    sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
  }
  const bool bias = pr.bias && q0 == 0;
  float total = 0.f;
  if (bias) {
#pragma unroll 8
    for (int s = odd; s < w.shares; s += 2) total += src[s * step + BN * kTileP + (threadIdx.x & 127)];
  }
  if (odd) {
    other[threadIdx.x & 127] = sum;
    other_bias[threadIdx.x & 127] = total;
  }
  __syncthreads();
  if (!odd) {
    const float4 v = other[threadIdx.x];
    float *to = &turned[at / kTileP][at % kTileP];
    to[0] = sum.x + v.x; to[1] = sum.y + v.y; to[2] = sum.z + v.z; to[3] = sum.w + v.w;
    if (bias && p0 + threadIdx.x < pr.p)
      static_cast<T *>(pr.bias)[p0 + threadIdx.x] = narrow<T>(total + other_bias[threadIdx.x]);
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
  for (int i = 0; i < count; ++i) n += (w[i].p + 2 * kTileP - 1) / (2 * kTileP) * ((w[i].q + width - 1) / width);
  return n;
}
// As many shares of the rows as pairs of SMs allow in one wave, of four steps at least (what a share leaves behind takes about as long
// to write and read back as four steps do), none without rows.
int shares_for(long long rows, int tiles) {
  const long long steps = (rows + kDepth - 1) / kDepth, pairs = sm_count() / 2, most = tiles < pairs ? pairs / tiles : 1;
  const long long s = (steps + 3) / 4;
  return (int)(s < most ? s : most);
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
    q.tiles += (w[i].p + 2 * kTileP - 1) / (2 * kTileP) * o.tiles_q;
    if (!describe_matrix(o.g, dtype, w[i].g.data, rows, w[i].p, w[i].g.pitch, 64, kDepth) ||
        !describe_matrix(o.x, dtype, w[i].x.data, rows, w[i].q, w[i].x.pitch, L::box, kDepth))
      return cudaErrorInvalidValue;
  }
  q.shares = shares_for(rows, q.tiles);
  q.steps = (int)((rows + kDepth - 1) / kDepth);
  q.partial = static_cast<float *>(workspace);
  constexpr auto kernel = &weight_gradient_kernel<T, BN>;
  cudaError_t rc = allow_shared<kernel>(L::bytes);
  if (rc != cudaSuccess) return rc;
  rc = launch_after(kernel, 2 * q.tiles * q.shares, kThreads8, L::bytes, s, q);
  if (rc != cudaSuccess) return rc;
  return launch_after(&weight_gradient_sum_kernel<T, BN>, 2 * q.tiles * (BN / kSumColumns), 256, 0, s, q);
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
  return (long long)shares_for(rows, tiles) * tiles * 2 * (width + 1) * kTileP * 4;
}

cudaError_t launch_weight_gradient(int dtype, long long rows, const WeightProblem *w, int count, void *workspace, cudaStream_t s) {
  if (const cudaError_t rc = bind_context()) return rc;
  return dtype == DFA3D_DTYPE_F16 ? launch_typed<__half>(dtype, rows, w, count, workspace, s)
                                  : launch_typed<__nv_bfloat16>(dtype, rows, w, count, workspace, s);
}

}  // namespace dfa3d
