// Internal: matrix products over the rows of a feed-forward block on the tensor cores (dfa3d_product.cu, dfa3d_weight_gradient.cu)
// and the 8-bit checkpoints of their inputs (dfa3d_checkpoint8.cu).  Matrices are row-major, 16-bit; operands of a product begin on a
// 16-byte boundary and have a row pitch of a multiple of eight elements, results and residuals may lie anywhere.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace dfa3d {

struct Operand {
  const void *data = nullptr;
  long long pitch = 0;      // elements
};

enum ProductKind {
  kLinear,        // out = act(a0 b0^T + bias0) [+ in]                                        b0 (n, k0)
  kSlope,         // out = in * act'(a0 b0^T + bias0)
  kGated,         // out = act(a0 b0^T + bias0) * (a0 b1^T + bias1)                           b0, b1 (n, k0)
  kGatedGrad,     // with gate, up as above and d = a1 b2: out = d up act'(gate), d act(gate), act(gate) up      b2 (k1, n)
  kInputGrad,     // out = a0 b0 [+ a1 b1] [+ in]                                             b0 (k0, n), b1 (k1, n)
};

struct ProductArgs {
  ProductKind kind;
  int dtype;                // DFA3D_DTYPE_BF16 or _F16
  bool wide = false;        // kLinear: in and out are fp32; kSlope: in is
  long long rows = 0;
  int n = 0, k0 = 0, k1 = 0;
  Operand a0, a1, b0, b1, b2, in;
  const void *bias0 = nullptr, *bias1 = nullptr;
  int act = 0;
  void *out[3] = {nullptr, nullptr, nullptr};
  long long out_pitch = 0;
};
cudaError_t launch_product(const ProductArgs &a, cudaStream_t s);

// The whole gated block with one kernel (dfa3d_gated_block.cu): a0 = x, b0, b1 = gate and up (hidden, k0), b2 = down (n, hidden), in =
// residual, out[0]; bias2 of the result.  Where it is the faster one.
bool gated_block_covers(const ProductArgs &a, int hidden);
cudaError_t launch_gated_block(const ProductArgs &a, int hidden, const void *bias2, cudaStream_t s);

// out (p, q) = g^T x over the rows of g (rows, p) and x (rows, q), bias (p) = column sums of g (or null); up to three at once.
struct WeightProblem {
  Operand g, x;
  int p = 0, q = 0;
  void *out = nullptr, *bias = nullptr;      // of the operands' type, rows of q elements
};
constexpr int kMaxWeightProblems = 3;
long long weight_gradient_workspace(long long rows, const WeightProblem *w, int count);
cudaError_t launch_weight_gradient(int dtype, long long rows, const WeightProblem *w, int count, void *workspace, cudaStream_t s);

// Copies of matrices into rows that begin on a 16-byte boundary; fp32 ones are rounded.
struct RowCopy {
  const void *src;
  void *dst;
  long long rows, cols, src_pitch, dst_pitch;
  int wide;
};
constexpr int kMaxRowCopies = 8;
cudaError_t launch_copy_rows(int dtype, const RowCopy *c, int count, cudaStream_t s);

// 8-bit checkpoints; format: DFA3D_FORMAT_*
cudaError_t launch_compress8(const void *x, int dtype, long long rows, int cols, int format, uint8_t *codes, uint8_t *scales,
                             cudaStream_t s);
cudaError_t launch_decompress8(const uint8_t *codes, const uint8_t *scales, int format, long long rows, int cols, int dtype, void *x,
                               long long pitch, cudaStream_t s);

}  // namespace dfa3d
