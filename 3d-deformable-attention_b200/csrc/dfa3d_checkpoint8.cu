// Activations kept in 8 bits until the backward: blocks of 32 neighbours of a row under one power of two, the smallest for which no
// element is beyond the format's largest number.  Under a power of two a code times the block's factor is a number of the 16-bit
// types too (7 or 4 bits behind the factor), so that the products of a backward read exactly what the codes stand for.
//
// HBM binds: bytes of both sides are all there is.  Measured: bf16 184 950 x 256 to e4m3 (144 MB, 22 us at 6.55 TB/s) 28 us in, 21
// out; fp32 40 000 x 512 to int8 (103 MB, 16 us) 17 in, 25 out (82 MB of it written, which a fill does in 14).  A
// thread has four items, whose loads are on their way together.
#include <cuda_fp8.h>

#include "dfa3d_b200.h"
#include "dfa3d_common.cuh"
#include "dfa3d_product.h"
#include "dfa3d_rowvec.cuh"

namespace dfa3d {
namespace {

constexpr int kPack = 8, kBlock = 32;      // elements of a thread, of a block (four threads)
constexpr int kThreads8 = 256, kItems = 4;

// The factor's exponent + 127 for a largest magnitude of `top` (its bits); 255 where that is no number.
template <int FORMAT> __device__ __forceinline__ uint32_t scale_of(uint32_t top) {
  constexpr uint32_t most = FORMAT == DFA3D_FORMAT_INT8 ? 0x7e0000u : 0x600000u;      // 127 = 1.984375 x 2^6, 448 = 1.75 x 2^8
  constexpr int shift = FORMAT == DFA3D_FORMAT_INT8 ? 6 : 8;
  if (top >= 0x7f800000u) return 255u;
  const int e = (int)(top >> 23) - shift + ((top & 0x7fffffu) > most);
  return (uint32_t)(e < 0 ? 0 : e);
}
__device__ __forceinline__ float power_of(uint32_t scale) {      // 2^(scale - 127), not a number for 255
  return __uint_as_float(scale == 0 ? 0x00400000u : scale == 255 ? 0x7fffffffu : scale << 23);
}
__device__ __forceinline__ float inverse_of(uint32_t scale) { return power_of(scale == 255 ? 127u : 254u - scale); }

template <int FORMAT> __device__ __forceinline__ uint2 encode(const float (&f)[kPack], float inverse) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if constexpr (FORMAT == DFA3D_FORMAT_INT8) {
      uint32_t b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) b[i] = (uint32_t)__float2int_rn(f[h * 4 + i] * inverse);
      w[h] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    } else {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[h * 4] * inverse, f[h * 4 + 1] * inverse), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[h * 4 + 2] * inverse, f[h * 4 + 3] * inverse), __NV_SATFINITE, __NV_E4M3);
      w[h] = lo | hi << 16;
    }
  }
  return make_uint2(w[0], w[1]);
}

template <typename T> __device__ __forceinline__ float largest();
template <> __device__ __forceinline__ float largest<float>() { return __uint_as_float(0x7f7fffffu); }
template <> __device__ __forceinline__ float largest<__nv_bfloat16>() { return __uint_as_float(0x7f7f0000u); }
template <> __device__ __forceinline__ float largest<__half>() { return 65504.f; }

template <typename T, int FORMAT> __device__ __forceinline__ void decode(uint2 codes, uint32_t scale, float (&f)[kPack]) {
  const float power = power_of(scale), most = largest<T>();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t w = h ? codes.y : codes.x;
    if constexpr (FORMAT == DFA3D_FORMAT_INT8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) f[h * 4 + i] = (float)(int8_t)(w >> (8 * i));
    } else {
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (8 * i)), __NV_E4M3);
        const float2 v = __half22float2(__half2(r));
        f[h * 4 + i] = v.x;
        f[h * 4 + i + 1] = v.y;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kPack; ++i) {      // a largest element that was rounded up may be beyond the type: comparisons let NaN through
    const float v = f[i] * power;
    f[i] = v > most ? most : v < -most ? -most : v;
  }
}

// Item = eight elements of a row: (row, piece), `pieces` a row.  How they lie: kFlat, whole blocks in every row, so that neither rows
// nor blocks have to be found (a division costs more than the rest of an item); kWords, rows of whole items; kAny.
enum Lie { kFlat, kWords, kAny };
template <Lie LIE> struct Items {
  long long items;
  int pieces;
  __device__ __forceinline__ void find(long long item, long long &row, int &col) const {
    if constexpr (LIE == kFlat) {
      row = 0;
      col = 0;
    } else {
      row = item >> 31 ? item / pieces : (long long)((uint32_t)item / (uint32_t)pieces);
      col = (int)(item - row * pieces) * kPack;
    }
  }
};

template <typename T, int FORMAT, Lie LIE>
__global__ void __launch_bounds__(kThreads8) compress8_kernel(const T *__restrict__ x, long long rows, int cols, uint8_t *__restrict__ codes,
                                                               uint8_t *__restrict__ scales) {
  const int blocks = (cols + kBlock - 1) / kBlock;
  const Items<LIE> all{rows * blocks * 4, blocks * 4};
  for (long long first = (long long)blockIdx.x * (kThreads8 * kItems); first < all.items;
       first += (long long)gridDim.x * (kThreads8 * kItems)) {
    float f[kItems][kPack];
    long long row[kItems];
    int col[kItems];
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const long long item = first + k * kThreads8 + threadIdx.x;
      all.find(item, row[k], col[k]);
#pragma unroll
      for (int i = 0; i < kPack; ++i) f[k][i] = 0.f;
      if (item >= all.items) continue;
      const T *src = LIE == kFlat ? x + item * kPack : x + row[k] * cols + col[k];
      if constexpr (LIE != kAny) {
        if (col[k] < cols) {
          constexpr int V = 16 / (int)sizeof(T);
#pragma unroll
          for (int i = 0; i < kPack; i += V) {
            float g[V];
            widen_word<T, V>(load_once<T, V>(src + i), g);
#pragma unroll
            for (int j = 0; j < V; ++j) f[k][i + j] = g[j];
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < kPack; ++i)
          if (col[k] + i < cols) f[k][i] = wide(src[i]);
      }
    }
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const long long item = first + k * kThreads8 + threadIdx.x;
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < kPack; ++i) top = max(top, __float_as_uint(f[k][i]) & 0x7fffffffu);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const uint32_t scale = scale_of<FORMAT>(top);
      if (item >= all.items) continue;
      if (scale == 255) {
#pragma unroll
        for (int i = 0; i < kPack; ++i) f[k][i] = 0.f;
      }
      if constexpr (LIE == kFlat) {
        if (item % 4 == 0) scales[item / 4] = (uint8_t)scale;
      } else {
        if (col[k] % kBlock == 0) scales[row[k] * blocks + col[k] / kBlock] = (uint8_t)scale;
      }
      const uint2 w = encode<FORMAT>(f[k], inverse_of(scale));
      uint8_t *dst = LIE == kFlat ? codes + item * kPack : codes + row[k] * cols + col[k];
      if constexpr (LIE != kAny) {
        if (col[k] < cols) *reinterpret_cast<uint2 *>(dst) = w;
      } else {
#pragma unroll
        for (int i = 0; i < kPack; ++i)
          if (col[k] + i < cols) dst[i] = (uint8_t)((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
      }
    }
  }
}

template <typename T, int FORMAT, Lie LIE>
__global__ void __launch_bounds__(kThreads8) decompress8_kernel(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales,
                                                                 long long rows, int cols, T *__restrict__ x, long long pitch) {
  const int blocks = (cols + kBlock - 1) / kBlock, pieces = (cols + kPack - 1) / kPack;
  const Items<LIE> all{rows * pieces, pieces};
  for (long long first = (long long)blockIdx.x * (kThreads8 * kItems); first < all.items;
       first += (long long)gridDim.x * (kThreads8 * kItems)) {
    uint2 w[kItems];
    uint32_t scale[kItems];
    long long row[kItems];
    int col[kItems];
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const long long item = first + k * kThreads8 + threadIdx.x;
      all.find(item, row[k], col[k]);
      w[k] = make_uint2(0, 0);
      scale[k] = 0;
      if (item >= all.items) continue;
      const uint8_t *src = LIE == kFlat ? codes + item * kPack : codes + row[k] * cols + col[k];
      if constexpr (LIE != kAny) {
        w[k] = __ldcs(reinterpret_cast<const uint2 *>(src));
      } else {
#pragma unroll
        for (int i = 0; i < kPack; ++i)
          if (col[k] + i < cols) (i < 4 ? w[k].x : w[k].y) |= (uint32_t)src[i] << (8 * (i & 3));
      }
      scale[k] = scales[LIE == kFlat ? item / 4 : row[k] * blocks + col[k] / kBlock];
    }
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const long long item = first + k * kThreads8 + threadIdx.x;
      if (item >= all.items) continue;
      float f[kPack];
      decode<T, FORMAT>(w[k], scale[k], f);
      T *dst = LIE == kFlat ? x + item * kPack : x + row[k] * pitch + col[k];
      if constexpr (LIE != kAny) {
        constexpr int V = 16 / (int)sizeof(T);
#pragma unroll
        for (int i = 0; i < kPack; i += V) {
          float g[V];
#pragma unroll
          for (int j = 0; j < V; ++j) g[j] = f[i + j];
          store_word<T, V>(dst + i, g);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kPack; ++i)
          if (col[k] + i < cols) dst[i] = narrow<T>(f[i]);
      }
    }
  }
}

bool on_grid(const void *p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

unsigned grid_of(long long items) {
  const long long ctas = (items + kThreads8 * kItems - 1) / (kThreads8 * kItems);
  return (unsigned)(ctas < (1 << 30) ? ctas : 1 << 30);
}

template <typename T, int FORMAT>
void compress_typed(const void *x, long long rows, int cols, uint8_t *codes, uint8_t *scales, cudaStream_t s) {
  const unsigned grid = grid_of(rows * ((cols + kBlock - 1) / kBlock) * 4);
  const T *src = static_cast<const T *>(x);
  const bool words = cols % kPack == 0 && on_grid(x, 16) && on_grid(codes, 8);
  if (words && cols % kBlock == 0) compress8_kernel<T, FORMAT, kFlat><<<grid, kThreads8, 0, s>>>(src, rows, cols, codes, scales);
  else if (words) compress8_kernel<T, FORMAT, kWords><<<grid, kThreads8, 0, s>>>(src, rows, cols, codes, scales);
  else compress8_kernel<T, FORMAT, kAny><<<grid, kThreads8, 0, s>>>(src, rows, cols, codes, scales);
}
template <typename T, int FORMAT>
void decompress_typed(const uint8_t *codes, const uint8_t *scales, long long rows, int cols, void *x, long long pitch, cudaStream_t s) {
  const unsigned grid = grid_of(rows * ((cols + kPack - 1) / kPack));
  T *dst = static_cast<T *>(x);
  const bool words = cols % kPack == 0 && pitch % kPack == 0 && on_grid(x, 16) && on_grid(codes, 8);
  if (words && cols % kBlock == 0 && pitch == cols)
    decompress8_kernel<T, FORMAT, kFlat><<<grid, kThreads8, 0, s>>>(codes, scales, rows, cols, dst, pitch);
  else if (words) decompress8_kernel<T, FORMAT, kWords><<<grid, kThreads8, 0, s>>>(codes, scales, rows, cols, dst, pitch);
  else decompress8_kernel<T, FORMAT, kAny><<<grid, kThreads8, 0, s>>>(codes, scales, rows, cols, dst, pitch);
}

// ------------------------------------------------------------------------------------------------
struct Copies {
  RowCopy of[kMaxRowCopies];
  int words[kMaxRowCopies];      // eight elements at a time
};
template <typename T> __global__ void __launch_bounds__(256) copy_rows_kernel(const __grid_constant__ Copies c) {
  const RowCopy &m = c.of[blockIdx.y];
  const int each = c.words[blockIdx.y] ? 8 : 1;
  const long long n = m.rows * m.cols / each, across = m.cols / each;
  T *dst = static_cast<T *>(m.dst);
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const long long row = (i | across) >> 31 ? i / across : (long long)((uint32_t)i / (uint32_t)across), col = (i - row * across) * each;
    T *to = dst + row * m.dst_pitch + col;
    if (each == 1) {
      *to = m.wide ? narrow<T>(static_cast<const float *>(m.src)[row * m.src_pitch + col])
                   : static_cast<const T *>(m.src)[row * m.src_pitch + col];
    } else if (m.wide) {
      const float *from = static_cast<const float *>(m.src) + row * m.src_pitch + col;
      float f[8], a[4], b[4];
      widen_word<float, 4>(load_once<float, 4>(from), a);
      widen_word<float, 4>(load_once<float, 4>(from + 4), b);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        f[k] = a[k];
        f[4 + k] = b[k];
      }
      store_word<T, 8>(to, f);
    } else {
      *reinterpret_cast<uint4 *>(to) = *reinterpret_cast<const uint4 *>(static_cast<const T *>(m.src) + row * m.src_pitch + col);
    }
  }
}

}  // namespace

cudaError_t launch_compress8(const void *x, int dtype, long long rows, int cols, int format, uint8_t *codes, uint8_t *scales,
                             cudaStream_t s) {
#define TYPED(T)                                                                                                     \
  format == DFA3D_FORMAT_INT8 ? compress_typed<T, DFA3D_FORMAT_INT8>(x, rows, cols, codes, scales, s)               \
                              : compress_typed<T, DFA3D_FORMAT_E4M3>(x, rows, cols, codes, scales, s)
  if (dtype == DFA3D_DTYPE_F32) TYPED(float);
  else if (dtype == DFA3D_DTYPE_F16) TYPED(__half);
  else TYPED(__nv_bfloat16);
#undef TYPED
  return cudaGetLastError();
}

cudaError_t launch_decompress8(const uint8_t *codes, const uint8_t *scales, int format, long long rows, int cols, int dtype, void *x,
                               long long pitch, cudaStream_t s) {
#define TYPED(T)                                                                                                     \
  format == DFA3D_FORMAT_INT8 ? decompress_typed<T, DFA3D_FORMAT_INT8>(codes, scales, rows, cols, x, pitch, s)      \
                              : decompress_typed<T, DFA3D_FORMAT_E4M3>(codes, scales, rows, cols, x, pitch, s)
  if (dtype == DFA3D_DTYPE_F32) TYPED(float);
  else if (dtype == DFA3D_DTYPE_F16) TYPED(__half);
  else TYPED(__nv_bfloat16);
#undef TYPED
  return cudaGetLastError();
}

cudaError_t launch_copy_rows(int dtype, const RowCopy *c, int count, cudaStream_t s) {
  Copies m{};
  long long most = 0;
  for (int i = 0; i < count; ++i) {
    m.of[i] = c[i];
    m.words[i] = c[i].cols % 8 == 0 && c[i].src_pitch % (c[i].wide ? 4 : 8) == 0 && c[i].dst_pitch % 8 == 0 && on_grid(c[i].src, 16) &&
                 on_grid(c[i].dst, 16);
    const long long n = c[i].rows * c[i].cols / (m.words[i] ? 8 : 1);
    most = n > most ? n : most;
  }
  const long long ctas = (most + 511) / 512, wave = 8LL * sm_count();
  const dim3 grid((unsigned)(ctas < wave ? ctas : wave), count);
  if (dtype == DFA3D_DTYPE_F16) copy_rows_kernel<__half><<<grid, 256, 0, s>>>(m);
  else copy_rows_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(m);
  return cudaGetLastError();
}

}  // namespace dfa3d
