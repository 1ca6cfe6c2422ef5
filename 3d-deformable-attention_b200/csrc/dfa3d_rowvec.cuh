// Runs of V consecutive elements of a row as 32-bit floats: loads and stores in one word of up to 16 bytes where V elements are
// aligned for it, one element at a time otherwise.  Arithmetic of the row operators is 32-bit whatever the storage type; a store
// rounds once, to nearest even.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace dfa3d {

template <int BYTES> struct WordOf;
template <> struct WordOf<16> { using type = uint4; };
template <> struct WordOf<8> { using type = uint2; };
template <> struct WordOf<4> { using type = uint32_t; };
template <> struct WordOf<2> { using type = uint16_t; };

template <typename T, int V> using Word = typename WordOf<V * (int)sizeof(T)>::type;

__device__ __forceinline__ float wide(float x) { return x; }
__device__ __forceinline__ float wide(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float wide(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T narrow(float x);
template <> __device__ __forceinline__ float narrow<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half narrow<__half>(float x) { return __float2half_rn(x); }

__device__ __forceinline__ void widen2(uint32_t w, float &lo, float &hi, __nv_bfloat16 *) {
  lo = __uint_as_float(w << 16);
  hi = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ void widen2(uint32_t w, float &lo, float &hi, __half *) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
  lo = f.x;
  hi = f.y;
}
__device__ __forceinline__ uint32_t narrow2(float lo, float hi, __nv_bfloat16 *) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t narrow2(float lo, float hi, __half *) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}

template <typename T, int V>
__device__ __forceinline__ void widen_word(const Word<T, V> &w, float (&f)[V]) {
  if constexpr (sizeof(T) == 4) {
    const float *s = reinterpret_cast<const float *>(&w);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = s[i];
  } else if constexpr (V == 1) {
    f[0] = wide(*reinterpret_cast<const T *>(&w));
  } else {
    const uint32_t *s = reinterpret_cast<const uint32_t *>(&w);
#pragma unroll
    for (int i = 0; i < V; i += 2) widen2(s[i / 2], f[i], f[i + 1], (T *)nullptr);
  }
}

template <typename T, int V>
__device__ __forceinline__ Word<T, V> narrow_word(const float (&f)[V]) {
  Word<T, V> w;
  if constexpr (sizeof(T) == 4) {
    float *d = reinterpret_cast<float *>(&w);
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] = f[i];
  } else if constexpr (V == 1) {
    *reinterpret_cast<T *>(&w) = narrow<T>(f[0]);
  } else {
    uint32_t *d = reinterpret_cast<uint32_t *>(&w);
#pragma unroll
    for (int i = 0; i < V; i += 2) d[i / 2] = narrow2(f[i], f[i + 1], (T *)nullptr);
  }
  return w;
}

// Loads for data that this launch reads once (they leave the caches first), and plain ones.
template <typename T, int V>
__device__ __forceinline__ Word<T, V> load_once(const T *p) {
  return __ldcs(reinterpret_cast<const Word<T, V> *>(p));
}
template <typename T, int V>
__device__ __forceinline__ Word<T, V> load_word(const T *p) {
  return *reinterpret_cast<const Word<T, V> *>(p);
}
template <typename T, int V>
__device__ __forceinline__ void store_word(T *p, const float (&f)[V]) {
  *reinterpret_cast<Word<T, V> *>(p) = narrow_word<T, V>(f);
}

template <typename T, int V>
__device__ __forceinline__ void store_once(T *p, const float (&f)[V]) {
  __stcs(reinterpret_cast<Word<T, V> *>(p), narrow_word<T, V>(f));
}

// A 16-byte copy into shared memory that nobody waits for yet; the thread that asked for it may read it after copies_wait().
__device__ __forceinline__ void copy_async16(unsigned shared, const void *global) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(shared), "l"(global) : "memory");
}
__device__ __forceinline__ void copies_asked() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_wait() {      // all but the last LEFT groups are there
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}
__device__ __forceinline__ uint4 read_shared16(unsigned shared) {
  uint4 w;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(shared) : "memory");
  return w;
}

}  // namespace dfa3d
