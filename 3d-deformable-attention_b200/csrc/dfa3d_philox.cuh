// The mask of a dropout as a function of (seed, site, element), so that a backward forms it again and nobody stores it.
//
// Element i of a tensor in row-major order takes word i mod 4 of Philox4x32 at counter (i / 4 low, i / 4 high, site, 0) under the
// key (seed low, seed high), and is kept where word >= p * 2^32.  The generator is Philox4x32 of Salmon, Moraes, Dror and Shaw,
// "Parallel random numbers: as easy as 1, 2, 3" (SC 2011), with 7 rounds, the fewest that the authors found to pass all of
// TestU01's BigCrush: a block of four words then costs 43 instructions, counted on the device (25 are the 12 products and 13 logic
// operations that the rounds take where the counter's upper half and the site are the CTA's; the rest forms round keys and counters), and
// a 16-bit dropout stays near the speed of HBM.
#pragma once
#include <stdint.h>

namespace dfa3d {

// What a kernel gets to know of a dropout.  `last` is the largest word that is dropped; `rng` is false where nothing is (p below
// 2^-33), and no word is formed then.
struct DropRule {
  const int64_t *seed;      // device, one element
  uint32_t site;
  uint32_t last;
  float scale;              // 1 / (1 - p)
  bool rng;
};

// p in [0, 1]
inline DropRule drop_rule(double p, const int64_t *seed, uint32_t site) {
  const uint64_t dropped = (uint64_t)(p * 4294967296.0 + 0.5);
  DropRule r;
  r.seed = seed;
  r.site = site;
  r.rng = dropped > 0;
  r.last = dropped > 0 ? (uint32_t)(dropped - 1) : 0u;
  r.scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.f;
  return r;
}

struct DropKey {
  uint32_t k0, k1;
};
struct PhiloxWords {
  uint32_t x, y, z, w;
};

// The block of element base + e, for a base that is a multiple of `width` (2048 or 4096, the elements of a CTA) and e < width: no carry
// leaves the lower half, so that the upper one is the same for the whole CTA, and so is what the first round makes of it.
#ifdef __CUDACC__
__host__ __device__ __forceinline__
#else
inline
#endif
unsigned long long block_of(unsigned long long base, uint32_t e) {
  const unsigned long long block = base >> 2;
  return (block & 0xffffffff00000000ull) | (uint32_t)((uint32_t)block + (e >> 2));
}

#ifdef __CUDACC__
__host__ __device__ __forceinline__
#else
inline
#endif
PhiloxWords philox_words(unsigned long long block, uint32_t site, DropKey k) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = site, c3 = 0u;
#ifdef __CUDACC__
#pragma unroll
#endif
  for (int r = 0; r < 7; ++r) {
    const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k.k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k.k1;
    c3 = (uint32_t)a;
    k.k0 += 0x9E3779B9u;
    k.k1 += 0xBB67AE85u;
  }
  return {c0, c1, c2, c3};
}

#ifdef __CUDACC__
__device__ __forceinline__ DropKey drop_key(const DropRule &d) {
  DropKey k = {0u, 0u};
  if (d.rng) {
    const unsigned long long s = (unsigned long long)__ldg(reinterpret_cast<const long long *>(d.seed));
    k.k0 = (uint32_t)s;
    k.k1 = (uint32_t)(s >> 32);
  }
  return k;
}

// words[i] is that of element `first` + i, a multiple of 4; above `last` where nothing is dropped.
template <int V>
__device__ __forceinline__ void words_of(const DropRule &d, DropKey k, unsigned long long first, uint32_t (&words)[V]) {
  if (!d.rng) {
#pragma unroll
    for (int i = 0; i < V; ++i) words[i] = ~0u;
    return;
  }
#pragma unroll
  for (int i = 0; i < V; i += 4) {
    const PhiloxWords w = philox_words((first >> 2) + i / 4, d.site, k);
    words[i] = w.x; words[i + 1] = w.y; words[i + 2] = w.z; words[i + 3] = w.w;
  }
}
#endif

}  // namespace dfa3d
