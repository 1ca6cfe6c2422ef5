// The sm_100a instructions that the matrix products are made of: barriers in shared memory, tiled copies, tensor-core products whose
// accumulators live in tensor memory.  Thin wrappers; operand layouts are described where the descriptors are made.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace dfa3d {
namespace tc {

__device__ __forceinline__ uint32_t shared_address(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ bool one_lane() {
  uint32_t p;
  asm volatile("{\n.reg .pred q;\nelect.sync _|q, 0xffffffff;\nselp.u32 %0, 1, 0, q;\n}" : "=r"(p));
  return p != 0;
}

// ---- barriers ----------------------------------------------------------------------------------
__device__ __forceinline__ void barrier_init(uint32_t bar, uint32_t arrivals) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(arrivals) : "memory");
}
__device__ __forceinline__ void barriers_visible() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void arrive_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool try_wait(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n.reg .pred q;\nmbarrier.try_wait.parity.shared::cta.b64 q, [%1], %2;\nselp.u32 %0, 1, 0, q;\n}"
               : "=r"(done)
               : "r"(bar), "r"(parity)
               : "memory");
  return done != 0;
}
__device__ __forceinline__ uint64_t nanoseconds() {
  uint64_t t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}
constexpr uint64_t kPatience = 4000000000ull;      // ns; waits here last microseconds

// Waits for the phase of `parity` to end; false when that took longer than any sound run could.
static __device__ __noinline__ bool wait_long(uint32_t bar, uint32_t parity) {
  const uint64_t start = nanoseconds();
  do {
    for (int i = 0; i < 64; ++i)
      if (try_wait(bar, parity)) return true;
  } while (nanoseconds() - start < kPatience);
  return false;
}
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity) {
  for (int i = 0; i < 16; ++i)
    if (try_wait(bar, parity)) return true;
  return wait_long(bar, parity);
}

// The same for a whole warp, with one answer.
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)); }

// ---- pairs of CTAs -----------------------------------------------------------------------------
__device__ __forceinline__ uint32_t rank_in_pair() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t address_in(uint32_t at, uint32_t rank) {      // the same place in another CTA's shared memory
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
  return r;
}
// At an address_in().  It hands over nothing but tensor memory that has been read, which order_before() and order_after() see to:
// releasing this CTA's writes to the other one as well took 1600 cycles of a warp at each arrival.
__device__ __forceinline__ void arrive_in(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// The same behind writes to the own CTA's shared memory that the products of both CTAs read there.  An arrival without a scope releases
// to the own CTA only, while the thread that waits and issues the products may sit in the other one.  That rests on an assumption: no
// thread of the other CTA reads what was written, the tensor cores of this SM do, through the async proxy, to which shared_to_async() has
// made it visible before the arrival leaves this SM, and the products that read it are issued when the arrival has been seen.  A
// release to the pair is what the memory model would ask for besides; with it the gated block's forward takes 42 us for 35.7 (40 000 rows,
// 256 -> 512 -> 256, no activation).
__device__ __forceinline__ void hand_over_in(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void pair_sync() {      // all threads of both
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---- kernels that follow one another -------------------------------------------------------------
// A kernel launched by launch_after() may begin while the one before it in the stream ends; it reads and writes nothing before this.
__device__ __forceinline__ void wait_for_last_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_kernel_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// ---- tiled copies ------------------------------------------------------------------------------
__device__ __forceinline__ void tile_load(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
               "l"(map), "r"(x), "r"(y), "r"(bar)
               : "memory");
}
// The same for one of a pair, whose barrier may be the other's.
__device__ __forceinline__ void tile_load_pair(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tile_to_l2(const CUtensorMap *map, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void tile_store(const CUtensorMap *map, int x, int y, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y), "r"(src)
               : "memory");
}
__device__ __forceinline__ void stores_asked() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void stores_read() {      // all but the last LEFT groups have left shared memory
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(LEFT) : "memory");
}
__device__ __forceinline__ void stores_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
// ordinary accesses of shared memory before it, tiled copies and products of it after it
__device__ __forceinline__ void shared_to_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---- tensor memory -----------------------------------------------------------------------------
// By one warp of each of the pair's CTAs, for products of both.
template <int COLUMNS> __device__ __forceinline__ void tensor_memory_take(uint32_t where) {
  static_assert(COLUMNS >= 32 && COLUMNS <= 512 && (COLUMNS & (COLUMNS - 1)) == 0, "power of two");
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(where), "n"(COLUMNS) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
}
template <int COLUMNS> __device__ __forceinline__ void tensor_memory_give(uint32_t base) {       // the same warp
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "n"(COLUMNS));
}
__device__ __forceinline__ void order_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void order_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Columns of the 32 lanes that this warp may read: thread = lane = row of the accumulator.  They are not there before
// tensor_loads_done(), through which they pass so that nothing that uses them can be moved in front of it.
__device__ __forceinline__ void tensor_load(float (&v)[32], uint32_t at) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,"
      "%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
      "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
        "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
        "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(at));
}
__device__ __forceinline__ void tensor_loads_done(float (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
      : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
        "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]),
        "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]),
        "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
      :
      : "memory");
}
__device__ __forceinline__ void tensor_load(float (&v)[16], uint32_t at) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
      : "r"(at));
}
__device__ __forceinline__ void tensor_loads_done(float (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
      : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
        "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
      :
      : "memory");
}

// ---- products ----------------------------------------------------------------------------------
// Operand tiles are rows of 128 bytes (64 elements of 16 bits) whose 16-byte pieces are permuted by the low three bits of the row
// number (the 128-byte swizzle of tiled copies), on a 1024-byte boundary.
//   k_major:  a row is 64 elements along the summed axis; eight rows, 1024 bytes, further come the next eight of the other axis.  A
//             step of 16 along the summed axis is 32 bytes.
//   mn_major: a row is 64 elements along the other axis, one row for each element of the summed one; eight rows, 1024 bytes, further
//             come the next eight of the summed axis; `group` bytes further the next 64 of the other.  A step of 16 is 2048 bytes.
//   mn_major_narrow: the same with rows of 64 bytes, 32 elements, and the 64-byte swizzle.  A step of 16 is 1024 bytes.
constexpr uint64_t kOperandBits = (uint64_t(1) << 46) | (uint64_t(2) << 61) | (uint64_t(1024 >> 4) << 32);
constexpr uint64_t kNarrowBits = (uint64_t(1) << 46) | (uint64_t(4) << 61) | (uint64_t(512 >> 4) << 32);
__device__ __forceinline__ uint64_t k_major(uint32_t at) { return kOperandBits | (uint64_t(1) << 16) | ((at >> 4) & 0x3fff); }
__device__ __forceinline__ uint64_t mn_major(uint32_t at, uint32_t group) {
  return kOperandBits | (uint64_t(group >> 4) << 16) | ((at >> 4) & 0x3fff);
}
__device__ __forceinline__ uint64_t mn_major_narrow(uint32_t at) { return kNarrowBits | (uint64_t(1) << 16) | ((at >> 4) & 0x3fff); }
template <typename T> constexpr uint32_t kOperandType = 0;                     // fp16
template <> inline constexpr uint32_t kOperandType<__nv_bfloat16> = 1;
// the pair's 256 rows; n columns; 32-bit sums
template <typename T> __host__ __device__ constexpr uint32_t product_shape(int rows, int n, bool a_mn_major, bool b_mn_major) {
  return (1u << 4) | (kOperandType<T> << 7) | (kOperandType<T> << 10) | (uint32_t(a_mn_major) << 15) | (uint32_t(b_mn_major) << 16) |
         (uint32_t(n / 8) << 17) | (uint32_t(rows / 16) << 24);
}
// D (+)= A B over 16 elements of the summed axis; one thread of the pair's first CTA.  Each CTA holds its 128 rows of A and of D and half
// of B's columns, all at the same places.
__device__ __forceinline__ void product(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, bool add) {
  asm volatile("{\n.reg .pred q;\nsetp.ne.u32 q, %4, 0;\ntcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, q;\n}" ::"r"(d), "l"(a),
               "l"(b), "r"(shape), "r"((uint32_t)add)
               : "memory");
}
// The barrier of both CTAs is arrived at when the products that this thread has issued so far are done.
__device__ __forceinline__ void products_arrive(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
               "h"((uint16_t)3)
               : "memory");
}

// ---- shared memory by address ------------------------------------------------------------------
__device__ __forceinline__ uint4 read16(uint32_t at) {
  uint4 w;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(at) : "memory");
  return w;
}
__device__ __forceinline__ void write16(uint32_t at, uint4 w) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w) : "memory");
}
template <typename O> __device__ __forceinline__ O read_one(uint32_t at) {
  O v;
  if constexpr (sizeof(O) == 4) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  else asm volatile("ld.shared.u16 %0, [%1];" : "=h"(reinterpret_cast<uint16_t &>(v)) : "r"(at) : "memory");
  return v;
}
template <typename O> __device__ __forceinline__ void write_one(uint32_t at, O v) {
  if constexpr (sizeof(O) == 4) asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory");
  else asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"(reinterpret_cast<const uint16_t &>(v)) : "memory");
}
__device__ __forceinline__ float4 read_four(uint32_t at) {
  float4 w;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(w.x), "=f"(w.y), "=f"(w.z), "=f"(w.w) : "r"(at) : "memory");
  return w;
}

}  // namespace tc
}  // namespace dfa3d
