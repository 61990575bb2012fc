// nsb_tcgen05.cuh -- mbarriers, TMA loads and the fifth-generation tensor core (tcgen05) as inline
// PTX, for the NVFP4 product.  Every wait is bounded.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace nsb {

__device__ __forceinline__ uint32_t shared_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// One thread of a converged warp, the same one each time.
__device__ __forceinline__ bool elect_one() {
  uint32_t elected;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(elected));
  return elected != 0;
}

// Until the kernels ahead in the stream are complete (a launch that may overlap them).
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// A word, one float32, or four, of CTA `rank`'s shared memory in the cluster, where this CTA's `address` would be.
__device__ __forceinline__ uint32_t remote_address(uint32_t address, int rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(address), "r"(rank));
  return remote;
}
__device__ __forceinline__ void remote_store(int* own, int rank, int v) {
  asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(remote_address(shared_addr(own), rank)), "r"(v) : "memory");
}
__device__ __forceinline__ void remote_load(uint32_t address, int rank, float (&v)[1]) {
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[0]) : "r"(remote_address(address, rank)) : "memory");
}
__device__ __forceinline__ void remote_load(uint32_t address, int rank, float (&v)[4]) {
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(remote_address(address, rank)) : "memory");
}

// ---------------------------------------------------------------------------
// mbarriers
// ---------------------------------------------------------------------------
__device__ __forceinline__ void barrier_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(shared_addr(bar)), "r"(count) : "memory");
}

__device__ __forceinline__ void barrier_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(shared_addr(bar)) : "memory");
}

__device__ __forceinline__ void barrier_arrive_expect(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(shared_addr(bar)), "r"(bytes) : "memory");
}

__device__ __forceinline__ bool barrier_try(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(shared_addr(bar)), "r"(parity)
      : "memory");
  return done != 0;
}

// Arrives on the barrier that lies at `bar` in the shared memory of the cluster's CTA `rank`.  It tells that the
// warp's tensor memory has been read: tcgen05.wait::ld and the tcgen05 fences order that, no plain memory access.
__device__ __forceinline__ void barrier_arrive_at(uint64_t* bar, int rank) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(remote_address(shared_addr(bar), rank)) : "memory");
}

// Counts `bytes` as arrived that no copy will bring.
__device__ __forceinline__ void barrier_forgo(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(shared_addr(bar)), "r"(bytes) : "memory");
}

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Polls before a wait gives up: 4 us each, 17 s (a sum over 2^31 columns takes about two).
constexpr int kBarrierPolls = 1 << 22;

// Waits for the phase `parity` of `bar`.  At every 256th poll it gives up where another role of the CTA has
// (`*aborted`), or after `polls`.
__device__ __forceinline__ bool barrier_wait(uint64_t* bar, uint32_t parity, volatile int* aborted, int polls) {
  for (int i = 1;; ++i) {
    if (barrier_try(bar, parity)) return true;
    if ((i & 255) == 0 && (*aborted || i >= polls)) return false;
  }
}

// After a wait has given up: for work in flight, which ends by itself; bounded all the same.
__device__ __forceinline__ void barrier_drain(uint64_t* bar, uint32_t parity) {
  for (int i = 0; i < kBarrierPolls && !barrier_try(bar, parity); ++i) {
  }
}

// ---------------------------------------------------------------------------
// Copies into shared memory (completion counted in bytes on an mbarrier)
// ---------------------------------------------------------------------------
// A box of a two-dimensional byte tensor; x (bytes) is a multiple of 16.
__device__ __forceinline__ void load_box(void* to, const void* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          shared_addr(to)),
      "l"(map), "r"(x), "r"(y), "r"(shared_addr(bar))
      : "memory");
}

// The same of a pair's CTA, to its own shared memory, and a box of 2,048 bytes at the start of a row of a
// three-dimensional tensor.  `bar`: an address in the cluster's shared memory, so the barrier may be the other CTA's.
__device__ __forceinline__ void load_box_pair(void* to, const void* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          shared_addr(to)),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void load_row_pair(void* to, const void* map, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          shared_addr(to)),
      "l"(map), "r"(0), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

// `bytes` consecutive bytes; both addresses and the size are multiples of 16.
__device__ __forceinline__ void load_bytes(void* to, const void* from, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   shared_addr(to)),
               "l"(from), "r"(bytes), "r"(shared_addr(bar))
               : "memory");
}

// ---------------------------------------------------------------------------
// Tensor memory: 128 lanes x 512 columns of 32 bits; an address is lane << 16 | column.
// ---------------------------------------------------------------------------
// By one whole warp (kPair: of each of the two CTAs), which also frees it.  The address lands in *slot (shared memory).
template <bool kPair>
__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t columns) {
  if constexpr (kPair) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_addr(slot)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_addr(slot)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
}

template <bool kPair>
__device__ __forceinline__ void tmem_free(uint32_t address, uint32_t columns) {
  if constexpr (kPair) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns));
  else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns));
}

__device__ __forceinline__ void tcgen05_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tcgen05_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 16 columns of the warp's 32 lanes, one lane per thread; tmem_wait() before they are used.
__device__ __forceinline__ void tmem_load16(uint32_t address, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(address));
}
// Waits for the warp's loads; then tmem_loaded() of each set, so that no use of its values moves ahead of the wait.
__device__ __forceinline__ void tmem_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_loaded(uint32_t (&v)[16]) {
  asm volatile(""
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]),
                 "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]));
}

// ---------------------------------------------------------------------------
// Shared-memory descriptors: address and strides in units of 16 bytes, bit 46 the descriptor's version.
// ---------------------------------------------------------------------------
// Rows of 128 bytes in the 128-byte swizzle (as load_box leaves them), groups of 8 rows 1,024 bytes apart.
__device__ __forceinline__ uint64_t swizzled_descriptor(uint32_t address) {
  return static_cast<uint64_t>((address >> 4) & 0x3fff) | (uint64_t{1} << 16) | (uint64_t{64} << 32) | (uint64_t{1} << 46) |
         (uint64_t{2} << 61);
}
// Rows of 16 bytes without a swizzle, groups of 8 rows 128 bytes apart.
__device__ __forceinline__ uint64_t plain_descriptor(uint32_t address) {
  return static_cast<uint64_t>((address >> 4) & 0x3fff) | (uint64_t{1} << 16) | (uint64_t{8} << 32) | (uint64_t{1} << 46);
}

// ---------------------------------------------------------------------------
// Block-scaled products of E2M1 operands with a UE4M3 scale per 16 elements
// ---------------------------------------------------------------------------
// A pair (kPair) is a cluster of two CTAs whose tensor cores work on one product: its first CTA issues for
// both.  Each holds its half of the lanes and sums, its half of B's rows, and the scales of its lanes and
// of all of B, at the same places.

// 512 bytes of scales (32 rows of 16 bytes) to 4 columns, in each of the four 32-lane quarters (of both
// CTAs, from the shared memory of each).  Ordered before the products that the same thread issues after it.
template <bool kPair>
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint64_t descriptor) {
  if constexpr (kPair) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(descriptor) : "memory");
  else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(descriptor) : "memory");
}

// The instruction descriptor: E2M1 x E2M1, UE4M3 scales, M lanes (128, of a pair 256), N columns, both operands K-major.
__device__ __forceinline__ uint32_t nvfp4_instruction(int m, int n) {
  return (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// One thread: D[m, n] (+)= A[m, 64] B[n, 64]^T with the scales at scale_a / scale_b in tensor memory.
template <bool kPair>
__device__ __forceinline__ void nvfp4_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t instruction, uint32_t scale_a,
                                          uint32_t scale_b, bool accumulate) {
  if constexpr (kPair)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(instruction), "r"(scale_a), "r"(scale_b), "r"(accumulate ? 1u : 0u)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(instruction), "r"(scale_a), "r"(scale_b), "r"(accumulate ? 1u : 0u)
        : "memory");
}

// Arrives on `bar` (of a pair: in both CTAs) once all tcgen05 work that this thread has issued is complete.
template <bool kPair>
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  if constexpr (kPair)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(shared_addr(bar)),
                 "h"(static_cast<uint16_t>(3))
                 : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(shared_addr(bar)) : "memory");
}

}  // namespace nsb
