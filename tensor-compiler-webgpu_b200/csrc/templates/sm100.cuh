// tcb/sm100.cuh -- the sm_100a primitives the tensor-core templates share: mbarriers with bounded waits,
// TMA tile copies, tcgen05 commits, fences and accumulator reads.
#pragma once

namespace tcb {

struct alignas(64) TmaDesc { u64 v[16]; };
struct GemmParams {
  TmaDesc maps[5];  // A_hi / raw A, A_lo, B_hi / raw B, B_lo (3-D: {cols, rows, batch}); [4] the output
  Args a;
};

#ifndef TCB_WAIT_NS
#define TCB_WAIT_NS 2000000000u  // 2 s: far above any legitimate wait
#endif
constexpr u32 WAIT_NS = TCB_WAIT_NS;

__device__ __forceinline__ u32 smem_u32(const void* p) { return (u32)__cvta_generic_to_shared(p); }
__device__ __forceinline__ u64 now_ns() { u64 t; asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t)); return t; }

__device__ __forceinline__ void mbar_init(u32 bar, u32 count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(u32 bar, u32 bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(u32 bar, u32 parity) {
  u32 ok;
  asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
               : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
// Bounded wait: false (and the error word set) if the barrier phase never completes, or the word is set already.
__device__ __forceinline__ bool mbar_wait(u32 bar, u32 parity, u32* err, u32 code) {
  if (mbar_try(bar, parity)) return true;
  const u64 t0 = now_ns();
  for (u32 it = 0;; ++it) {
    if (mbar_try(bar, parity)) return true;
    if ((it & 255) == 0 && (now_ns() - t0 > WAIT_NS || (err && *(volatile u32*)err))) {
      if (err) atomicCAS(err, 0u, code);
      return false;
    }
  }
}

// The CTA's barrier before it gives up its shared and tensor memory.  Where one of its waits gave up, copies and
// products of its own may still be in flight: 1 ms, they take microseconds, and they have ended.
__device__ __forceinline__ void sync_settled(bool gave_up) {
  if (__syncthreads_or(gave_up))
    for (const u64 t0 = now_ns(); now_ns() - t0 < 1000000u;) { }
}

// Shared -> global tensor store of one box (rows outside the tensor are not written); completion is
// tracked per thread in bulk groups.
__device__ __forceinline__ void tma_store_3d(const TmaDesc* map, u32 src, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];"
               :: "l"(reinterpret_cast<u64>(map)), "r"(src), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// wait until at most one committed group still has to read its shared-memory source
__device__ __forceinline__ void bulk_wait_read1() { asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

__device__ __forceinline__ void tma_load_3d(u32 dst, const TmaDesc* map, u32 bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      :: "r"(dst), "l"(reinterpret_cast<u64>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
}

__device__ __forceinline__ void mma_commit(u32 bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(bar) : "memory");
}
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tmem_ld16(u32 taddr, float (&r)[16]) {
  u32 v[16];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                 "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
               : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int j = 0; j < 16; ++j) r[j] = __uint_as_float(v[j]);
}

}  // namespace tcb
