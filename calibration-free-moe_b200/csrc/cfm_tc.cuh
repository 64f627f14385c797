// Barriers, bulk copies and tensor memory of the tcgen05 kernels (sm_100a).
#pragma once

#include "cfm_device.cuh"

// How long a wait goes on, how long, once one has run out, those for what is still in flight do, in
// nanoseconds, and how they ask.  (A build for tests has short waits run out.)
#ifndef CFM_SCREEN_WAIT_NS
#define CFM_SCREEN_WAIT_NS 1000000000u
#define CFM_SCREEN_DRAIN_NS 1000000000u
#define CFM_SCREEN_WAIT "try_wait"
#endif

namespace cfm {
namespace tc {

// By the threads with `leader` set.
__device__ __forceinline__ void barrier_arrive(uint32_t bar, int leader) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.s32 p, %1, 0;\n\t"
      "@p mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}" ::"r"(bar),
      "r"(leader)
      : "memory");
}

__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}

// `bytes` (a multiple of 16) from global to shared memory, both on 16-byte boundaries; arrives at
// the barrier.
__device__ __forceinline__ void copy_bulk(uint32_t shared, const void* global, uint32_t bytes,
                                          uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(shared),
               "l"(global), "r"(bytes), "r"(bar)
               : "memory");
}

__device__ __forceinline__ void barrier_init(uint32_t bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}

// Waits for the phase with the given parity, `limit` nanoseconds at most: then the word at `abort` is set.
// A thread that gives up, because its time ran out or another thread's has, clears `alive`; a phase that
// is complete counts all the same.  (One try suspends for up to 4 us.)
__device__ __forceinline__ void barrier_wait(uint32_t bar, uint32_t parity, uint32_t abort, int& alive,
                                             uint32_t limit = CFM_SCREEN_WAIT_NS) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .u32 start, now;\n\t"
      "mbarrier." CFM_SCREEN_WAIT ".parity.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra done;\n\t"
      "mov.u32 start, %%globaltimer_lo;\n"
      "again:\n\t"
      "ld.volatile.shared.u32 now, [%3];\n\t"
      "setp.ne.u32 p, now, 0;\n\t"
      "@p bra gone;\n\t"
      "mbarrier." CFM_SCREEN_WAIT ".parity.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra done;\n\t"
      "mov.u32 now, %%globaltimer_lo;\n\t"
      "sub.u32 now, now, start;\n\t"
      "setp.lt.u32 p, now, %4;\n\t"
      "@p bra again;\n\t"
      "st.volatile.shared.u32 [%3], 1;\n"
      "gone:\n\t"
      "mov.u32 %0, 0;\n"
      "done:\n\t}"
      : "+r"(alive)
      : "r"(bar), "r"(parity), "r"(abort), "r"(limit)
      : "memory");
}

// The same for the end of a product, whose rows and sums the thread is about to touch: having given up it
// goes on waiting, until the word at `late` is set or, after CFM_SCREEN_DRAIN_NS, sets that.  (By then no driver
// issues a product any more.  A vote of the warp before it goes on, instead, cost 2 us of 55.)
__device__ __forceinline__ void barrier_wait_product(uint32_t bar, uint32_t parity, uint32_t abort, uint32_t late,
                                                     int& alive) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .u32 start, now;\n\t"
      "mbarrier." CFM_SCREEN_WAIT ".parity.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra done;\n\t"
      "mov.u32 start, %%globaltimer_lo;\n"
      "again:\n\t"
      "ld.volatile.shared.u32 now, [%3];\n\t"
      "setp.ne.u32 p, now, 0;\n\t"
      "@p bra gone;\n\t"
      "mbarrier." CFM_SCREEN_WAIT ".parity.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra done;\n\t"
      "mov.u32 now, %%globaltimer_lo;\n\t"
      "sub.u32 now, now, start;\n\t"
      "setp.lt.u32 p, now, %5;\n\t"
      "@p bra again;\n\t"
      "st.volatile.shared.u32 [%3], 1;\n"
      "gone:\n\t"
      "mov.u32 %0, 0;\n\t"
      "mov.u32 start, %%globaltimer_lo;\n"
      "drain:\n\t"
      "mbarrier." CFM_SCREEN_WAIT ".parity.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra done;\n\t"
      "ld.volatile.shared.u32 now, [%4];\n\t"
      "setp.ne.u32 p, now, 0;\n\t"
      "@p bra done;\n\t"
      "mov.u32 now, %%globaltimer_lo;\n\t"
      "sub.u32 now, now, start;\n\t"
      "setp.lt.u32 p, now, %6;\n\t"
      "@p bra drain;\n\t"
      "st.volatile.shared.u32 [%4], 1;\n"
      "done:\n\t}"
      : "+r"(alive)
      : "r"(bar), "r"(parity), "r"(abort), "r"(late), "r"(static_cast<uint32_t>(CFM_SCREEN_WAIT_NS)),
        "r"(CFM_SCREEN_DRAIN_NS)
      : "memory");
}

// One lane of the warp, known to the compiler as one (instructions of a single thread then need no
// search for the active lane).
__device__ __forceinline__ bool elect_lane() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}

__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
               : "memory");
}

// Accumulators of this thread's row, complete once load_wait() has returned.
__device__ __forceinline__ void load_columns16(uint32_t address, int* c) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3]), "=r"(c[4]), "=r"(c[5]), "=r"(c[6]),
        "=r"(c[7]), "=r"(c[8]), "=r"(c[9]), "=r"(c[10]), "=r"(c[11]), "=r"(c[12]), "=r"(c[13]),
        "=r"(c[14]), "=r"(c[15])
      : "r"(address)
      : "memory");
}
__device__ __forceinline__ void load_columns8(uint32_t address, int* c) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
      : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3]), "=r"(c[4]), "=r"(c[5]), "=r"(c[6]),
        "=r"(c[7])
      : "r"(address)
      : "memory");
}
__device__ __forceinline__ void load_wait() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

}  // namespace tc
}  // namespace cfm
