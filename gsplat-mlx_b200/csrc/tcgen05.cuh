// The few tcgen05, TMA and mbarrier instructions that the grouped products use, and
// the formats of their descriptors (PTX ISA, "tcgen05" and "matrix
// descriptors").  Operands lie in shared memory K-major with the 128-byte
// swizzle: row r of a panel is 128 bytes at r * 128, its 16-byte chunk c at
// (c ^ (r & 7)) * 16; panels start on 1024 bytes.
#pragma once

#include <stdint.h>

namespace gsb {
namespace tc {

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// Shared-memory descriptor: start and stride (8 rows = 1024 bytes) in units
// of 16 bytes, version 1, swizzle mode 2 (128 bytes).  A step along K inside
// the 128-byte row adds its bytes to the start.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFF) | (uint64_t(1) << 16) |
         (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}

// The same panel as an operand whose rows are the depth (MN-major): 64
// columns of 16-bit values to a row, the next 64 `blocks` bytes on, 8 rows to
// 1024 bytes.  A step of 16 rows adds 2048 to the start.
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t addr, uint32_t blocks) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFF) | (uint64_t(blocks >> 4) << 16) |
         (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}

enum Format : uint32_t { kF16 = 0, kBF16 = 1, kTF32 = 2 };

// Instruction descriptor: fp32 accumulators, A and B of one format, both
// K-major unless the flags say MN-major, M = 128 lanes, N columns (a multiple
// of 16).
constexpr uint32_t kMnMajorA = 1u << 15, kMnMajorB = 1u << 16;
__device__ __forceinline__ uint32_t instr_desc(uint32_t format, uint32_t n) {
  return (1u << 4) | (format << 7) | (format << 10) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

// One lane of the (converged) warp.  The whole warp runs the issuing code and
// only the instructions themselves are predicated: with a branch around it
// the descriptors, which the instruction takes from uniform registers, are
// moved there one by one, which took longer than the multiplication.
__device__ __forceinline__ uint32_t elected() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}"
               : "=r"(p));
  return p;
}

template <bool TF32>
__device__ __forceinline__ void mma(uint32_t leader, uint32_t d, uint64_t a, uint64_t b,
                                    uint32_t idesc, bool accumulate) {
  const uint32_t acc = accumulate;
  if (TF32)
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::tf32 [%0], %1, %2, %3, p;\n}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(leader) : "memory");
  else
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(leader) : "memory");
}

// Arrives on the barrier once every MMA that the leader issued is done.
__device__ __forceinline__ void commit(uint32_t leader, uint32_t bar) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}"
      ::"r"(bar), "r"(leader) : "memory");
}

__device__ __forceinline__ void fence_before_sync() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after_sync() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// Generic writes to shared memory become visible to the tensor core.
__device__ __forceinline__ void fence_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// One warp; columns a power of two from 32 to 512.
__device__ __forceinline__ void alloc(uint32_t* smem_slot, uint32_t columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
               ::"r"(smem_addr(smem_slot)), "r"(columns) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void dealloc(uint32_t tmem, uint32_t columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns)
               : "memory");
}

// 16 columns of the warp's 32 lanes: thread l gets lane l's.  The wait is in
// the same statement, so that no use of the values can move in front of it.
__device__ __forceinline__ void load16(uint32_t taddr, float (&v)[16]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr) : "memory");
}

__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_init_done() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Arrives when the asynchronous copies that this thread has sent are there.
__device__ __forceinline__ void arrive_copied(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
// Arrives, and has the phase wait for `bytes` of bulk copies.
__device__ __forceinline__ void expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}
// A box of a 2-D tensor map, from (x, row) on, to shared memory.
__device__ __forceinline__ void load_box(uint32_t to, const void* map, int x, int row,
                                         uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];"
      ::"r"(to), "l"(map), "r"(x), "r"(row), "r"(bar) : "memory");
}
// Four rows of a map whose box is one row high, from column x on, one behind
// the other; a row outside the map reads as zeros.
__device__ __forceinline__ void load_rows4(uint32_t to, const void* map, int x, const int (&row)[4],
                                           uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
      ::"r"(to), "l"(map), "r"(x), "r"(row[0]), "r"(row[1]), "r"(row[2]), "r"(row[3]), "r"(bar)
      : "memory");
}
// A barrier of `threads` of the CTA's threads.
__device__ __forceinline__ void bar_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// A whole warp waits for the phase to end, for a poll and up to `limit` more, which
// are the hardware's own waits (4 us each on a B200, whatever the hint), and not past
// the first one behind which *stop (where given) is set; false, for every lane, when
// it gave up.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, uint32_t limit,
                                         const volatile uint32_t* stop) {
  while (true) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n"
        " mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(done) : "r"(bar), "r"(parity), "r"(20000u) : "memory");
    if (__all_sync(0xffffffffu, done)) return true;
    if (limit-- == 0 || __any_sync(0xffffffffu, stop && *stop)) return false;
  }
}

}  // namespace tc
}  // namespace gsb
