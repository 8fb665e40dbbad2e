// Fifth-generation tensor cores for the delta rule kernels: bounded mbarrier waits, tensor memory, operand descriptors.
//
// Operand tiles in shared memory are blocks of rows of 128 bytes (64 bf16) with the 128-byte swizzle: piece p of row r lies at piece
// p ^ (r & 7), a block starts at a multiple of 1024 bytes.  One and the same tile serves both ways round: with the contraction
// along its rows (K-major; the next sixteen are 32 bytes further, the next eight rows 1024) and with the contraction across them
// (MN-major; the next sixteen are 2048 bytes further, the next 64 of the other index one block further).
#pragma once
#include <cuda.h>

#include "dism_common.cuh"

namespace dism {

// Every wait is bounded, by about a second.  When one runs out, `abort` is set, the code is recorded and every later wait of the CTA
// returns at once: no copy or product is issued any more, those in flight are waited for (tm_settle), the other roles run to their ends
// and write NaN, tensor memory is freed.  Whoever has passed a wait of the CTA after another role gave up sees `abort` set.
constexpr unsigned TM_WAIT_TRIES = 1u << 16, TM_PARK_NANOSECONDS = 20000;

__device__ __forceinline__ uint32_t tm_address(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void tm_barrier_init(uint64_t* bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(tm_address(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void tm_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(tm_address(bar)) : "memory");
}
// The hardware may park the warp for a while: a polling warp takes issue slots from the working ones.
__device__ __forceinline__ bool tm_test_parked(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{.reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3; selp.u32 %0, 1, 0, p;}"
                 : "=r"(done) : "r"(tm_address(bar)), "r"(parity), "r"(TM_PARK_NANOSECONDS) : "memory");
    return done != 0;
}
// False: this wait ran out or another role's did.
__device__ __forceinline__ bool tm_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int* fault, int code, unsigned limit) {
    for (unsigned tries = 0; tries < limit; ++tries) {
        if (tm_test_parked(bar, parity)) return true;
        if (*abort) return false;
    }
    *abort = 1;
    atomicCAS(fault, 0, code);
    return false;
}
// What the role itself has in flight lands before its memory is given back: bounded like any wait, whatever has happened.
__device__ __forceinline__ void tm_settle(uint64_t* bar, uint32_t parity) {
    for (unsigned tries = 0; tries < TM_WAIT_TRIES; ++tries)
        if (tm_test_parked(bar, parity)) return;
}

// Contiguous bytes (a multiple of 16, both addresses 16-byte aligned) into shared memory; the barrier counts them.
__device__ __forceinline__ void tm_expect(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(tm_address(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tm_copy(uint32_t to, const void* from, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(to), "l"(from), "r"(bytes), "r"(tm_address(bar)) : "memory");
}
// A box of a tensor map, by its first column and row.
__device__ __forceinline__ void tm_load_box(uint32_t to, const CUtensorMap* map, int column, int row, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(to), "l"(map), "r"(column), "r"(row), "r"(tm_address(bar)) : "memory");
}
// Tensor map of a bf16 matrix [rows, columns] (row stride in elements) in boxes of 64 columns by box_rows rows, 128-byte swizzle
// (labels_tcgen05.cu).  False: the driver has no such entry point or refuses the shape.
bool encode_rows(CUtensorMap* map, const void* data, uint64_t rows, uint64_t columns, uint64_t row_stride, int box_rows);
__device__ __forceinline__ bool tm_elect() {  // one lane of a converged warp
    uint32_t elected;
    asm volatile("{.reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p;}" : "=r"(elected));
    return elected != 0;
}
__device__ __forceinline__ void tm_allocate(uint32_t* to, uint32_t columns) {  // one whole warp
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tm_address(to)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tm_free(uint32_t at, uint32_t columns) {  // the same warp
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns) : "memory");
}
__device__ __forceinline__ void tm_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_fence_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(tm_address(bar)) : "memory");
}

// Redistribution of a CTA's registers: every warp of four consecutive ones, counts from the launch's own share.
template <int COUNT>
__device__ __forceinline__ void tm_more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(COUNT)); }
template <int COUNT>
__device__ __forceinline__ void tm_fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(COUNT)); }

// Lane = row, register i = column i; the warp's 32 lanes are rows 32 (warp % 4) .. of the tile.
__device__ __forceinline__ void tm_load16(float (&v)[16], uint32_t at) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
                   "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]) : "r"(at) : "memory");
}

// Descriptors of swizzled tiles; `across` is the distance in bytes between blocks of 64 of the index that is not contracted (MN-major).
__device__ __forceinline__ uint64_t tm_descriptor(uint32_t address, uint32_t across = 16) {
    return uint64_t((address & 0x3ffff) >> 4) | (uint64_t(across >> 4) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
// The same for tiles of 8 x 8 blocks of 128 contiguous bytes, a block's rows along the contraction (MN-major, no swizzle): distances
// between blocks along the other index and along the contraction.
__device__ __forceinline__ uint64_t tm_block_descriptor(uint32_t address, uint32_t other, uint32_t contracted) {
    return uint64_t((address & 0x3ffff) >> 4) | (uint64_t(contracted >> 4) << 16) | (uint64_t(other >> 4) << 32) | (uint64_t(1) << 46);
}
// bf16 x bf16 -> f32 with M = 128 rows and `columns` columns
__host__ __device__ constexpr uint32_t tm_instruction(int columns, bool a_across, bool b_across) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (a_across ? 1u << 15 : 0u) | (b_across ? 1u << 16 : 0u) | (uint32_t(columns >> 3) << 17) | (uint32_t(128 >> 4) << 24);
}
__device__ __forceinline__ void tm_mma_shared(uint32_t accumulator, uint64_t a, uint64_t b, uint32_t instruction, bool accumulate) {
    asm volatile("{.reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;}"
                 ::"r"(accumulator), "l"(a), "l"(b), "r"(instruction), "r"(uint32_t(accumulate)) : "memory");
}

}  // namespace dism
