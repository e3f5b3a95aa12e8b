// The few PTX instructions of the 5th-generation tensor cores that this library uses: tensor memory
// allocation, matrix products from shared-memory descriptors, commits to mbarriers, loads of accumulators.
#pragma once
#include "common.cuh"

namespace nb200 {
namespace tc {

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// ---- mbarriers; every wait is bounded -----------------------------------------------------------------
constexpr long long kWaitCycles = 4000000000LL;      // about two seconds: a wait that long means a mistake, not load

__device__ __forceinline__ void mbar_init(uint64_t* bar, unsigned count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.shared::cta.b64 st, [%0];\n\t}" :: "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t addr, unsigned parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(addr), "r"(parity) : "memory");
    return ok != 0;
}
// False when the wait ran out, or when another warp's has (`gave_up`): the caller leaves its loop.
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, unsigned parity, volatile int* gave_up) {
    const uint32_t addr = smem_u32(bar);
    if (mbar_try(addr, parity)) return true;
    const long long t0 = clock64();
    while (!mbar_try(addr, parity))
        if (*gave_up || clock64() - t0 > kWaitCycles) {
            *gave_up = 1;
            return false;
        }
    return true;
}

// The same for a whole warp, which leaves together: a lane that was let through would go on to instructions that the
// warp has to run as one.
__device__ __forceinline__ bool mbar_wait_warp(uint64_t* bar, unsigned parity, volatile int* gave_up) {
    return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, gave_up));
}

// ---- tensor memory ------------------------------------------------------------------------------------
// Whole warp; `columns` a power of two, 32..512.
__device__ __forceinline__ void tmem_alloc(uint32_t* where, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(where)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t base, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(base), "r"(columns));
}
// 16 consecutive columns of the warp's 32 lanes: thread l receives lane l's.  The values are there after tmem_wait.
__device__ __forceinline__ void tmem_load16(uint32_t addr, float (&v)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
                   "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
                 : "r"(addr));
}
// Ties the loaded values to the wait, so that no use of them moves in front of it.
__device__ __forceinline__ void tmem_wait16(float* v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]),
                   "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]) :: "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const float (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 :: "r"(addr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]),
                    "f"(v[9]), "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]) : "memory");
}
__device__ __forceinline__ void tmem_stores_done() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Shared memory written by this thread becomes visible to the tensor cores and bulk copies.
__device__ __forceinline__ void fence_smem_for_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---- operands in shared memory ------------------------------------------------------------------------
// Both layouts are made of 1024-byte atoms of eight 128-byte lines, 16-byte unit u of line l stored at unit u ^ l.
// K-major: a line is one row's 64 values along the sum; atoms follow one another every eight rows, 1024 bytes.
// MN-major: a line is one sum index's 64 rows; the next eight sum indices are 1024 bytes further, the next 64
// rows `block` bytes further.
__device__ __forceinline__ uint64_t smem_descriptor(uint32_t addr, uint32_t leading_bytes, uint32_t stride_bytes) {
    return static_cast<uint64_t>((addr >> 4) & 0x3FFF) | static_cast<uint64_t>((leading_bytes >> 4) & 0x3FFF) << 16 |
           static_cast<uint64_t>((stride_bytes >> 4) & 0x3FFF) << 32 | uint64_t(1) << 46 /* version */ |
           uint64_t(2) << 61 /* 128-byte swizzle */;
}
// kind::f16 with float accumulators, M = 128.
__host__ __device__ constexpr uint32_t instruction_descriptor(bool bf16, bool a_mn_major, bool b_mn_major, int n) {
    return 1u << 4 | (bf16 ? 1u : 0u) << 7 | (bf16 ? 1u : 0u) << 10 | (a_mn_major ? 1u : 0u) << 15 | (b_mn_major ? 1u : 0u) << 16 |
           static_cast<uint32_t>(n / 8) << 17 | (128u / 16) << 24;
}
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u) : "memory");
}
// Arrives on `bar` when all products issued so far by this thread are done.
__device__ __forceinline__ void commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(smem_u32(bar)) : "memory");
}

// ---- tiled bulk copies (TMA) ------------------------------------------------------------------------------
__device__ __forceinline__ void mbar_expect(uint64_t* bar, uint32_t bytes) {
    asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}"
                 :: "r"(smem_u32(bar)), "r"(bytes) : "memory");
}
// The box at element (x, y); x a multiple of 16 bytes.
__device__ __forceinline__ void tile_load(uint32_t dst, const void* map, int x, int y, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar)) : "memory");
}

// A box from shared memory to element (x, y, z); what lies outside the array is not written.  Groups of stores are
// counted per thread.
__device__ __forceinline__ void tile_store(const void* map, int x, int y, int z, uint32_t src) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];"
                 :: "l"(map), "r"(x), "r"(y), "r"(z), "r"(src) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// The thread's stores have read their shared memory / are done.
__device__ __forceinline__ void stores_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void stores_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
// The same box into L2 only.
__device__ __forceinline__ void tile_prefetch(const void* map, int x, int y) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" :: "l"(map), "r"(x), "r"(y) : "memory");
}

// ---- registers: moved between warpgroups; the sum after all moves must not exceed the sum at launch ---------
template <int N> __device__ __forceinline__ void registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(N)); }
template <int N> __device__ __forceinline__ void registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(N)); }

}  // namespace tc
}  // namespace nb200
