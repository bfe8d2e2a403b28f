// The sm_100a tensor cores (tcgen05) for bf16 operands with fp32 accumulators in tensor memory, and tiled bulk copies that leave
// their operands in the 128-byte swizzle.
//
// An operand tile in shared memory is a column of boxes: 64 bf16 (128 bytes) a row, rows one behind the other, each group of 8 rows
// (1024 bytes, aligned) swizzled: the 16-byte piece p of row r sits at piece p ^ (r & 7).  A tiled copy with the 128-byte swizzle
// writes it so.  The same tile serves as an operand whose contracted index runs along the rows' columns ("by columns", K-major: rows
// are M or N) or along the rows ("by rows", MN-major: columns are M or N).
//
// Rules kept by every user: one thread (the elected lane of one warp) issues the products and their commits; A and B are both bf16; waits are bounded.
#ifndef ACRO_B200_KERNELS_UMMA_CUH
#define ACRO_B200_KERNELS_UMMA_CUH

#include <cstdint>
#include <cuda.h>
#include "tma.cuh"
#include "tmem.cuh"

namespace acro_b200_detail
{

constexpr uint32_t kBoxColumns = 64;        // bf16 of one row of a box

// Shared-memory operand descriptor: address, leading and stride byte offsets in units of 16 bytes, version 1, 128-byte swizzle.
// By columns: stride = distance of 8-row groups; the leading offset is not used.  By rows: stride = distance of 8-row groups along the
// contracted index, leading = distance of boxes along M or N.
__device__ __forceinline__ uint64_t umma_operand(uint32_t address, uint32_t leading, uint32_t stride)
{
    return static_cast<uint64_t>((address & 0x3ffffu) >> 4) | static_cast<uint64_t>(leading >> 4) << 16 | static_cast<uint64_t>(stride >> 4) << 32 |
           1ull << 46 | 2ull << 61;
}

// Instruction descriptor: fp32 accumulators, bf16 operands, M = 128, N columns; by_rows as above.
__host__ __device__ constexpr uint32_t umma_shape(int n, bool a_by_rows, bool b_by_rows)
{
    return 1u << 4 | 1u << 7 | 1u << 10 | static_cast<uint32_t>(a_by_rows) << 15 | static_cast<uint32_t>(b_by_rows) << 16 |
           static_cast<uint32_t>(n >> 3) << 17 | static_cast<uint32_t>(128 >> 4) << 24;
}

// One in one lane of a converged warp (the leader below), zero in the others.
__device__ __forceinline__ uint32_t elect_lane()
{
    uint32_t one;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "elect.sync _|p, 0xffffffff;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(one)
        :
        : "memory");
    return one;
}

// D[128 lanes][n columns] (+)= A (16 columns) * B, A and B in shared memory; executed by the leader, walked through by its whole warp.
__device__ __forceinline__ void umma(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t shape, bool add)
{
    asm volatile(
        "{\n"
        ".reg .pred p, q;\n"
        "setp.ne.u32 p, %4, 0;\n"
        "setp.ne.u32 q, %5, 0;\n"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(d), "l"(a), "l"(b), "r"(shape), "r"(static_cast<uint32_t>(add)), "r"(leader)
        : "memory");
}

// The same with A in tensor memory: lane = row of A, a 32-bit column holds two neighbouring entries of the contracted index.
__device__ __forceinline__ void umma_tmem(uint32_t leader, uint32_t d, uint32_t a, uint64_t b, uint32_t shape, bool add)
{
    asm volatile(
        "{\n"
        ".reg .pred p, q;\n"
        "setp.ne.u32 p, %4, 0;\n"
        "setp.ne.u32 q, %5, 0;\n"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
        "}\n" ::"r"(d), "r"(a), "l"(b), "r"(shape), "r"(static_cast<uint32_t>(add)), "r"(leader)
        : "memory");
}

// One arrival on `bar` when every product the leader has issued so far is complete.
__device__ __forceinline__ void umma_commit(uint32_t leader, uint64_t *bar)
{
    asm volatile(
        "{\n"
        ".reg .pred q;\n"
        "setp.ne.u32 q, %1, 0;\n"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n"
        "}\n" ::"r"(smem_addr(bar)), "r"(leader)
        : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint64_t *bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// mbar_wait for warps that wait for much of their time: a try may suspend the thread for up to a millisecond, so that the waiting
// warps leave the issue slots to the others.  Bounded like mbar_wait (about a second).
__device__ __forceinline__ bool mbar_wait_asleep(uint64_t *bar, uint32_t parity)
{
    if (mbar_try_wait(bar, parity)) return true;
    const long long start = clock64();
    do
    {
        uint32_t done;
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n"
            "selp.u32 %0, 1, 0, p;\n"
            "}\n"
            : "=r"(done)
            : "r"(smem_addr(bar)), "r"(parity), "r"(1000000u)
            : "memory");
        if (done) return true;
    } while (clock64() - start < kMbarWaitLimitCycles);
    return false;
}

// One box of a four-dimensional array (column, head, token, sequence).
__device__ __forceinline__ void box_load(void *smem, const CUtensorMap *map, int column, int head, int token, int sequence, uint64_t *bar)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_addr(smem)),
                 "l"(map), "r"(column), "r"(head), "r"(token), "r"(sequence), "r"(smem_addr(bar))
                 : "memory");
}

// 16 columns of this thread's lane.  The wait is part of the statement, so that no use of the registers can move in front of it.
__device__ __forceinline__ void tmem_load_16(uint32_t addr, uint32_t (&r)[16])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                   "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr)
                 : "memory");
}

// 8 columns of this thread's lane.
__device__ __forceinline__ void tmem_load_8(uint32_t addr, uint32_t (&r)[8])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(addr)
                 : "memory");
}

// 8 columns of this thread's lane.
__device__ __forceinline__ void tmem_store_8(uint32_t addr, const uint32_t (&r)[8])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
                 "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

}

#endif
