// tensor_core.cuh — sm_100a building blocks of products on the 5th-generation tensor cores: bulk copies into
// shared memory, mbarriers, tensor memory, and the descriptors of tcgen05.mma on 128-byte swizzled operands.
#pragma once

#include <stdint.h>

namespace arcqml {
namespace tc {

__device__ __forceinline__ uint32_t shared_address(const void *p) { return uint32_t(__cvta_generic_to_shared(p)); }

// ------------------------------------------------------------------ mbarriers

__device__ __forceinline__ void barrier_init(uint64_t *b, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(shared_address(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint64_t *b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(shared_address(b)), "r"(bytes) : "memory");
}
// The address of `b` in the cluster's block `rank`.
__device__ __forceinline__ uint32_t in_block(const void *b, uint32_t rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(shared_address(b)), "r"(rank));
    return at;
}
// Barriers of a pair of blocks (CG = 2) are arrived at by one block and waited for by the other, which orders what
// the two have done only in the scope of their cluster. What an arrival releases lies in its own block's shared
// memory (operands that copies have brought) or in tensor memory (ordered by fence_before): a fence of
// shared memory alone is enough, and one of everything costs some 1000 cycles between a stage's arrival and its
// products (8 large bf16 matrices 11.1 ms with it in one warp, 8.4 in three, 8.0 as it is).
template <int CG> __device__ __forceinline__ void barrier_arrive_at(uint32_t cluster_address) {
    if constexpr (CG == 1)
        asm volatile("mbarrier.arrive.release.cta.shared::cluster.b64 _, [%0];" ::"r"(cluster_address) : "memory");
    else
        asm volatile("fence.release.sync_restrict::shared::cta.cluster;\n"
                     " mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_address)
                     : "memory");
}
template <int CG> __device__ __forceinline__ bool barrier_try(uint64_t *b, uint32_t parity) {
    uint32_t done;
    if constexpr (CG == 1)
        asm volatile("{\n .reg .pred p;\n"
                     " mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n"
                     " selp.u32 %0, 1, 0, p;\n}"
                     : "=r"(done)
                     : "r"(shared_address(b)), "r"(parity)
                     : "memory");
    else
        asm volatile("{\n .reg .pred p;\n"
                     " mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
                     " selp.u32 %0, 1, 0, p;\n}"
                     : "=r"(done)
                     : "r"(shared_address(b)), "r"(parity)
                     : "memory");
    return done != 0;
}
__device__ __forceinline__ void barrier_init_fence() {
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}

// ------------------------------------------------------------------ copies

// `bytes` (a multiple of 16) from global to this block's shared memory, both on 16 bytes; counted by `b`.
__device__ __forceinline__ void copy_in(void *to, const void *from, uint32_t bytes, uint64_t *b) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     shared_address(to)),
                 "l"(from), "r"(bytes), "r"(shared_address(b))
                 : "memory");
}

// ------------------------------------------------------------------ clusters

__device__ __forceinline__ uint32_t block_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ------------------------------------------------------------------ tensor memory

template <int CG> __device__ __forceinline__ void tmem_alloc(uint32_t *to, uint32_t columns) {
    if constexpr (CG == 1)
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_address(to)),
                     "r"(columns)
                     : "memory");
    else
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_address(to)),
                     "r"(columns)
                     : "memory");
}
template <int CG> __device__ __forceinline__ void tmem_free(uint32_t at, uint32_t columns) {
    if constexpr (CG == 1) {
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns));
    } else {
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns));
    }
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 columns of this warp's 32 lanes: thread i holds lane i.
__device__ __forceinline__ void tmem_load(float (&v)[32], uint32_t at) {
    uint32_t r[32];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
                 " tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(at)
                 : "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// 16 columns, added to v.
__device__ __forceinline__ void tmem_add(float *v, uint32_t at) {
    uint32_t r[16];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
                 " tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(at)
                 : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] += __uint_as_float(r[i]);
}

// The sum of 16 columns at two places.
__device__ __forceinline__ void tmem_load2(float (&v)[16], uint32_t at, uint32_t too) {
    uint32_t r[32];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%32];\n"
                 " tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                 "{%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%33];\n"
                 " tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(at), "r"(too)
                 : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]) + __uint_as_float(r[i + 16]);
}

// ------------------------------------------------------------------ tcgen05.mma

// Operands lie in atoms of 8 rows of 128 bytes (1024 bytes, aligned to them) whose 16-byte pieces are
// permuted by piece ^= row % 8.
//   by depth   a row holds 64 values of the product's depth for one of the operand's rows: atoms of 8 rows
//              follow each other; 16 steps of depth are 32 bytes on
//   by width   a row holds 64 of the operand's rows for one step of depth: 8 steps of depth an atom, the
//              next 64 rows `apart` bytes on; 16 steps of depth are 2048 bytes on
__device__ __forceinline__ uint64_t descriptor(uint32_t address, uint32_t apart) {
    constexpr uint64_t version = 1, swizzle_128 = 2;
    return uint64_t((address >> 4) & 0x3fff) | uint64_t((apart >> 4) & 0x3fff) << 16 | uint64_t(1024 >> 4) << 32 |
           version << 46 | swizzle_128 << 61;
}
// f16 operands, f32 sums; the right operand lies by depth or by width.
__host__ __device__ constexpr uint32_t instruction(uint32_t rows, uint32_t columns, bool right_by_width) {
    return 1u << 4 | (right_by_width ? 1u << 16 : 0u) | columns / 8 << 17 | rows / 16 << 24;
}

template <int CG>
__device__ __forceinline__ void mma(uint32_t sums, uint64_t left, uint64_t right, uint32_t instr, bool add) {
    if constexpr (CG == 1)
        asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                     " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(sums),
                     "l"(left), "l"(right), "r"(instr), "r"(uint32_t(add))
                     : "memory");
    else
        asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                     " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(sums),
                     "l"(left), "l"(right), "r"(instr), "r"(uint32_t(add))
                     : "memory");
}
// `b` (of both blocks of a pair) is told when the products issued so far are done.
template <int CG> __device__ __forceinline__ void commit(uint64_t *b) {
    if constexpr (CG == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                         shared_address(b))
                     : "memory");
    else
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                shared_address(b)),
            "h"(uint16_t(3))
            : "memory");
}

}  // namespace tc
}  // namespace arcqml
