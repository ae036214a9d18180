// tcgen05.cuh — inline PTX for the 5th-generation tensor cores, tensor memory
// and TMA as the e4m3 products use them (sm_100a).
#pragma once
#include "sync.cuh"

#include <cuda.h>        // CUtensorMap

__device__ __forceinline__ void t5_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void t5_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Descriptor of a K-major operand in shared memory with the 128-byte swizzle:
// rows of 128 bytes, groups of 8 rows 1024 bytes apart.  The upper word does not
// depend on the address; 32 bytes further along K is 2 more in the lower.
#define T5_DESC_HI ((1u << 14) | (2u << 29) | (1024u >> 4))
__device__ __forceinline__ uint32_t t5_desc_lo(uint32_t saddr) { return ((saddr >> 4) & 0x3FFFu) | 1u << 16; }

// Instruction descriptor of kind::f8f6f4: f32 accumulators, e4m3 operands, both K-major.
__host__ __device__ constexpr uint32_t t5_idesc_e4m3(int m, int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// D = A . B^T (ACC: D += A . B^T) over 32 e4m3 values of K; one thread issues it.
// da, db: lower words of the descriptors.
template <bool ACC>
__device__ __forceinline__ void t5_mma_e4m3(uint32_t d, uint32_t da, uint32_t db, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %3, p;\n\t}\n" ::"r"(d),
        "r"(da), "r"(db), "r"(idesc), "n"((int)ACC), "n"(T5_DESC_HI)
        : "memory");
}

// Arrives on `bar` once every product this thread issued so far has completed.
__device__ __forceinline__ void t5_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}

// Tensor memory of one CTA: a power of two of columns, at least 32.
__device__ __forceinline__ void t5_alloc(uint32_t *slot, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void t5_dealloc(uint32_t tmem, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
}

// 8 / 16 / 32 consecutive columns of this thread's tensor-memory lane.  The
// values are there after t5_wait_ld().
__device__ __forceinline__ void t5_ld(uint32_t t, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(t));
}
__device__ __forceinline__ void t5_ld(uint32_t t, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(t));
}
__device__ __forceinline__ void t5_ld(uint32_t t, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(t));
}
// Waits for this thread's tensor-memory loads.  The registers pass through, so
// that no use of them is moved above the wait.
template <int N>
__device__ __forceinline__ void t5_wait_ld(uint32_t (&r)[N]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; i++) asm volatile("" : "+r"(r[i]));
}

// TMA copy of one box at (x, y) of `map` into shared memory, completing in
// bytes on `bar`.  x times the element size is a multiple of 16.
__device__ __forceinline__ void t5_tma_2d(void *dst, const CUtensorMap *map, int x, int y, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::
            "r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
        : "memory");
}
// TMA copy of one box from shared memory to (x, y) of `map` (what lies past the
// tensor is not written): after t5_fence_proxy() by the threads that wrote the
// box; commit closes a group of the issuing thread's copies (an empty one too), and
// the waits are for all but the last PENDING groups to have read their boxes, or
// for all to be done.
__device__ __forceinline__ void t5_tma_store_2d(const CUtensorMap *map, int x, int y, const void *src) {
    asm volatile(
        "cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
            reinterpret_cast<uint64_t>(map)),
        "r"(smem_u32(src)), "r"(x), "r"(y)
        : "memory");
}
__device__ __forceinline__ void t5_tma_store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void t5_fence_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void t5_tma_store_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(PENDING) : "memory"); }
__device__ __forceinline__ void t5_tma_store_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

__device__ __forceinline__ void t5_prefetch_map(const CUtensorMap *map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

// Cluster: the address of shared offset `saddr` in CTA `rank`, a store to it, and
// the barrier over all threads of the cluster.
__device__ __forceinline__ uint32_t t5_cluster_addr(uint32_t saddr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}
__device__ __forceinline__ void t5_cluster_st(uint32_t a, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory");
}
__device__ __forceinline__ void t5_cluster_arrive_all() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void t5_cluster_wait_all() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void t5_cluster_sync() {
    t5_cluster_arrive_all();
    t5_cluster_wait_all();
}

// ---- two CTAs of a cluster on one product (cta_group::2) ----
// Rank 0 issues the products: A's and D's rows and B's rows are split between
// the CTAs (each holds half of them at the same shared-memory offsets).
__device__ __forceinline__ uint32_t t5_cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
template <bool ACC>
__device__ __forceinline__ void t5_mma2_e4m3(uint32_t d, uint32_t da, uint32_t db, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a, b, %3, p;\n\t}\n" ::"r"(d),
        "r"(da), "r"(db), "r"(idesc), "n"((int)ACC), "n"(T5_DESC_HI)
        : "memory");
}
// As t5_commit, on the barrier at this offset in both CTAs.
__device__ __forceinline__ void t5_commit2(uint64_t *bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
}
__device__ __forceinline__ void t5_alloc2(uint32_t *slot, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void t5_dealloc2(uint32_t tmem, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
}
// As t5_tma_2d into this CTA, completing on a barrier of either CTA, given by
// its cluster address.
__device__ __forceinline__ void t5_tma2_2d(void *dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
        "[%4];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
// Arrives on a barrier given by its cluster address.  Relaxed: what the arrival
// orders is tensor memory, by the tcgen05 fences around it and the wait for the
// loads before it; a release at cluster scope waits for every outstanding access
// of the thread, ~1000 clocks beside loads from global memory.
__device__ __forceinline__ void t5_cluster_arrive(uint32_t bar, bool who) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %1, 0;\n\t"
        "@p mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n\t}" ::"r"(bar),
        "r"((uint32_t)who)
        : "memory");
}

// Arrives on a barrier of this CTA from one thread of a warp, without a branch
// that would part the warp.
__device__ __forceinline__ void t5_arrive(uint64_t *bar, bool who) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 st;\n\tsetp.ne.b32 p, %1, 0;\n\t"
        "@p mbarrier.arrive.shared::cta.b64 st, [%0];\n\t}" ::"r"(smem_u32(bar)),
        "r"((uint32_t)who)
        : "memory");
}

// Registers of the calling warpgroup, out of those the block was launched with.
template <int R>
__device__ __forceinline__ void t5_regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R)); }
template <int R>
__device__ __forceinline__ void t5_regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R)); }

// Two f32 in one register pair; d = a * b + c on both.
__device__ __forceinline__ uint64_t t5_pair(uint32_t lo, uint32_t hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
    return r;
}
__device__ __forceinline__ void t5_unpair(uint64_t v, float &lo, float &hi) {
    uint32_t a, b;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(v));
    lo = __uint_as_float(a);
    hi = __uint_as_float(b);
}
__device__ __forceinline__ uint64_t t5_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
