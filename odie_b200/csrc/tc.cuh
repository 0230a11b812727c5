// Blackwell (sm_100a) tensor-core primitives: tcgen05 MMA with TMEM accumulators.
//
// Shared-memory operands use the canonical no-swizzle ("interleaved") layout of
// 8 x 16-byte core matrices.  A [rows x cols] fp16 matrix is stored "blocked":
//   byte(r, c) = ((c / 8) * (rows / 8) + r / 8) * 128 + (r % 8) * 16 + (c % 8) * 2
// Read with cols as K (K-major operand): LBO = (rows / 8) * 128, SBO = 128,
// K-step s starts 2 * s * LBO bytes further.  Read with cols as M/N and rows as
// K (MN-major operand): LBO = 128, SBO = (rows / 8) * 128, K-step s starts
// 256 * s bytes further.  Descriptor and instruction-descriptor bit layouts
// follow the PTX ISA (tcgen05 matrix / instruction descriptors).
#pragma once
#include "common.cuh"

namespace odie {
namespace tc {

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// Byte offset of element (r, c) of a blocked [rows x cols] fp16 matrix.
__host__ __device__ constexpr int blocked(int rows, int r, int c) {
    return ((c >> 3) * (rows >> 3) + (r >> 3)) * 128 + (r & 7) * 16 + (c & 7) * 2;
}

// Shared-memory matrix descriptor, no swizzle, version 1 (Blackwell).
__device__ __forceinline__ uint64_t sdesc(uint32_t address, uint32_t lbo, uint32_t sbo) {
    return uint64_t((address >> 4) & 0x3FFFu) | (uint64_t((lbo >> 4) & 0x3FFFu) << 16) |
           (uint64_t((sbo >> 4) & 0x3FFFu) << 32) | (uint64_t(1) << 46);
}
// K-major view of a blocked [rows x cols] matrix (K along cols), K-step s.
__device__ __forceinline__ uint64_t kmajor(uint32_t base, int rows, int s) {
    const uint32_t lbo = uint32_t(rows >> 3) * 128u;
    return sdesc(base + 2u * uint32_t(s) * lbo, lbo, 128u);
}
// MN-major view of a blocked [rows x cols] matrix (M/N along cols, K along rows), K-step s.
__device__ __forceinline__ uint64_t mnmajor(uint32_t base, int rows, int s) {
    return sdesc(base + 256u * uint32_t(s), 128u, uint32_t(rows >> 3) * 128u);
}

// Instruction descriptor of kind::f16: fp16 A and B, fp32 D.
__host__ __device__ constexpr uint32_t idesc(int M, int N, int a_mn_major, int b_mn_major) {
    return (1u << 4) | (uint32_t(a_mn_major) << 15) | (uint32_t(b_mn_major) << 16) | (uint32_t(N >> 3) << 17) |
           (uint32_t(M >> 4) << 24);
}

// Matrices in the 128-byte swizzled layout a TMA load with SWIZZLE_128B leaves: lines of 128 bytes (64 16-bit
// elements), 8 lines to a swizzle atom of 1024 bytes, atoms on 1024-byte boundaries.
// K-major (a line holds 64 values of K of one row): 8-row groups 1024 bytes apart; K-step s (16 values) starts
// 32 s bytes further.
// MN-major (a line holds 64 rows at one value of K): 8-value groups of K 1024 bytes apart, the next 64 rows `lbo`
// bytes further; K-step s starts 2048 s bytes further.
__device__ __forceinline__ uint64_t sdesc_swizzled(uint32_t address, uint32_t lbo) {
    return sdesc(address, lbo, 1024u) | (uint64_t(2) << 61);
}
// Instruction descriptor of kind::f16 with bf16 operands.
__host__ __device__ constexpr uint32_t idesc_bf16(int M, int N, int a_mn_major, int b_mn_major) {
    return idesc(M, N, a_mn_major, b_mn_major) | (1u << 7) | (1u << 10);
}

// D[tmem] (+)= A * B, issued by one thread; CG CTAs (a pair's leader issues for both).
template <int CG>
__device__ __forceinline__ void mma_group(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
    if constexpr (CG == 2)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
            "l"(a), "l"(b), "r"(id), "r"(accumulate));
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
            "l"(a), "l"(b), "r"(id), "r"(accumulate));
}

// Products of microscaled 4-bit rows (kind::mxf4nvf4): A and B hold e2m1 values, two to a byte, K-major, one scale for
// each BLOCK of them: 16 (unsigned e4m3 scales, four to a K-step of 64) or 32 (powers of two, e8m0, two to a K-step).
// The scales lie in TMEM, one byte each, the four of a row in a 32-bit column, rows 32 q + l of 128 in lane l (of every
// quarter of the lanes) and column q; with BLOCK 32 a column serves two K-steps, `second` the later one.
template <int BLOCK>
__host__ __device__ constexpr uint32_t idesc_scaled(int M, int N, int second) {
    return (uint32_t(second * 2) << 4) | (1u << 7) | (1u << 10) | (uint32_t(N >> 3) << 17) | (uint32_t(BLOCK == 32) << 23) |
           (uint32_t(M >> 4) << 24) | (uint32_t(second * 2) << 29);
}
template <int CG, int BLOCK>
__device__ __forceinline__ void mma_scaled(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t id, uint32_t scale_a, uint32_t scale_b,
                                           uint32_t accumulate) {
    if constexpr (CG == 2 && BLOCK == 16)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d_tmem),
            "l"(a), "l"(b), "r"(id), "r"(scale_a), "r"(scale_b), "r"(accumulate));
    else if constexpr (CG == 2)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d_tmem),
            "l"(a), "l"(b), "r"(id), "r"(scale_a), "r"(scale_b), "r"(accumulate));
    else if constexpr (BLOCK == 16)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d_tmem),
            "l"(a), "l"(b), "r"(id), "r"(scale_a), "r"(scale_b), "r"(accumulate));
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d_tmem),
            "l"(a), "l"(b), "r"(id), "r"(scale_a), "r"(scale_b), "r"(accumulate));
}
// 512 bytes of shared memory (of each CTA of the group its own), the scales of 128 rows, into four TMEM columns.  Runs
// before the products that the same thread issues after it.
template <int CG>
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint32_t address) {
    const uint64_t from = sdesc(address, 128u, 128u);
    if constexpr (CG == 2) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n" ::"r"(tmem), "l"(from) : "memory");
    else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n" ::"r"(tmem), "l"(from) : "memory");
}

// D[tmem] (+)= A * B, issued by one thread.
__device__ __forceinline__ void mma(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
    const uint32_t mask = 0;
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}\n" ::"r"(d_tmem),
        "l"(a), "l"(b), "r"(id), "r"(accumulate), "r"(mask), "r"(mask), "r"(mask), "r"(mask));
}

// Arrive on an mbarrier once every tcgen05 operation issued so far by this thread has completed.
__device__ __forceinline__ void commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(smem_u32(bar))
                 : "memory");
}

__device__ __forceinline__ void bar_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void fence_bar_init() { asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory"); }

// Bounded wait for the phase with the given parity; false when the limit ran out.
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, uint32_t limit) {
    const uint32_t address = smem_u32(bar);
    for (uint32_t i = 0; i < limit; ++i) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
            : "=r"(done)
            : "r"(address), "r"(parity)
            : "memory");
        if (done) return true;
    }
    return false;
}

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }
__device__ __forceinline__ void fence_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }

// TMEM allocation by one full warp; the base address is written to shared memory.
__device__ __forceinline__ void tmem_alloc(uint32_t* dst, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(dst)),
                 "r"(columns)
                 : "memory");
}
__device__ __forceinline__ void tmem_relinquish() {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t base, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(base), "r"(columns) : "memory");
}

// The same for a group of CG CTAs, and for a pair the arrival at the barrier in both CTAs.
template <int CG>
__device__ __forceinline__ void commit_group(uint64_t* bar) {
    if constexpr (CG == 2)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(
                smem_u32(bar)),
            "h"(uint16_t(3))
            : "memory");
    else
        commit(bar);
}
template <int CG>
__device__ __forceinline__ void tmem_alloc_group(uint32_t* dst, uint32_t columns) {
    if constexpr (CG == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(dst)), "r"(columns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
    } else {
        tmem_alloc(dst, columns);
        tmem_relinquish();
    }
}
template <int CG>
__device__ __forceinline__ void tmem_dealloc_group(uint32_t base, uint32_t columns) {
    if constexpr (CG == 2)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(base), "r"(columns) : "memory");
    else
        tmem_dealloc(base, columns);
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(one));
    return one != 0;
}

// Cluster helpers: this CTA's rank, the shared::cluster address of CTA 0's copy of a shared variable, and the
// barrier over all threads of the cluster.
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t leader_address(const void* p) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
    return r;
}
// Four floats at `address` of this CTA's shared memory, from CTA `rank`'s.
__device__ __forceinline__ float4 load_cluster(uint32_t address, int rank) {
    float4 v;
    asm volatile("{\n\t.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %4, %5;\n\tld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n\t}"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(address), "r"(rank)
                 : "memory");
    return v;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// Orders nothing but what tcgen05 fences order: a release would wait for the warp's stores to global memory.
__device__ __forceinline__ void bar_arrive_cluster(uint32_t address) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(address) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void bar_expect(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}

// Takes bytes off the barrier's count as a copy would whose bytes were expected and that is not issued.
__device__ __forceinline__ void bar_unexpect(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;\n" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
// A word of both CTAs' copies of a shared variable, or of CTA 0's.
template <int CG>
__device__ __forceinline__ void store_both(uint32_t* p, uint32_t v) {
    if constexpr (CG == 2)
        asm volatile(
            "{\n\t.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %0, 0;\n\tst.shared::cluster.u32 [a], %1;\n\t"
            "mapa.shared::cluster.u32 a, %0, 1;\n\tst.shared::cluster.u32 [a], %1;\n\t}\n" ::"r"(smem_u32(p)),
            "r"(v)
            : "memory");
    else
        asm volatile("st.shared.u32 [%0], %1;\n" ::"r"(smem_u32(p)), "r"(v) : "memory");
}
template <int CG>
__device__ __forceinline__ void store_leader(uint32_t* p, uint32_t v) {
    if constexpr (CG == 2) asm volatile("st.shared::cluster.u32 [%0], %1;\n" ::"r"(leader_address(p)), "r"(v) : "memory");
    else asm volatile("st.shared.u32 [%0], %1;\n" ::"r"(smem_u32(p)), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t load_shared(const uint32_t* p) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];\n" : "=r"(v) : "r"(smem_u32(p)) : "memory");
    return v;
}

// TMA loads of one box into this CTA's shared memory, their bytes counted at `bar` (a shared::cluster address:
// for a pair the leader's barrier).  No multicast.
template <int CG>
__device__ __forceinline__ void tma_load_2d(void* dst, const void* map, int x, int y, uint32_t bar) {
    if constexpr (CG == 2)
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(
                smem_u32(dst)),
            "l"(map), "r"(x), "r"(y), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(
                smem_u32(dst)),
            "l"(map), "r"(x), "r"(y), "r"(bar)
            : "memory");
}
template <int CG>
__device__ __forceinline__ void tma_load_3d(void* dst, const void* map, int x, int y, int z, uint32_t bar) {
    if constexpr (CG == 2)
        asm volatile(
            "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(
                smem_u32(dst)),
            "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(
                smem_u32(dst)),
            "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
            : "memory");
}

template <int CG>
__device__ __forceinline__ void tma_load_4d(void* dst, const void* map, int x, int y, int z, int w, uint32_t bar) {
    if constexpr (CG == 2)
        asm volatile(
            "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];\n" ::"r"(
                smem_u32(dst)),
            "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];\n" ::"r"(
                smem_u32(dst)),
            "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
            : "memory");
}

__device__ __forceinline__ void tma_prefetch_2d(const void* map, int x, int y) {  // to L2
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];\n" ::"l"(map), "r"(x), "r"(y) : "memory");
}
// A TMA store of one box from shared memory, as a group of this thread's bulk copies; stores_read: their shared memory is
// free again; stores_done: they are through.
__device__ __forceinline__ void tma_store_2d(const void* map, int x, int y, const void* src) {
    asm volatile(
        "cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];\n\tcp.async.bulk.commit_group;\n" ::"l"(map), "r"(x),
        "r"(y), "r"(smem_u32(src))
        : "memory");
}
__device__ __forceinline__ void stores_read() { asm volatile("cp.async.bulk.wait_group.read 0;\n" ::: "memory"); }
__device__ __forceinline__ void stores_done() { asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory"); }

// 16 consecutive fp32 columns of this thread's TMEM lane (32x32b shape, warp-collective).
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float* v) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// Load 32 consecutive fp32 columns of this thread's TMEM lane: one load and its wait in one
// statement, so nothing reads the registers before they land (32x32b shape, warp-collective).
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
        "tcgen05.wait::ld.sync.aligned;\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// COLS (64 or 32) columns of the 32 lanes from taddr on, as 8 x 8 fragments (16x256b shape, warp-collective): lane l has, in
// low for lanes 0..15 and in high for lanes 16..31, element [4 u + 2 h + i] = lane l / 4 + 8 h, column 8 u + 2 (l % 4) + i.
template <int COLS>
__device__ __forceinline__ void tmem_ld_rows(uint32_t taddr, float* low, float* high) {
    uint32_t r[COLS];
    if constexpr (COLS == 64)
        asm volatile(
            "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
            "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%64];\n"
            "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
            "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%65];\n"
            "tcgen05.wait::ld.sync.aligned;\n"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
              "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
              "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
              "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
              "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
              "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
              "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
              "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
            : "r"(taddr), "r"(taddr + (16u << 16))
            : "memory");
    else
        asm volatile(
            "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%32];\n"
            "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%33];\n"
            "tcgen05.wait::ld.sync.aligned;\n"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
              "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
              "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
              "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
            : "r"(taddr), "r"(taddr + (16u << 16))
            : "memory");
#pragma unroll
    for (int i = 0; i < COLS / 2; ++i) {
        low[i] = __uint_as_float(r[i]);
        high[i] = __uint_as_float(r[COLS / 2 + i]);
    }
}
// Four 8 x 8 matrices of 16-bit elements from or to shared memory: lane 8 m + r has the address of row r of matrix m, and
// in v[m] its elements of row lane / 4, columns 2 (lane % 4) + 0, 1.
__device__ __forceinline__ void load_matrices(uint32_t address, uint32_t (&v)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];\n" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(address) : "memory");
}
__device__ __forceinline__ void store_matrices(uint32_t address, const uint32_t (&v)[4]) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};\n" ::"r"(address), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}

// Store 16 consecutive fp32 columns of this thread's TMEM lane (32x32b shape, warp-collective).
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const float* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(taddr),
        "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])), "r"(__float_as_uint(v[3])),
        "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])), "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7])),
        "r"(__float_as_uint(v[8])), "r"(__float_as_uint(v[9])), "r"(__float_as_uint(v[10])), "r"(__float_as_uint(v[11])),
        "r"(__float_as_uint(v[12])), "r"(__float_as_uint(v[13])), "r"(__float_as_uint(v[14])), "r"(__float_as_uint(v[15]))
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

}  // namespace tc
}  // namespace odie
