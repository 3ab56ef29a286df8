// tma.cuh -- bulk tensor copies, 128-byte-swizzled operand tiles and bounded
// waits for the dense-layer kernels (linear.cu).
//
// Operand tiles: a box of R rows x 64 16-bit values, row r at byte 128 r, the
// 16-byte piece p of a row at piece p ^ (r & 7) (the 128-byte swizzle of
// cp.async.bulk.tensor; tiles start on 1024-byte boundaries).  The box is read
// by the tensor core in two ways:
//   K-major   rows = M or N, the 64 contiguous values along K.  Stride between
//             8-row groups 1024 bytes; K-step s (16 values) starts 32 s bytes in.
//   MN-major  rows = K, the 64 contiguous values along M or N; a wider tile is
//             a sequence of 64-wide boxes.  Stride between 8-row groups (along
//             K) 1024 bytes, between boxes (along M / N) the box's bytes;
//             K-step s (16 rows) starts 2048 s bytes in.
#pragma once
#include <cuda.h>

#include "umma.cuh"

namespace nb {
namespace tma {

constexpr uint32_t kBoxCols = 64;  // 128 bytes of 16-bit values

// Shared-memory matrix descriptor with the 128-byte swizzle (layout type 2).
NB_DEV uint64_t desc_sw128(uint32_t smem_addr, uint32_t lbo_bytes, uint32_t sbo_bytes) {
    return umma::smem_desc(smem_addr, lbo_bytes, sbo_bytes) | (2ull << 61);
}

// Instruction descriptor of kind::f16 with fp16 or bf16 operands (both the
// same), fp32 accumulator.
__host__ __device__ constexpr uint32_t idesc_16bit(uint32_t M, uint32_t N, uint32_t a_mn, uint32_t b_mn, uint32_t bf16) {
    return umma::idesc_f16(M, N, a_mn, b_mn) | (bf16 << 7) | (bf16 << 10);
}

NB_DEV void load_2d(uint32_t dst, const CUtensorMap* map, int32_t x, int32_t y, uint64_t* mbar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(smem_u32(mbar))
        : "memory");
}
// The same with the completion signalled at a barrier of the cluster's leading
// CTA (mbar: its shared::cluster address), for a pair of CTAs on one MMA.
NB_DEV void load_2d_pair(uint32_t dst, const CUtensorMap* map, int32_t x, int32_t y, uint32_t mbar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(
            dst),
        "l"(map), "r"(x), "r"(y), "r"(mbar)
        : "memory");
}
// Shared memory -> global; out-of-range rows and columns of the box are not written.
NB_DEV void store_2d(const CUtensorMap* map, uint32_t src, int32_t x, int32_t y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];\n" ::"l"(map), "r"(x), "r"(y), "r"(src)
                 : "memory");
}
// A box into the L2 cache, ahead of its loads.
NB_DEV void prefetch_2d(const CUtensorMap* map, int32_t x, int32_t y) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];\n" ::"l"(map), "r"(x), "r"(y) : "memory");
}
NB_DEV void store_commit() { asm volatile("cp.async.bulk.commit_group;\n" ::: "memory"); }
// At most N of this thread's store groups still read shared memory.
template <int N>
NB_DEV void store_wait_read() {
    asm volatile("cp.async.bulk.wait_group.read %0;\n" ::"n"(N) : "memory");
}
NB_DEV void store_wait_all() { asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory"); }
NB_DEV void prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];\n" ::"l"(map) : "memory"); }

NB_DEV void expect_tx(uint64_t* mbar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(smem_u32(mbar)), "r"(bytes) : "memory");
}
NB_DEV void arrive(uint64_t* mbar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(smem_u32(mbar)) : "memory");
}

// Waits for the phase of the given parity; false after kWaitLimitNs.  The
// clock is read every 64 polls only, so a wait that ends soon never reads it;
// it runs on while the GPU works for another process, so a wait that is late
// polls on for a while before it gives up.
constexpr uint64_t kWaitLimitNs = 1000000000ull;
constexpr uint32_t kLatePolls = 64u * 64u;
NB_DEV bool wait(uint64_t* mbar, uint32_t parity) {
    const uint32_t a = smem_u32(mbar);
    uint64_t t0 = 0u;
    uint32_t late = 0u;
    for (uint32_t i = 0;; ++i) {
        uint32_t done;
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
            "selp.u32 %0, 1, 0, p;\n"
            "}\n"
            : "=r"(done)
            : "r"(a), "r"(parity)
            : "memory");
        if (done) return true;
        if ((i & 63u) == 63u) {
            const uint64_t t = umma::globaltimer();
            if (t0 == 0u) t0 = t;
            else if (t - t0 > kWaitLimitNs && (late += 64u) > kLatePolls) return false;
        }
    }
}

// Registers of the executing warpgroup's threads from here on.
template <int N>
NB_DEV void registers_down() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(N));
}
template <int N>
NB_DEV void registers_up() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(N));
}

// ---- a pair of CTAs on one MMA (cta_group::2) ----
NB_DEV void tmem_alloc_pair(uint32_t* slot, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(slot)), "r"(ncols) : "memory");
}
NB_DEV void tmem_relinquish_pair() { asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory"); }
NB_DEV void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(taddr), "r"(ncols) : "memory");
}
NB_DEV void mma_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Arrival at the same barrier of both CTAs when the MMAs issued so far are done.
NB_DEV void commit_pair(uint64_t* mbar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(smem_u32(mbar)),
        "h"(static_cast<uint16_t>(3u))
        : "memory");
}

// ---- clusters ----
// shared::cluster address of another CTA's variable (addr: this CTA's address of it).
NB_DEV uint32_t peer_addr(uint32_t addr, uint32_t rank) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(remote) : "r"(addr), "r"(rank));
    return remote;
}
NB_DEV void arrive_at(uint32_t mbar_cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(mbar_cluster_addr) : "memory");
}
NB_DEV uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
    return r;
}
NB_DEV void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// A float of another CTA's shared memory (addr: this CTA's address of the same variable).
NB_DEV float peer_f32(uint32_t addr, uint32_t rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(peer_addr(addr, rank)) : "memory");
    return v;
}

NB_DEV double peer_f64(uint32_t addr, uint32_t rank) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];\n" : "=d"(v) : "r"(peer_addr(addr, rank)) : "memory");
    return v;
}
NB_DEV uint32_t peer_u32(uint32_t addr, uint32_t rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];\n" : "=r"(v) : "r"(peer_addr(addr, rank)) : "memory");
    return v;
}

}  // namespace tma
}  // namespace nb
