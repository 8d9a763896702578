// The sm_100a instructions the block-scaled product is written in: barriers with
// bounded waits, tensor-map loads, tensor memory and tcgen05.
#ifndef PS_B200_TENSOR_CORE_CUH
#define PS_B200_TENSOR_CORE_CUH

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace tc {

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// ---------------------------------------------------------------------------
// barriers
// ---------------------------------------------------------------------------
__device__ __forceinline__ void bar_init(uint64_t* bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_init_fence() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void bar_expect(uint64_t* bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Arrival on the barrier at the same place in CTA `rank` of the cluster.
__device__ __forceinline__ void bar_arrive_at(uint64_t* bar, uint32_t rank)
{
    asm volatile(
        "{\n"
        ".reg .b32 r;\n"
        "mapa.shared::cluster.u32 r, %0, %1;\n"
        "mbarrier.arrive.shared::cluster.b64 _, [r];\n"
        "}\n" ::"r"(smem_u32(bar)),
        "r"(rank)
        : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t addr, uint32_t parity)
{
    uint32_t done;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(done)
        : "r"(addr), "r"(parity)
        : "memory");
    return done != 0;
}
// True in one lane of a converged warp.  A branch on it tells the compiler that a single thread runs what is
// inside, so that descriptors and addresses of tcgen05 and of tensor-map copies stay in uniform registers;
// a branch on the lane's number makes it loop over lanes before each of them (product 8192^3: 458 us, not 390).
__device__ __forceinline__ bool elect_one()
{
    uint32_t one;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(one));
    return one != 0;
}
__device__ __forceinline__ uint64_t now_ns()
{
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}

// How long a wait may last before its CTA gives up.  What is waited for takes microseconds.
constexpr uint64_t kWaitLimitNs = 2000000000ull;

// Waits for the phase of the given parity.  False: it did not come within the limit, or another warp of
// the CTA has given up (`gave_up` is set).
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, volatile int* gave_up)
{
    const uint32_t addr = smem_u32(bar);
    for (int i = 0; i < 64; ++i)
        if (bar_try(addr, parity)) return true;
    const uint64_t start = now_ns();
    for (;;) {
        for (int i = 0; i < 16; ++i)
            if (bar_try(addr, parity)) return true;
        if (*gave_up) return false;
        if (now_ns() - start > kWaitLimitNs) {
            *gave_up = 1;
            return false;
        }
    }
}

__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
    return r;
}
// 16 bytes of another CTA's shared memory
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t local_addr, uint32_t rank)
{
    float4 v;
    asm volatile(
        "{\n"
        ".reg .b32 r;\n"
        "mapa.shared::cluster.u32 r, %4, %5;\n"
        "ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [r];\n"
        "}\n"
        : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
        : "r"(local_addr), "r"(rank)
        : "memory");
    return v;
}

// ---------------------------------------------------------------------------
// tensor-map loads
// ---------------------------------------------------------------------------
__device__ __forceinline__ void prefetch_map(const CUtensorMap* m)
{
    asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
}
// `bytes` (a multiple of 16) from global memory, both on 16-byte boundaries.
__device__ __forceinline__ void load_bulk(void* dst, const void* src, uint32_t bytes, uint64_t* bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     smem_u32(dst)),
                 "l"(src), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void load_bulk(void* dst, const void* src, uint32_t bytes, uint64_t* bar, uint64_t policy)
{
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(
            smem_u32(dst)),
        "l"(src), "r"(bytes), "r"(smem_u32(bar)), "l"(policy)
        : "memory");
}
__device__ __forceinline__ uint64_t evict_first_policy()
{
    uint64_t p;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    return p;
}
// One CTA's load; completion counts on this CTA's barrier.
__device__ __forceinline__ void load_box(const CUtensorMap* m, uint32_t dst, uint64_t* bar, int x, int y)
{
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::
            "r"(dst),
        "l"(m), "r"(smem_u32(bar)), "r"(x), "r"(y)
        : "memory");
}
// Address of `p` in CTA `rank`'s shared memory
__device__ __forceinline__ uint32_t cluster_addr(const void* p, uint32_t rank)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
    return r;
}
// A CTA of a pair loads into its own memory; completion counts on a barrier of either (cluster_addr).
__device__ __forceinline__ void load_box_pair(const CUtensorMap* m, uint32_t dst, uint32_t bar, int x, int y)
{
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, "
        "%4}], [%2];" ::"r"(dst),
        "l"(m), "r"(bar), "r"(x), "r"(y)
        : "memory");
}

// A box of shared memory to global memory; boxes reach over the matrix's end without writing there.
__device__ __forceinline__ void store_box(const CUtensorMap* m, uint32_t src, int x, int y)
{
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(m), "r"(src),
                 "r"(x), "r"(y)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// Until at most `kLeft` of this thread's stores still read shared memory.
template <int kLeft>
__device__ __forceinline__ void store_wait_read()
{
    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kLeft) : "memory");
}
// What this thread wrote to shared memory is seen by the copies it issues from now on.
__device__ __forceinline__ void fence_to_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---------------------------------------------------------------------------
// tensor memory
// ---------------------------------------------------------------------------
template <int kCtas>
__device__ __forceinline__ void tmem_alloc(uint32_t* dst, uint32_t columns)
{
    if constexpr (kCtas == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)),
                     "r"(columns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)),
                     "r"(columns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
}
template <int kCtas>
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t columns)
{
    if constexpr (kCtas == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns));
    else
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns));
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 columns of this warp's 32 lanes
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&v)[32])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// ---------------------------------------------------------------------------
// tcgen05
// ---------------------------------------------------------------------------
constexpr uint64_t kSwizzle128 = 2, kSwizzleNone = 0;

// Shared-memory matrix descriptor; offsets in bytes.
__device__ __forceinline__ uint64_t matrix_desc(uint32_t addr, uint32_t lead, uint32_t stride, uint64_t swizzle)
{
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(stride >> 4) << 32) |
           (1ull << 46) | (swizzle << 61);
}

// Instruction descriptor of kind::mxf8f6f4: formats 0 = e4m3, 1 = e5m2; a transposed operand has its outer
// dimension contiguous; scales are powers of two (8 exponent bits).
__host__ __device__ constexpr uint32_t mx_idesc(int m, int n, int fmt_a, int fmt_b, int transpose_a, int transpose_b)
{
    return ((uint32_t)fmt_a << 7) | ((uint32_t)fmt_b << 10) | ((uint32_t)transpose_a << 15) |
           ((uint32_t)transpose_b << 16) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 7) << 27);
}
// The same with byte `i` of the scale words selected for both operands.
__device__ __forceinline__ uint32_t mx_idesc_select(uint32_t d, uint32_t i) { return d | (i << 4) | (i << 29); }

template <int kCtas>
__device__ __forceinline__ void mx_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                       uint32_t accumulate)
{
    if constexpr (kCtas == 1)
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "setp.ne.b32 p, %6, 0;\n"
            "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], p;\n"
            "}\n" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "setp.ne.b32 p, %6, 0;\n"
            "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], p;\n"
            "}\n" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
}
// 128 scale words (32 rows of 16 bytes in shared memory) into 4 columns, for all four groups of lanes
template <int kCtas>
__device__ __forceinline__ void scale_copy(uint32_t dst, uint64_t desc)
{
    if constexpr (kCtas == 1)
        asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(dst), "l"(desc) : "memory");
    else
        asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(dst), "l"(desc) : "memory");
}
// Arrival on `bar` (of both CTAs of a pair) when all that this thread issued so far is done.
template <int kCtas>
__device__ __forceinline__ void mma_commit(uint64_t* bar)
{
    if constexpr (kCtas == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                     : "memory");
    else
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                smem_u32(bar)),
            "h"((uint16_t)3)
            : "memory");
}

}  // namespace tc

#endif
