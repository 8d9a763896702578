// Product of two matrices held in 8-bit floating point with a power-of-two scale
// for each block of 128 along the contracted dimension:
//
//   out[i, j] = sum_k a(i, k) 2^ea(i, k / 128) b(j, k) 2^eb(j, k / 128)  (+ bias[j])
//
// accumulated in 32 bits and rounded once to the output's type.  The scales are
// powers of two, so the tensor core applies them itself (kind::mxf8f6f4: one
// scale byte for 32 consecutive k; the four 32s of a block select the same
// byte), and nothing between the first product and the output touches the
// accumulator.
//
// Either operand may have the contracted dimension or the outer one contiguous
// (the instruction descriptor's transpose bits): the weight that the forward
// product reads is read as it lies by the input-gradient product, and the
// weight gradient contracts over the rows of both operands.  Both forms use the
// same 128 x 128-byte box with the 128-byte swizzle, with the coordinates
// swapped.
#include "ps_b200.h"

#include "ps_internal.h"
#include "ps_launch.cuh"
#include "ps_tensor_core.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <cstring>

namespace {

constexpr uint32_t kTile = 128;                   // rows of A, rows of B and k of one box
constexpr uint32_t kBoxBytes = kTile * kTile;     // 16 KB
constexpr uint32_t kScaleBytes = 512;             // scales of 128 outer elements, four k blocks

__device__ unsigned int g_gave_up;  // CTAs that ran into the limit of a wait

struct ProductArgs {
    const void* bias;
    void* out;
    uint64_t ldo;
    uint32_t m, n, n_kb;
    uint32_t tiles_m, tiles_n;
    uint32_t scale_blocks_a, scale_blocks_b;
    uint32_t idesc;
    int a_k_inner, b_k_inner;  // the contracted dimension is the contiguous one
    int bias_dtype, out_dtype;
    int vec, n_vec;            // output rows start, and end, on 16-byte boundaries
};

__device__ __forceinline__ float bias_at(const ProductArgs& p, uint32_t col)
{
    if (p.bias_dtype == PS_DTYPE_F16) return __half2float(reinterpret_cast<const __half*>(p.bias)[col]);
    if (p.bias_dtype == PS_DTYPE_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.bias)[col]);
    return reinterpret_cast<const float*>(p.bias)[col];
}
__device__ __forceinline__ uint32_t pack2(int dtype, float lo, float hi)
{
    if (dtype == PS_DTYPE_F16) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void store1(const ProductArgs& p, uint64_t at, float v)
{
    if (p.out_dtype == PS_DTYPE_F16)
        reinterpret_cast<__half*>(p.out)[at] = __float2half_rn(v);
    else if (p.out_dtype == PS_DTYPE_BF16)
        reinterpret_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
    else
        reinterpret_cast<float*>(p.out)[at] = v;
}

// Shared-memory descriptor of the box at `addr`: k contiguous (8-row groups 1024 bytes apart), or the outer
// dimension contiguous (groups of 8 k 1024 bytes apart).  The next 32 k are 32 bytes resp. 32 rows on.
__device__ __forceinline__ uint64_t box_desc(uint32_t addr)
{
    return tc::matrix_desc(addr, 1024, 1024, tc::kSwizzle128);
}
__device__ __forceinline__ uint64_t scale_desc(uint32_t addr)
{
    return tc::matrix_desc(addr, 128, 128, tc::kSwizzleNone);
}

// ---------------------------------------------------------------------------
// One 128 x 128 tile a cluster: its CTAs share the k blocks, and join their
// partial sums over distributed shared memory in the order of their ranks.
// ---------------------------------------------------------------------------
constexpr int kSplitStages = 3;
constexpr uint32_t kSplitStageBytes = 2 * kBoxBytes + 2 * kScaleBytes;
constexpr uint32_t kSplitThreads = 192;  // warps 0-3 epilogue, 4 loads, 5 tensor core
constexpr uint32_t kPartialPitch = 132;  // floats; 16-byte accesses of 8 rows fall into different banks
constexpr uint32_t kSplitSmem = 1024 + kSplitStages * kSplitStageBytes;
constexpr uint32_t kSplitColumns = 256;  // accumulator 128, scales behind it
static_assert(kTile * kPartialPitch * 4 <= kSplitStages * kSplitStageBytes, "the partial tile lies over the stages");

__global__ void __launch_bounds__(kSplitThreads)
block_matmul_split_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                          const __grid_constant__ CUtensorMap map_sa, const __grid_constant__ CUtensorMap map_sb,
                          const __grid_constant__ ProductArgs p, const uint32_t splits)
{
    extern __shared__ unsigned char smem_raw[];
    __shared__ uint64_t full[kSplitStages], empty[kSplitStages], done;
    __shared__ uint32_t tmem_base;
    __shared__ volatile int gave_up;

    const uint32_t base = (tc::smem_u32(smem_raw) + 1023u) & ~1023u;
    unsigned char* const base_ptr = smem_raw + (base - tc::smem_u32(smem_raw));
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = blockIdx.x % splits, tile = blockIdx.x / splits;
    const uint32_t tm = tile % p.tiles_m, tn = tile / p.tiles_m;
    const uint32_t kb0 = (uint32_t)((uint64_t)p.n_kb * rank / splits);
    const uint32_t kb1 = (uint32_t)((uint64_t)p.n_kb * (rank + 1) / splits);

    if (warp == 4 && p.n_kb > 0 && tc::elect_one())
        tc::prefetch_map(&map_a), tc::prefetch_map(&map_b), tc::prefetch_map(&map_sa), tc::prefetch_map(&map_sb);
    if (threadIdx.x == 0) {
        for (int s = 0; s < kSplitStages; ++s) tc::bar_init(&full[s], 1), tc::bar_init(&empty[s], 1);
        tc::bar_init(&done, 1);
        gave_up = 0;
        tc::bar_init_fence();
    }
    if (warp == 5) tc::tmem_alloc<1>(&tmem_base, kSplitColumns);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = tmem_base;
    cudaTriggerProgrammaticLaunchCompletion();
    cudaGridDependencySynchronize();  // up to here nothing that another kernel writes was touched

    if (warp == 4 && tc::elect_one()) {
        uint32_t issued = 0;
        for (uint32_t kb = kb0; kb < kb1; ++kb, ++issued) {
            const uint32_t s = issued % kSplitStages, round = issued / kSplitStages;
            if (round > 0 && !tc::bar_wait(&empty[s], (round - 1) & 1, &gave_up)) break;
            const bool scales = kb == kb0 || (kb & 3) == 0;
            const uint32_t at = base + s * kSplitStageBytes;
            tc::bar_expect(&full[s], 2 * kBoxBytes + (scales ? 2 * kScaleBytes : 0));
            const int k = (int)(kb * kTile), i = (int)(tm * kTile), j = (int)(tn * kTile);
            tc::load_box(&map_a, at, &full[s], p.a_k_inner ? k : i, p.a_k_inner ? i : k);
            tc::load_box(&map_b, at + kBoxBytes, &full[s], p.b_k_inner ? k : j, p.b_k_inner ? j : k);
            if (scales) {
                tc::load_box(&map_sa, at + 2 * kBoxBytes, &full[s], 0, (int)((kb >> 2) * p.scale_blocks_a + tm));
                tc::load_box(&map_sb, at + 2 * kBoxBytes + kScaleBytes, &full[s], 0,
                             (int)((kb >> 2) * p.scale_blocks_b + tn));
            }
        }
        if (gave_up) {
            // copies may still be landing in this CTA's memory: the stages in flight, each waited for with the
            // same limit
            int ignore = 0;
            for (uint32_t i = issued < kSplitStages ? 0 : issued - kSplitStages; i < issued; ++i)
                tc::bar_wait(&full[i % kSplitStages], (i / kSplitStages) & 1, &ignore);
        }
    } else if (warp == 5 && tc::elect_one()) {
        const uint32_t a_step = p.a_k_inner ? 32 : 32 * kTile, b_step = p.b_k_inner ? 32 : 32 * kTile;
        uint32_t used = 0, groups = 0;
        for (uint32_t kb = kb0; kb < kb1; ++kb, ++used) {
            const uint32_t s = used % kSplitStages;
            if (!tc::bar_wait(&full[s], (used / kSplitStages) & 1, &gave_up)) break;
            tc::fence_after();
            const uint32_t at = base + s * kSplitStageBytes;
            if (kb == kb0 || (kb & 3) == 0) {
                ++groups;
                const uint32_t sf = tmem + kTile + (groups & 1) * 8;
                tc::scale_copy<1>(sf, scale_desc(at + 2 * kBoxBytes));
                tc::scale_copy<1>(sf + 4, scale_desc(at + 2 * kBoxBytes + kScaleBytes));
            }
            const uint32_t sf = tmem + kTile + (groups & 1) * 8;
            const uint32_t idesc = tc::mx_idesc_select(p.idesc, kb & 3);
#pragma unroll
            for (uint32_t q = 0; q < 4; ++q)
                tc::mx_mma<1>(tmem, box_desc(at + q * a_step), box_desc(at + kBoxBytes + q * b_step), idesc, sf, sf + 4,
                              used > 0 || q > 0);
            tc::mma_commit<1>(&empty[s]);
        }
        tc::mma_commit<1>(&done);
        if (gave_up) {
            int ignore = 0;
            tc::bar_wait(&done, 0, &ignore);
        }
    } else if (warp < 4) {
        // this CTA's partial tile into shared memory, over the stages (all of them are read by now)
        const bool ok = tc::bar_wait(&done, 0, &gave_up);
        tc::fence_after();
        float* row = reinterpret_cast<float*>(base_ptr) + (size_t)(warp * 32 + lane) * kPartialPitch;
        const bool good = ok && !gave_up;
        for (uint32_t c = 0; c < kTile && tm * kTile + warp * 32 < p.m; c += 32) {  // rows that there are
            uint32_t v[32];
            if (kb0 < kb1) {
                tc::tmem_ld32(tmem + (warp << 21) + c, v);
                tc::tmem_ld_wait();
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float4 f = make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]),
                                       __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]));
                if (kb0 >= kb1) f = make_float4(0.f, 0.f, 0.f, 0.f);
                if (!good) f.x = f.y = f.z = f.w = __int_as_float(0x7fffffff);
                *reinterpret_cast<float4*>(row + c + 4 * i) = f;
            }
        }
        tc::fence_before();
    }

    __syncwarp();
    __syncthreads();
    if (warp == 5) tc::tmem_free<1>(tmem, kSplitColumns);
    if (splits > 1) tc::cluster_sync();

    // rows [lo, hi) of the tile: the sum of the partial tiles, one row a warp
    const uint32_t lo = rank * kTile / splits, hi = (rank + 1) * kTile / splits;
    for (uint32_t r = lo + warp; r < hi; r += kSplitThreads / 32) {
        const uint32_t i = tm * kTile + r, j = tn * kTile + lane * 4;
        if (i >= p.m) break;
        const uint32_t at = base + (r * kPartialPitch + lane * 4) * 4;
        float4 t = tc::ld_cluster_f4(at, 0);
        for (uint32_t s = 1; s < splits; ++s) {
            const float4 u = tc::ld_cluster_f4(at, s);
            t.x += u.x, t.y += u.y, t.z += u.z, t.w += u.w;
        }
        if (p.bias != nullptr) {
            if (j < p.n) t.x += bias_at(p, j);
            if (j + 1 < p.n) t.y += bias_at(p, j + 1);
            if (j + 2 < p.n) t.z += bias_at(p, j + 2);
            if (j + 3 < p.n) t.w += bias_at(p, j + 3);
        }
        const uint64_t o = (uint64_t)i * p.ldo + j;
        if (p.vec && j + 4 <= p.n) {
            if (p.out_dtype == PS_DTYPE_F32)
                *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + o) = t;
            else
                *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.out) + o) =
                    make_uint2(pack2(p.out_dtype, t.x, t.y), pack2(p.out_dtype, t.z, t.w));
        } else {
            const float f[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (j + q < p.n) store1(p, o + q, f[q]);
        }
    }
    if (splits > 1) tc::cluster_sync();  // no CTA leaves while its partial tile is read
    if (threadIdx.x == 0 && gave_up) atomicAdd(&g_gave_up, 1u);
}

// ---------------------------------------------------------------------------
// 256 x 256 tiles, one after another on each pair of SMs: the pair's tensor
// cores work as one (cta_group::2), each CTA holding 128 rows of A, 128 rows of
// B and 128 rows of the accumulator.
//
// A k block keeps an SM's tensor core busy for 512 cycles and brings it 32 KB, 64 bytes a cycle, all that an SM can
// read; tiles of 128 x 128 would need twice that.  8192^3: 363 us in a burst (3.03 PF), 444 us at the power cap; a
// sixth stage of 34 KB instead of the second store buffer gains nothing there.
//
// Two accumulators of 256 columns and the scales do not fit into 512 columns of
// tensor memory, so the accumulators overlap in 32 columns: the epilogue reads
// those first, and the next tile starts as soon as they are out.
// ---------------------------------------------------------------------------
constexpr uint32_t kPairTile = 256;
constexpr int kPairStages = 5;
constexpr uint32_t kPairStageBytes = 2 * kBoxBytes + 4 * kScaleBytes;  // scales: 1 of A, 2 of B, 1 unused
constexpr uint32_t kPairWarps = 8;                                     // of the epilogue; behind them loads, tensor core
constexpr uint32_t kPairThreads = 32 * (kPairWarps + 2);
constexpr uint32_t kStoreBytes = 32 * 128;                             // 32 rows of 128 bytes a warp
constexpr uint32_t kPairSmem = 1024 + kPairStages * kPairStageBytes + kPairWarps * kStoreBytes;
constexpr uint32_t kAccStride = 224;
constexpr uint32_t kScaleColumn = kAccStride + kPairTile;  // 480: twice 4 columns of A and 8 of B
static_assert(kScaleColumn + 2 * 12 <= 512, "tensor memory");
static_assert(kPairSmem <= 227 * 1024, "shared memory");
static_assert(kPairStages >= 5 && kPairStageBytes % 1024 == 0, "scale columns, swizzled boxes");
constexpr uint32_t kGroupRows = 8;  // tiles of A that are worked on together

__device__ __forceinline__ void tile_at(const ProductArgs& p, uint32_t t, uint32_t* tm, uint32_t* tn)
{
    const uint32_t per = kGroupRows * p.tiles_n, g = t / per, r = t % per;
    const uint32_t first = g * kGroupRows, rows = min(kGroupRows, p.tiles_m - first);
    *tm = first + r % rows, *tn = r / rows;
}

// 128 bytes of an output row from the accumulator's values; kOut is its type.
template <int kOut>
__device__ __forceinline__ void stage_row(unsigned char* buf, const ProductArgs& p, const float* bias, uint32_t tmem,
                                          bool good, bool first, uint64_t* drained)
{
    const uint32_t row = threadIdx.x & 31;
    constexpr uint32_t kCols = kOut == PS_DTYPE_F32 ? 32 : 64;
    uint32_t v[kCols / 32][32];
#pragma unroll
    for (uint32_t h = 0; h < kCols / 32; ++h) tc::tmem_ld32(tmem + 32 * h, v[h]);
    tc::tmem_ld_wait();
    if (first) {
        tc::fence_before();
        __syncwarp();
        if (row == 0) tc::bar_arrive_at(drained, 0);
    }
    if (p.vec) {  // the store before has read the buffer
        if (row == 0) tc::store_wait_read<0>();
        __syncwarp();
    }
#pragma unroll
    for (uint32_t q = 0; q < 8; ++q) {  // 16 bytes each, swizzled as the store's map says
        constexpr uint32_t kPer = kOut == PS_DTYPE_F32 ? 4 : 8;
        float f[kPer];
#pragma unroll
        for (uint32_t i = 0; i < kPer; ++i) f[i] = __uint_as_float(v[q * kPer / 32][(q * kPer + i) % 32]);
        if (p.bias != nullptr) {
#pragma unroll
            for (uint32_t i = 0; i < kPer; i += 4) {
                const float4 b = *reinterpret_cast<const float4*>(bias + q * kPer + i);
                f[i] += b.x, f[i + 1] += b.y, f[i + 2] += b.z, f[i + 3] += b.w;
            }
        }
        if (!good) {
#pragma unroll
            for (uint32_t i = 0; i < kPer; ++i) f[i] = __int_as_float(0x7fffffff);
        }
        uint4 w;
        if constexpr (kOut == PS_DTYPE_F32)
            w = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
        else
            w = make_uint4(pack2(kOut, f[0], f[1]), pack2(kOut, f[2], f[3]), pack2(kOut, f[4], f[5]), pack2(kOut, f[6], f[7]));
        *reinterpret_cast<uint4*>(buf + row * 128 + ((q ^ (row & 7)) << 4)) = w;
    }
}

// The staged 32 rows to an output whose rows start anywhere: eight rows at a time, 4 bytes a lane.  In 16 bits
// the pairs of a row begin with its first or its second element, whichever is on a 4-byte boundary; what is left
// at the ends of the row is stored by itself.
template <int kOut>
__device__ __forceinline__ void store_rows(const ProductArgs& p, const unsigned char* buf, uint32_t row0, uint32_t col)
{
    constexpr uint32_t kCols = kOut == PS_DTYPE_F32 ? 32 : 64;
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t rows = min(32u, p.m - row0), cols = min(kCols, p.n - col);
    for (uint32_t r0 = 0; r0 < rows; r0 += 8) {
        if constexpr (kOut == PS_DTYPE_F32) {
            float v[8];
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i)
                v[i] = *reinterpret_cast<const float*>(buf + (r0 + i) * 128 + (((lane >> 2) ^ i) << 4) + (lane & 3) * 4);
            float* o = reinterpret_cast<float*>(p.out) + (uint64_t)(row0 + r0) * p.ldo + col + lane;
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i)
                if (r0 + i < rows && lane < cols) o[i * p.ldo] = v[i];
        } else {
            uint16_t* const out = reinterpret_cast<uint16_t*>(p.out) + (uint64_t)(row0 + r0) * p.ldo + col;
            uint32_t lo[8], hi[8];
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                const uint32_t odd = (uint32_t)((uintptr_t)(out + i * p.ldo) >> 1) & 1;
                const uint32_t e = 2 * lane + odd, f = min(e + 1, kCols - 1);
                const unsigned char* const row = buf + (r0 + i) * 128;
                lo[i] = *reinterpret_cast<const uint16_t*>(row + (((e >> 3) ^ i) << 4) + (e & 7) * 2);
                hi[i] = *reinterpret_cast<const uint16_t*>(row + (((f >> 3) ^ i) << 4) + (f & 7) * 2);
            }
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                if (r0 + i >= rows) break;
                uint16_t* const o = out + i * p.ldo;
                const uint32_t odd = (uint32_t)((uintptr_t)o >> 1) & 1, e = 2 * lane + odd;
                if (e + 1 < cols)
                    *reinterpret_cast<uint32_t*>(o + e) = lo[i] | (hi[i] << 16);
                else if (e < cols)
                    o[e] = (uint16_t)lo[i];
                if (odd && lane == 0) o[0] = *reinterpret_cast<const uint16_t*>(buf + (r0 + i) * 128 + (i << 4));
            }
        }
    }
}

template <int kOut>
__global__ void __launch_bounds__(kPairThreads)
block_matmul_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                         const __grid_constant__ CUtensorMap map_sa, const __grid_constant__ CUtensorMap map_sb,
                         const __grid_constant__ CUtensorMap map_out, const __grid_constant__ ProductArgs p)
{
    extern __shared__ unsigned char smem_raw[];
    __shared__ uint64_t full[kPairStages], empty[kPairStages], done, drained, ended;
    __shared__ uint32_t tmem_base;
    __shared__ __align__(16) float s_bias[kPairWarps][kPairTile / 2];
    __shared__ volatile int gave_up;

    const uint32_t base = (tc::smem_u32(smem_raw) + 1023u) & ~1023u;
    unsigned char* const base_ptr = smem_raw + (base - tc::smem_u32(smem_raw));
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = tc::cluster_rank();
    const uint32_t tiles = p.tiles_m * p.tiles_n, first = blockIdx.x / 2, step = gridDim.x / 2;

    if (warp == kPairWarps && tc::elect_one())
        tc::prefetch_map(&map_a), tc::prefetch_map(&map_b), tc::prefetch_map(&map_sa), tc::prefetch_map(&map_sb);
    if (threadIdx.x == 0) {
        for (int s = 0; s < kPairStages; ++s) tc::bar_init(&full[s], 1), tc::bar_init(&empty[s], 1);
        tc::bar_init(&done, 1);
        tc::bar_init(&drained, 2 * kPairWarps);  // the epilogue's warps of both CTAs
        tc::bar_init(&ended, 1);
        gave_up = 0;
        tc::bar_init_fence();
    }
    if (warp == kPairWarps + 1) tc::tmem_alloc<2>(&tmem_base, 512);
    tc::fence_before();
    __syncthreads();
    tc::cluster_sync();
    tc::fence_after();
    const uint32_t tmem = tmem_base;
    cudaTriggerProgrammaticLaunchCompletion();
    cudaGridDependencySynchronize();  // up to here nothing that another kernel writes was touched

    if (warp == kPairWarps && tc::elect_one()) {
        uint32_t issued = 0;
        bool ok = true;
        for (uint32_t t = first; t < tiles && ok; t += step) {
            uint32_t tm, tn;
            tile_at(p, t, &tm, &tn);
            const int i = (int)(tm * kPairTile + rank * kTile), j = (int)(tn * kPairTile + rank * kTile);
            for (uint32_t kb = 0; kb < p.n_kb; ++kb, ++issued) {
                const uint32_t s = issued % kPairStages, round = issued / kPairStages;
                if (round > 0 && !tc::bar_wait(&empty[s], (round - 1) & 1, &gave_up)) {
                    ok = false;
                    break;
                }
                const bool scales = (kb & 3) == 0;
                const uint32_t at = base + s * kPairStageBytes;
                if (rank == 0) tc::bar_expect(&full[s], 2 * (2 * kBoxBytes + (scales ? 3 * kScaleBytes : 0)));
                const uint32_t bar = tc::cluster_addr(&full[s], 0);
                const int k = (int)(kb * kTile);
                tc::load_box_pair(&map_a, at, bar, p.a_k_inner ? k : i, p.a_k_inner ? i : k);
                tc::load_box_pair(&map_b, at + kBoxBytes, bar, p.b_k_inner ? k : j, p.b_k_inner ? j : k);
                if (scales) {
                    // of A those of this CTA's rows, of B those of both CTAs'
                    const uint32_t sf = at + 2 * kBoxBytes;
                    tc::load_box_pair(&map_sa, sf, bar, 0, (int)((kb >> 2) * p.scale_blocks_a + 2 * tm + rank));
                    const int y = (int)((kb >> 2) * p.scale_blocks_b + 2 * tn);
                    tc::load_box_pair(&map_sb, sf + kScaleBytes, bar, 0, y);
                    tc::load_box_pair(&map_sb, sf + 2 * kScaleBytes, bar, 0, y + 1);
                }
            }
        }
        if (gave_up && rank == 0) {
            // copies may still be landing: the stages in flight, each waited for with the same limit (the barriers
            // of both CTAs' copies are this CTA's; the other stays until the cluster's barrier below)
            int ignore = 0;
            for (uint32_t i = issued < kPairStages ? 0 : issued - kPairStages; i < issued; ++i)
                tc::bar_wait(&full[i % kPairStages], (i / kPairStages) & 1, &ignore);
        }
    } else if (warp == kPairWarps + 1 && rank == 0 && tc::elect_one()) {
        const uint32_t a_step = p.a_k_inner ? 32 : 32 * kTile, b_step = p.b_k_inner ? 32 : 32 * kTile;
        uint32_t used = 0, groups = 0, it = 0;
        bool ok = true;
        for (uint32_t t = first; t < tiles && ok; t += step, ++it) {
            if (it > 0 && !tc::bar_wait(&drained, (it - 1) & 1, &gave_up)) break;
            tc::fence_after();
            const uint32_t acc = tmem + (it & 1) * kAccStride;
            for (uint32_t kb = 0; kb < p.n_kb; ++kb, ++used) {
                const uint32_t s = used % kPairStages;
                if (!tc::bar_wait(&full[s], (used / kPairStages) & 1, &gave_up)) {
                    ok = false;
                    break;
                }
                tc::fence_after();
                const uint32_t at = base + s * kPairStageBytes;
                if ((kb & 3) == 0) {
                    // into the columns of the group before the last: its products are done, since this stage's
                    // load waited for those five k blocks back, and a tile's first one for the tile before
                    ++groups;
                    const uint32_t sf = tmem + kScaleColumn + (groups & 1) * 12, from = at + 2 * kBoxBytes;
                    tc::scale_copy<2>(sf, scale_desc(from));
                    tc::scale_copy<2>(sf + 4, scale_desc(from + kScaleBytes));
                    tc::scale_copy<2>(sf + 8, scale_desc(from + 2 * kScaleBytes));
                }
                const uint32_t sf = tmem + kScaleColumn + (groups & 1) * 12;
                const uint32_t idesc = tc::mx_idesc_select(p.idesc, kb & 3);
#pragma unroll
                for (uint32_t q = 0; q < 4; ++q)
                    tc::mx_mma<2>(acc, box_desc(at + q * a_step), box_desc(at + kBoxBytes + q * b_step), idesc, sf,
                                  sf + 4, kb > 0 || q > 0);
                tc::mma_commit<2>(&empty[s]);
            }
            tc::mma_commit<2>(&done);
        }
        if (gave_up) {
            // the tensor cores may still be at work
            tc::mma_commit<2>(&ended);
            int ignore = 0;
            tc::bar_wait(&ended, 0, &ignore);
        }
    } else if (warp < kPairWarps) {
        // eight warps: four groups of 32 lanes, two halves of the columns
        constexpr uint32_t kCols = kOut == PS_DTYPE_F32 ? 32 : 64, kChunks = kPairTile / 2 / kCols;
        const uint32_t quarter = warp & 3, half = warp >> 2;
        unsigned char* const buf = base_ptr + kPairStages * kPairStageBytes + warp * kStoreBytes;
        uint32_t it = 0;
        bool good = true;
        for (uint32_t t = first; t < tiles; t += step, ++it) {
            uint32_t tm, tn;
            tile_at(p, t, &tm, &tn);
            const uint32_t row0 = tm * kPairTile + rank * kTile + quarter * 32;
            if (p.bias != nullptr) {
                for (uint32_t i = lane; i < kPairTile / 2; i += 32) {
                    const uint32_t col = tn * kPairTile + half * (kPairTile / 2) + i;
                    s_bias[warp][i] = col < p.n ? bias_at(p, col) : 0.f;
                }
                __syncwarp();
            }
            good = good && tc::bar_wait(&done, it & 1, &gave_up);
            good = __all_sync(0xffffffffu, good);
            tc::fence_after();
            const uint32_t acc = tmem + (it & 1) * kAccStride + (quarter << 21);
            for (uint32_t c = 0; c < kChunks; ++c) {
                // the overlapping columns first: the last ones of the lower accumulator, the first of the upper
                const uint32_t in_half = (it & 1) ? c : kChunks - 1 - c, at = half * (kPairTile / 2) + in_half * kCols;
                const uint32_t col = tn * kPairTile + at;
                stage_row<kOut>(buf, p, &s_bias[warp][in_half * kCols], acc + at, good, c == 0, &drained);
                if (p.vec) tc::fence_to_async();
                __syncwarp();
                if (row0 < p.m && col < p.n) {
                    // a box reaches over the last column in steps of 16 bytes: what is behind it would be written
                    if (p.vec && (p.n_vec || col + kCols <= p.n)) {
                        if (lane == 0) tc::store_box(&map_out, tc::smem_u32(buf), (int)col, (int)row0);
                    } else {
                        store_rows<kOut>(p, buf, row0, col);
                    }
                }
                __syncwarp();
            }
        }
        if (lane == 0) tc::store_wait_read<0>();
        tc::fence_before();
    }
    __syncwarp();
    __syncthreads();
    tc::cluster_sync();
    if (warp == kPairWarps + 1) tc::tmem_free<2>(tmem, 512);
    if (threadIdx.x == 0 && gave_up) atomicAdd(&g_gave_up, 1u);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encoder()
{
    static const EncodeTiled fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q);
        if (e != cudaSuccess || q != cudaDriverEntryPointSuccess) {
            ps_internal::set_cuda_error((int)e);
            cudaGetLastError();
            f = nullptr;
        }
        return (EncodeTiled)f;
    }();
    return fn;
}

int encode(CUtensorMap* m, CUtensorMapDataType type, const void* p, uint64_t inner, uint64_t rows, uint64_t row_bytes,
           uint32_t box_inner, uint32_t box_rows, CUtensorMapSwizzle swizzle)
{
    const EncodeTiled fn = encoder();
    if (fn == nullptr) return PS_ERR_CUDA;
    const cuuint64_t dims[2] = {inner, rows}, strides[1] = {row_bytes};
    const cuuint32_t box[2] = {box_inner, box_rows}, step[2] = {1, 1};
    const CUresult r = fn(m, type, 2, const_cast<void*>(p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? PS_OK : PS_ERR_INVALID;
}

int check_operand(const ps_block_operand* o, uint64_t outer, uint64_t k)
{
    if (o == nullptr || o->data == nullptr || o->scales == nullptr) return PS_ERR_INVALID;
    if (o->fmt != PS_FP8_E4M3 && o->fmt != PS_FP8_E5M2) return PS_ERR_INVALID;
    if (o->k_dim != 0 && o->k_dim != 1) return PS_ERR_INVALID;
    if (o->ld < (o->k_dim ? k : outer)) return PS_ERR_INVALID;
    if (o->ld % 16 || (uintptr_t)o->data % 16 || (uintptr_t)o->scales % 16) return PS_ERR_ALIGN;
    return PS_OK;
}

int encode_operand(const ps_block_operand* o, uint64_t outer, uint64_t k, uint32_t blocks, CUtensorMap* data,
                   CUtensorMap* scales)
{
    int rc = encode(data, CU_TENSOR_MAP_DATA_TYPE_UINT8, o->data, o->k_dim ? k : outer, o->k_dim ? outer : k, o->ld,
                    kTile, kTile, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc != PS_OK) return rc;
    return encode(scales, CU_TENSOR_MAP_DATA_TYPE_INT32, o->scales, kScaleBytes / 4, (uint64_t)((k + 511) / 512) * blocks,
                  kScaleBytes, kScaleBytes / 4, 1, CU_TENSOR_MAP_SWIZZLE_NONE);
}

uint32_t ceil_div(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }

// CTAs that share a tile of 128 x 128 along k: as many as fill the SMs, doubled while each has four k blocks: two
// blocks each at least.
uint32_t splits_of(uint64_t tiles, uint32_t n_kb, int sms)
{
    uint32_t splits = 1;
    while (splits < 8 && tiles * splits < (uint64_t)sms && splits * 4 <= n_kb) splits *= 2;
    return splits;
}

// 256 x 256 tiles on pairs of SMs, or 128 x 128 tiles, two to an SM and split along k, whichever should be done first.
// In hundredths of a microsecond, from a fit to measured products: 400 and 32 for each round and k block, or 650 and 60 (the
// small tile reads twice as much for a product, and its cluster meets twice).  Measured, large / small: 300 x 300 x 16000
// 73 / 18 us; 1 x 6400 x 1600 8.1 / 7.8; 64 x 1600 x 800 6.1 / 8.6; 1024 x 1600 x 4800 16.1 / 17.1; 1 x 20480 x 5120
// 35 / 42; 1600 x 1600 x 16385 45 / 73; 4096 x 4800 x 1600 28 / 59.
bool use_pairs(uint32_t m, uint32_t n, uint32_t n_kb, int sms)
{
    if (n_kb == 0) return false;
    const uint64_t large = (uint64_t)ceil_div(m, kPairTile) * ceil_div(n, kPairTile), pairs = (uint64_t)sms / 2;
    const uint64_t small = (uint64_t)ceil_div(m, kTile) * ceil_div(n, kTile), splits = splits_of(small, n_kb, sms);
    const uint64_t as_pairs = 400 + 32 * ((large + pairs - 1) / pairs) * n_kb;
    const uint64_t as_split = 650 + 60 * ((small * splits + 2 * sms - 1) / (2 * sms)) * ((n_kb + splits - 1) / splits);
    return as_pairs <= as_split;
}

template <int kOut>
int launch_pairs_as(const ProductArgs& p, const CUtensorMap* maps, const CUtensorMap& out, uint32_t grid, cudaStream_t st)
{
    static std::atomic<uint64_t> seen{0};
    const int rc = allow_smem(block_matmul_pair_kernel<kOut>, kPairSmem, seen);
    if (rc != PS_OK) return rc;
    launch_behind(block_matmul_pair_kernel<kOut>, grid, kPairThreads, kPairSmem, 2, st, maps[0], maps[1], maps[2],
                       maps[3], out, p);
    return ps_internal::after_launch();
}

int launch_pairs(ProductArgs& p, const CUtensorMap* maps, const ps_block_operand* a, const ps_block_operand* b,
                 uint64_t osize, int sms, cudaStream_t st)
{
    p.tiles_m = ceil_div(p.m, kPairTile), p.tiles_n = ceil_div(p.n, kPairTile);
    p.idesc = tc::mx_idesc(256, 256, a->fmt, b->fmt, !a->k_dim, !b->k_dim);
    const uint64_t tiles = (uint64_t)p.tiles_m * p.tiles_n;
    if (tiles > 0x7fffffffull) return PS_ERR_LIMIT;
    CUtensorMap out;
    memset(&out, 0, sizeof(out));
    if (p.vec) {
        const CUtensorMapDataType type = p.out_dtype == PS_DTYPE_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                         : p.out_dtype == PS_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                       : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
        const int rc = encode(&out, type, p.out, p.n, p.m, p.ldo * osize, (uint32_t)(128 / osize), 32,
                              CU_TENSOR_MAP_SWIZZLE_128B);
        if (rc != PS_OK) return rc;
    }
    const uint64_t pairs = (uint64_t)sms / 2;
    const uint32_t grid = 2 * (uint32_t)(tiles < pairs ? tiles : pairs);
    if (p.out_dtype == PS_DTYPE_F16) return launch_pairs_as<PS_DTYPE_F16>(p, maps, out, grid, st);
    if (p.out_dtype == PS_DTYPE_BF16) return launch_pairs_as<PS_DTYPE_BF16>(p, maps, out, grid, st);
    return launch_pairs_as<PS_DTYPE_F32>(p, maps, out, grid, st);
}

int launch_split(ProductArgs& p, const CUtensorMap* maps, const ps_block_operand* a, const ps_block_operand* b, int sms,
                 cudaStream_t st)
{
    p.tiles_m = ceil_div(p.m, kTile), p.tiles_n = ceil_div(p.n, kTile);
    if (p.n_kb > 0) p.idesc = tc::mx_idesc(128, 128, a->fmt, b->fmt, !a->k_dim, !b->k_dim);
    const uint64_t tiles = (uint64_t)p.tiles_m * p.tiles_n;
    const uint32_t splits = splits_of(tiles, p.n_kb, sms);
    if (tiles * splits > 0x7fffffffull) return PS_ERR_LIMIT;
    static std::atomic<uint64_t> seen{0};
    const int rc = allow_smem(block_matmul_split_kernel, kSplitSmem, seen);
    if (rc != PS_OK) return rc;
    launch_behind(block_matmul_split_kernel, (uint32_t)(tiles * splits), kSplitThreads, kSplitSmem, splits, st, maps[0],
                       maps[1], maps[2], maps[3], p, splits);
    return ps_internal::after_launch();
}

}  // namespace

extern "C" {

int ps_block_matmul(const ps_block_operand* a, const ps_block_operand* b, uint32_t m, uint32_t n, uint32_t k,
                    const void* bias_dev, int bias_dtype, void* out_dev, int out_dtype, uint64_t ldo, void* stream)
{
    if (out_dtype < PS_DTYPE_F16 || out_dtype > PS_DTYPE_F32) return PS_ERR_INVALID;
    if (bias_dev != nullptr && (bias_dtype < PS_DTYPE_F16 || bias_dtype > PS_DTYPE_F32)) return PS_ERR_INVALID;
    if (m == 0 || n == 0) return PS_OK;
    if (out_dev == nullptr || ldo < n) return PS_ERR_INVALID;
    if (m > 0x7fffff00u || n > 0x7fffff00u || k > 0x7fffff00u) return PS_ERR_LIMIT;
    const uint64_t osize = out_dtype == PS_DTYPE_F32 ? 4 : 2;
    if ((uintptr_t)out_dev % osize) return PS_ERR_ALIGN;
    ProductArgs p;
    memset(&p, 0, sizeof(p));
    CUtensorMap maps[4];
    memset(maps, 0, sizeof(maps));
    p.scale_blocks_a = ceil_div(m, kTile), p.scale_blocks_b = ceil_div(n, kTile);
    if (k > 0) {
        int rc = check_operand(a, m, k);
        if (rc == PS_OK) rc = check_operand(b, n, k);
        if (rc != PS_OK) return rc;
        if ((uint64_t)ceil_div(k, 512) * (p.scale_blocks_a > p.scale_blocks_b ? p.scale_blocks_a : p.scale_blocks_b) >
            0x7fffffffull)
            return PS_ERR_LIMIT;
        rc = encode_operand(a, m, k, p.scale_blocks_a, &maps[0], &maps[2]);
        if (rc == PS_OK) rc = encode_operand(b, n, k, p.scale_blocks_b, &maps[1], &maps[3]);
        if (rc != PS_OK) return rc;
        p.a_k_inner = a->k_dim, p.b_k_inner = b->k_dim;
    }
    p.bias = bias_dev, p.bias_dtype = bias_dtype, p.out = out_dev, p.out_dtype = out_dtype, p.ldo = ldo;
    p.m = m, p.n = n, p.n_kb = ceil_div(k, kTile);
    p.n_vec = (n * osize) % 16 == 0;
    p.vec = (uintptr_t)out_dev % 16 == 0 && (ldo * osize) % 16 == 0;
    const int sms = ps_internal::sm_count();
    if (sms < 0) return sms;

    if (use_pairs(m, n, p.n_kb, sms)) return launch_pairs(p, maps, a, b, osize, sms, (cudaStream_t)stream);
    return launch_split(p, maps, a, b, sms, (cudaStream_t)stream);
}

int ps_block_matmul_gave_up(uint32_t* count)
{
    if (count == nullptr) return PS_ERR_INVALID;
    const cudaError_t e = cudaMemcpyFromSymbol(count, g_gave_up, sizeof(*count));
    if (e != cudaSuccess) {
        ps_internal::set_cuda_error((int)e);
        cudaGetLastError();
        return PS_ERR_CUDA;
    }
    return PS_OK;
}

}  // extern "C"
