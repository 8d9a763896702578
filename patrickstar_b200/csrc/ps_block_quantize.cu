// Quantization into 8-bit floating point with one power-of-two scale for each
// block of 128 elements (1 x 128, 128 x 1 or 128 x 128).
//
//   amax = the largest finite magnitude of the block = m 2^E, 1 <= m < 2
//   e    = E - top + [m > 1.75]        top = 8 (e4m3: 448 = 1.75 2^8) or 15 (e5m2: 57344 = 1.75 2^15)
//   q    = x 2^-e rounded to nearest even
//
// The product with a power of two is exact, so the only rounding is the one to
// 8 bits, and the scale byte e + 127 is what the tensor core takes as a scale.
// The byte is held in [1, 254]; a block whose amax is zero or subnormal has
// byte 1.  An infinite or NaN element becomes NaN in e4m3 (which has no
// infinity) and stays itself in e5m2: a gradient that overflowed is seen by
// the overflow test behind the product.
//
// One CTA takes a 128 x 128 tile into registers with all of its loads in
// flight at once, reduces the magnitudes (two 16-bit ones to a word), and writes
// every output the caller wants from that one read: 2 bytes in and 1 or 2 bytes
// out per 16-bit element.  HBM-bound where it gets by with few instructions: rows
// alone 5.9 TB/s, columns alone 6.6 TB/s, both 5.2 to 5.8 TB/s (8192 x 5120 and
// 8192 x 20480 fp16), tiles 6.2 TB/s.
#include "ps_b200.h"

#include "ps_internal.h"
#include "ps_launch.cuh"
#include "ps_pair.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <type_traits>

namespace {

constexpr int kBlock = 128;
constexpr int kThreads = 256;
constexpr int kRowsPerThread = 8;  // 16 threads across 128 columns, 16 down, 8 rows each
constexpr int kWarps = kThreads / 32;

// ---------------------------------------------------------------------------
// eight consecutive elements of a row, as loaded, and magnitudes in the same words
// ---------------------------------------------------------------------------
template <typename T>
struct Vec8 {  // 16-bit types: two to a word
    static constexpr int kWords = 4;
    static constexpr uint32_t kInf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    uint32_t w[4];
    __device__ __forceinline__ void set(int j, const T* p)
    {
        w[j >> 1] |= (uint32_t)*reinterpret_cast<const unsigned short*>(p) << (16 * (j & 1));
    }
    __device__ __forceinline__ void get(float (&f)[8]) const
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same<T, __half>::value) {
                const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                f[2 * i] = t.x, f[2 * i + 1] = t.y;
            } else {
                f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
    // the larger of `m` and the magnitude of x; a NaN gives way
    static __device__ __forceinline__ uint32_t raise(uint32_t m, uint32_t x)
    {
        const T2 r = __hmax2(__habs2(*reinterpret_cast<const T2*>(&x)), *reinterpret_cast<const T2*>(&m));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    static __device__ __forceinline__ bool has_inf(uint32_t m) { return (m & 0xffffu) == kInf || (m >> 16) == kInf; }
    static __device__ __forceinline__ uint32_t without_inf(uint32_t x)
    {
        const uint32_t m = x & 0x7fff7fffu;
        return x & ~(((m & 0xffffu) == kInf ? 0xffffu : 0u) | ((m >> 16) == kInf ? 0xffff0000u : 0u));
    }
    // of the two magnitudes in a word
    static __device__ __forceinline__ uint32_t fold(uint32_t m) { return max(m & 0xffffu, m >> 16); }
    static __device__ __forceinline__ float magnitude(uint32_t m)  // in the low half
    {
        if constexpr (std::is_same<T, __half>::value)
            return __half2float(__ushort_as_half((unsigned short)m));
        else
            return __uint_as_float(m << 16);
    }
};
template <>
struct Vec8<float> {  // one to a word
    static constexpr int kWords = 8;
    static constexpr uint32_t kInf = 0x7f800000u;
    uint32_t w[8];
    __device__ __forceinline__ void set(int j, const float* p) { w[j] = __float_as_uint(*p); }
    __device__ __forceinline__ void get(float (&f)[8]) const
    {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
    }
    static __device__ __forceinline__ uint32_t raise(uint32_t m, uint32_t x)
    {
        return __float_as_uint(fmaxf(fabsf(__uint_as_float(x)), __uint_as_float(m)));
    }
    static __device__ __forceinline__ bool has_inf(uint32_t m) { return m == kInf; }
    static __device__ __forceinline__ uint32_t without_inf(uint32_t x) { return (x & 0x7fffffffu) == kInf ? 0u : x; }
    static __device__ __forceinline__ uint32_t fold(uint32_t m) { return m; }
    static __device__ __forceinline__ float magnitude(uint32_t m) { return __uint_as_float(m); }
};

// scale byte of a finite magnitude
template <int kFmt>
__device__ __forceinline__ uint32_t scale_byte(float amax)
{
    constexpr int kTop = kFmt == PS_FP8_E4M3 ? 8 : 15;
    const uint32_t u = __float_as_uint(amax);
    const int b = (int)(u >> 23) - kTop + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return b < 1 ? 1u : (uint32_t)b;
}
// 2^-(byte - 127).  The largest byte a finite float gives is 247, so this is a normal number.
__device__ __forceinline__ float scale_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

template <int kFmt>
__device__ __forceinline__ uint32_t to_fp8x2(float lo, float hi)
{
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE,
                                              kFmt == PS_FP8_E4M3 ? __NV_E4M3 : __NV_E5M2);
}
// The conversion saturates an infinity; this is what the format has for an element that is not finite.
template <int kFmt>
__device__ __forceinline__ uint32_t nonfinite_fp8(float v)
{
    const uint32_t u = __float_as_uint(v);
    const uint32_t sign = (u >> 24) & 0x80u;
    if (kFmt == PS_FP8_E5M2 && (u & 0x7fffffffu) == 0x7f800000u) return sign | 0x7cu;
    return sign | 0x7fu;
}

// Byte of block `kb` (along the contracted dimension) of outer element `o`: see ps_block_quantize.
__device__ __forceinline__ size_t scale_index(uint32_t o, uint32_t kb, uint32_t outer_blocks)
{
    const size_t g = (size_t)(kb >> 2) * outer_blocks + (o >> 7);
    return ((g * 32 + (o & 31)) * 4 + ((o >> 5) & 3)) * 4 + (kb & 3);
}

// Writes the byte of block kb and, when it is the last one, zeros behind it to the end of its group of four.
__device__ __forceinline__ void put_scale(uint8_t* s, uint32_t o, uint32_t kb, uint32_t n_kb, uint32_t outer_blocks,
                                          uint32_t byte)
{
    uint8_t* p = s + scale_index(o, kb, outer_blocks);
    *p = (uint8_t)byte;
    if (kb + 1 == n_kb)
        for (uint32_t k = kb + 1; k & 3; ++k) *++p = 0;
}

struct QuantArgs {
    const void* x;
    uint64_t ld, ldq;
    uint32_t rows, cols, row_blocks, col_blocks;
    uint8_t *q1, *q0, *s1, *s0;
    float* colsum;
    int vec;  // rows start on 16-byte boundaries
};

__host__ __device__ constexpr bool has_row(int mode) { return mode == PS_BLOCKS_ROW || mode == PS_BLOCKS_ROW_COL; }
__host__ __device__ constexpr bool has_col(int mode) { return mode == PS_BLOCKS_COL || mode == PS_BLOCKS_ROW_COL; }

// CTAs an SM holds: a tile is 32 registers a thread in 16 bits, 64 in 32.  (Both directions of 8192 x 5120 fp16: 35 us
// with four CTAs of 64 registers, some of them spilled, 38 us with three.)
template <typename T>
__host__ __device__ constexpr int ctas_of()
{
    return sizeof(T) == 2 ? 4 : 2;
}

struct Shared {
    uint32_t key[kWarps][16][8];
    float inv[kBlock];
    float sum[kWarps][kBlock];
};

template <typename T, int kMode, int kFmt, bool kSum>
__device__ __forceinline__ void quantize_tile(const QuantArgs& a, uint32_t tile, Shared& sh)
{
    using V = Vec8<T>;
    constexpr bool kRow = has_row(kMode), kCol = has_col(kMode), kTile = kMode == PS_BLOCKS_TILE;
    const uint32_t cb = tile % a.col_blocks, rb = tile / a.col_blocks;
    const uint32_t cg = threadIdx.x & 15, rg = threadIdx.x >> 4;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t c0 = cb * kBlock + cg * 8, r0 = rb * kBlock + rg;
    const T* x = reinterpret_cast<const T*>(a.x);

    V v[kRowsPerThread];
    const bool whole = a.vec && c0 + 8 <= a.cols;
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
        const uint32_t r = r0 + 16 * i;
#pragma unroll
        for (int k = 0; k < V::kWords; ++k) v[i].w[k] = 0u;
        if (r < a.rows) {
            const T* p = x + (size_t)r * a.ld + c0;
            if (whole) {
#pragma unroll
                for (int k = 0; k < V::kWords / 4; ++k) {
                    const uint4 q = __ldcs(reinterpret_cast<const uint4*>(p) + k);
                    v[i].w[4 * k] = q.x, v[i].w[4 * k + 1] = q.y, v[i].w[4 * k + 2] = q.z, v[i].w[4 * k + 3] = q.w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (c0 + j < a.cols) v[i].set(j, p + j);
            }
        }
    }

    // magnitudes: rk[i] over the 8 elements of row i, ck[k] over the thread's 8 rows
    uint32_t rk[kRowsPerThread], ck[V::kWords];
    bool odd = false;  // holds an infinity (a NaN gives way to any number, and converts to one)
    auto maxima = [&](auto&& of) {
#pragma unroll
        for (int k = 0; k < V::kWords; ++k) ck[k] = 0;
#pragma unroll
        for (int i = 0; i < kRowsPerThread; ++i) {
            rk[i] = 0;
#pragma unroll
            for (int k = 0; k < V::kWords; ++k) {
                if (kRow) rk[i] = V::raise(rk[i], of(v[i].w[k]));
                if (kCol || kTile) ck[k] = V::raise(ck[k], of(v[i].w[k]));
            }
        }
        uint32_t all = 0;
        if constexpr (kCol || kTile) {
#pragma unroll
            for (int k = 0; k < V::kWords; ++k) all = V::raise(all, ck[k]);
        } else {
#pragma unroll
            for (int i = 0; i < kRowsPerThread; ++i) all = V::raise(all, rk[i]);
        }
        return all;
    };
    const uint32_t thread_max = maxima([](uint32_t w) { return w; });
    if (V::has_inf(thread_max)) {
        odd = true;
        maxima([](uint32_t w) { return V::without_inf(w); });
    }

    float row_inv[kRowsPerThread];
    if constexpr (kRow) {
        if constexpr (sizeof(T) == 2) {  // two rows to a word
#pragma unroll
            for (int i = 0; i < kRowsPerThread; i += 2) {
                uint32_t m = V::fold(rk[i]) | (V::fold(rk[i + 1]) << 16);
#pragma unroll
                for (int d = 1; d < 16; d <<= 1) m = V::raise(m, __shfl_xor_sync(0xffffffffu, m, d));
                rk[i] = m & 0xffffu, rk[i + 1] = m >> 16;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kRowsPerThread; ++i)
#pragma unroll
                for (int d = 1; d < 16; d <<= 1) rk[i] = V::raise(rk[i], __shfl_xor_sync(0xffffffffu, rk[i], d));
        }
        uint32_t mine = 0;  // eight of the sixteen lanes of a row group write one row's byte each
#pragma unroll
        for (int i = 0; i < kRowsPerThread; ++i) {
            const uint32_t byte = scale_byte<kFmt>(V::magnitude(rk[i]));
            row_inv[i] = scale_inverse(byte);
            if (cg == i) mine = byte;
        }
        if (cg < kRowsPerThread) {
            const uint32_t r = r0 + 16 * cg;
            put_scale(a.s1, r, cb, a.col_blocks, a.row_blocks, r < a.rows ? mine : 0u);
        }
    }
    float col_inv[8];
    if constexpr (kCol) {
#pragma unroll
        for (int k = 0; k < V::kWords; ++k) {
            ck[k] = V::raise(ck[k], __shfl_xor_sync(0xffffffffu, ck[k], 16));
            if (lane < 16) sh.key[warp][cg][k] = ck[k];
        }
        __syncthreads();
        if (threadIdx.x < kBlock) {
            const uint32_t c = cb * kBlock + threadIdx.x, j = threadIdx.x & 7;
            uint32_t m = 0;
#pragma unroll
            for (int w = 0; w < kWarps; ++w)
                m = V::raise(m, sh.key[w][threadIdx.x >> 3][sizeof(T) == 2 ? j >> 1 : j]);
            if (sizeof(T) == 2) m = (m >> (16 * (j & 1))) & 0xffffu;
            const uint32_t byte = scale_byte<kFmt>(V::magnitude(m));
            sh.inv[threadIdx.x] = scale_inverse(byte);
            put_scale(a.s0, c, rb, a.row_blocks, a.col_blocks, c < a.cols ? byte : 0u);
        }
        __syncthreads();
        const float4 lo = *reinterpret_cast<const float4*>(&sh.inv[cg * 8]), hi = *reinterpret_cast<const float4*>(&sh.inv[cg * 8 + 4]);
        col_inv[0] = lo.x, col_inv[1] = lo.y, col_inv[2] = lo.z, col_inv[3] = lo.w;
        col_inv[4] = hi.x, col_inv[5] = hi.y, col_inv[6] = hi.z, col_inv[7] = hi.w;
    }
    if constexpr (kTile) {
        uint32_t m = 0;
#pragma unroll
        for (int k = 0; k < V::kWords; ++k) m = V::raise(m, ck[k]);
        m = __reduce_max_sync(0xffffffffu, V::fold(m));  // magnitudes order like their bits
        if (lane == 0) sh.key[warp][0][0] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; ++w) m = max(m, sh.key[w][0][0]);
        const uint32_t byte = scale_byte<kFmt>(V::magnitude(m));
#pragma unroll
        for (int i = 0; i < kRowsPerThread; ++i) row_inv[i] = scale_inverse(byte);
        if (threadIdx.x < kBlock) {
            const uint32_t r = rb * kBlock + threadIdx.x, c = cb * kBlock + threadIdx.x;
            put_scale(a.s1, r, cb, a.col_blocks, a.row_blocks, r < a.rows ? byte : 0u);
            put_scale(a.s0, c, rb, a.row_blocks, a.col_blocks, c < a.cols ? byte : 0u);
        }
    }

    // every row is unpacked once, for all that is made of it
    Pair sums[4] = {Pair(0.f, 0.f), Pair(0.f, 0.f), Pair(0.f, 0.f), Pair(0.f, 0.f)};
    uint8_t* q1 = a.q1 + (size_t)r0 * a.ldq + c0;
    uint8_t* q0 = a.q0 + (size_t)r0 * a.ldq + c0;
    auto convert = [&](const float(&f)[8], const Pair(&inv)[4], uint8_t* q) {
        uint32_t out[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float2 lo = mul2(Pair(f[4 * h], f[4 * h + 1]), inv[2 * h]).get();
            const float2 hi = mul2(Pair(f[4 * h + 2], f[4 * h + 3]), inv[2 * h + 1]).get();
            out[h] = to_fp8x2<kFmt>(lo.x, lo.y) | (to_fp8x2<kFmt>(hi.x, hi.y) << 16);
        }
        if (odd) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (!(fabsf(f[j]) < __int_as_float(0x7f800000)))
                    out[j >> 2] = (out[j >> 2] & ~(0xffu << (8 * (j & 3)))) | (nonfinite_fp8<kFmt>(f[j]) << (8 * (j & 3)));
        }
        *reinterpret_cast<uint2*>(q) = make_uint2(out[0], out[1]);
    };
    Pair col2[4];
    if constexpr (kCol) {
#pragma unroll
        for (int j = 0; j < 4; ++j) col2[j] = Pair(col_inv[2 * j], col_inv[2 * j + 1]);
    }
    const bool here = c0 < a.cols;
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
        float f[8];
        v[i].get(f);
        if constexpr (kSum) {
#pragma unroll
            for (int j = 0; j < 4; ++j) sums[j] = add2(sums[j], Pair(f[2 * j], f[2 * j + 1]));
        }
        if (here && r0 + 16 * i < a.rows) {
            if constexpr (kRow || kTile) {
                const Pair one(row_inv[i], row_inv[i]);
                const Pair all[4] = {one, one, one, one};
                convert(f, all, q1);
            }
            if constexpr (kCol) convert(f, col2, q0);
        }
        q1 += 16 * a.ldq, q0 += 16 * a.ldq;
    }

    if constexpr (kSum) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float2 t = sums[j].get();
            t.x += __shfl_xor_sync(0xffffffffu, t.x, 16), t.y += __shfl_xor_sync(0xffffffffu, t.y, 16);
            if (lane < 16) sh.sum[warp][cg * 8 + 2 * j] = t.x, sh.sum[warp][cg * 8 + 2 * j + 1] = t.y;
        }
        __syncthreads();
        if (threadIdx.x < kBlock) {
            const uint32_t c = cb * kBlock + threadIdx.x;
            float t = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) t += sh.sum[w][threadIdx.x];
            if (c < a.cols) a.colsum[(size_t)rb * a.cols + c] = t;
        }
    }
}

template <typename T, int kMode, int kFmt, bool kSum>
__global__ void __launch_bounds__(kThreads, ctas_of<T>()) block_quantize_kernel(const QuantArgs a)
{
    __shared__ Shared sh;
    cudaTriggerProgrammaticLaunchCompletion();
    cudaGridDependencySynchronize();
    quantize_tile<T, kMode, kFmt, kSum>(a, blockIdx.x, sh);
}

// Two matrices in one launch: the input of a layer (kMode) and, behind its `split` tiles, the weight.
template <typename T, int kMode>
__global__ void __launch_bounds__(kThreads, ctas_of<T>()) quantize_layer_kernel(const QuantArgs x, const QuantArgs w, uint32_t split)
{
    __shared__ Shared sh;
    cudaTriggerProgrammaticLaunchCompletion();
    cudaGridDependencySynchronize();
    if (blockIdx.x < split)
        quantize_tile<T, kMode, PS_FP8_E4M3, false>(x, blockIdx.x, sh);
    else
        quantize_tile<T, PS_BLOCKS_TILE, PS_FP8_E4M3, false>(w, blockIdx.x - split, sh);
}

// Sums of a column's blocks, in order, in 64 bits: one thread a column.
template <typename T>
__global__ void column_sum_kernel(const float* partial, uint32_t blocks, uint32_t cols, T* out)
{
    const uint32_t c = blockIdx.x * blockDim.x + threadIdx.x;
    cudaGridDependencySynchronize();
    if (c >= cols) return;
    double t = 0.0;
#pragma unroll 8
    for (uint32_t b = 0; b < blocks; ++b) t += (double)partial[(size_t)b * cols + c];
    out[c] = (T)(float)t;
}

template <typename T, int kFmt>
void launch(int mode, const QuantArgs& a, uint32_t tiles, cudaStream_t st)
{
    if (mode == PS_BLOCKS_ROW)
        launch_behind(block_quantize_kernel<T, PS_BLOCKS_ROW, kFmt, false>, tiles, kThreads, 0, 0, st, a);
    else if (mode == PS_BLOCKS_COL)
        launch_behind(block_quantize_kernel<T, PS_BLOCKS_COL, kFmt, false>, tiles, kThreads, 0, 0, st, a);
    else if (mode == PS_BLOCKS_TILE)
        launch_behind(block_quantize_kernel<T, PS_BLOCKS_TILE, kFmt, false>, tiles, kThreads, 0, 0, st, a);
    else if (a.colsum == nullptr)
        launch_behind(block_quantize_kernel<T, PS_BLOCKS_ROW_COL, kFmt, false>, tiles, kThreads, 0, 0, st, a);
    else
        launch_behind(block_quantize_kernel<T, PS_BLOCKS_ROW_COL, kFmt, true>, tiles, kThreads, 0, 0, st, a);
}

template <typename T>
void launch(int fmt, int mode, const QuantArgs& a, uint32_t tiles, cudaStream_t st)
{
    if (fmt == PS_FP8_E4M3)
        launch<T, PS_FP8_E4M3>(mode, a, tiles, st);
    else
        launch<T, PS_FP8_E5M2>(mode, a, tiles, st);
}

// Checks a job and makes its arguments; *tiles is 0 where there is nothing to do.
int prepare(const ps_internal::QuantizeJob& j, QuantArgs* a, uint32_t* tiles)
{
    *tiles = 0;
    if (j.dtype < PS_DTYPE_F16 || j.dtype > PS_DTYPE_F32 || j.blocks < PS_BLOCKS_ROW || j.blocks > PS_BLOCKS_TILE)
        return PS_ERR_INVALID;
    if (j.fmt != PS_FP8_E4M3 && j.fmt != PS_FP8_E5M2) return PS_ERR_INVALID;
    if (j.colsum != nullptr && j.blocks != PS_BLOCKS_ROW_COL) return PS_ERR_INVALID;
    if (j.rows == 0 || j.cols == 0) return PS_OK;
    const bool row = has_row(j.blocks) || j.blocks == PS_BLOCKS_TILE, col = has_col(j.blocks);
    if (j.x == nullptr || (row && (j.q1 == nullptr || j.s1 == nullptr)) || (col && (j.q0 == nullptr || j.s0 == nullptr)) ||
        (j.blocks == PS_BLOCKS_TILE && j.s0 == nullptr))
        return PS_ERR_INVALID;
    if (j.ldq < j.cols) return PS_ERR_INVALID;
    const uint64_t esize = j.dtype == PS_DTYPE_F32 ? 4 : 2;
    if ((uintptr_t)j.x % esize || j.ldq % 16 || (row && (uintptr_t)j.q1 % 16) || (col && (uintptr_t)j.q0 % 16))
        return PS_ERR_ALIGN;
    a->x = j.x, a->ld = j.ld, a->ldq = j.ldq, a->rows = j.rows, a->cols = j.cols;
    a->row_blocks = (uint32_t)(((uint64_t)j.rows + kBlock - 1) / kBlock);
    a->col_blocks = (uint32_t)(((uint64_t)j.cols + kBlock - 1) / kBlock);
    a->q1 = (uint8_t*)j.q1, a->q0 = (uint8_t*)j.q0, a->s1 = (uint8_t*)j.s1, a->s0 = (uint8_t*)j.s0;
    a->colsum = j.colsum;
    a->vec = (uintptr_t)j.x % 16 == 0 && (j.ld * esize) % 16 == 0;
    const uint64_t n = (uint64_t)a->row_blocks * a->col_blocks;
    if (n > 0x7fffffffull || j.cols > 0xffffff00u || j.rows > 0xffffff00u) return PS_ERR_LIMIT;
    *tiles = (uint32_t)n;
    return PS_OK;
}

template <typename T>
void launch_layer(int mode, const QuantArgs& x, uint32_t x_tiles, const QuantArgs& w, uint32_t w_tiles, cudaStream_t st)
{
    if (mode == PS_BLOCKS_ROW)
        launch_behind(quantize_layer_kernel<T, PS_BLOCKS_ROW>, x_tiles + w_tiles, kThreads, 0, 0, st, x, w, x_tiles);
    else
        launch_behind(quantize_layer_kernel<T, PS_BLOCKS_ROW_COL>, x_tiles + w_tiles, kThreads, 0, 0, st, x, w, x_tiles);
}

}  // namespace

namespace ps_internal {

int quantize(const QuantizeJob& j, cudaStream_t st)
{
    QuantArgs a;
    uint32_t tiles;
    const int rc = prepare(j, &a, &tiles);
    if (rc != PS_OK || tiles == 0) return rc;
    if (j.dtype == PS_DTYPE_F16)
        launch<__half>(j.fmt, j.blocks, a, tiles, st);
    else if (j.dtype == PS_DTYPE_BF16)
        launch<__nv_bfloat16>(j.fmt, j.blocks, a, tiles, st);
    else
        launch<float>(j.fmt, j.blocks, a, tiles, st);
    return after_launch();
}

int quantize_layer(const QuantizeJob& x, const QuantizeJob& w, cudaStream_t st)
{
    QuantArgs ax, aw;
    uint32_t x_tiles, w_tiles;
    int rc = prepare(x, &ax, &x_tiles);
    if (rc == PS_OK) rc = prepare(w, &aw, &w_tiles);
    if (rc != PS_OK) return rc;
    if (x_tiles == 0 || w_tiles == 0 || x.dtype != w.dtype || (uint64_t)x_tiles + w_tiles > 0x7fffffffull) {
        rc = quantize(x, st);
        return rc == PS_OK ? quantize(w, st) : rc;
    }
    if (x.dtype == PS_DTYPE_F16)
        launch_layer<__half>(x.blocks, ax, x_tiles, aw, w_tiles, st);
    else if (x.dtype == PS_DTYPE_BF16)
        launch_layer<__nv_bfloat16>(x.blocks, ax, x_tiles, aw, w_tiles, st);
    else
        launch_layer<float>(x.blocks, ax, x_tiles, aw, w_tiles, st);
    return after_launch();
}

}  // namespace ps_internal

extern "C" {

int ps_block_quantize(const void* x_dev, int dtype, uint64_t ld, uint32_t rows, uint32_t cols, int blocks, int fmt,
                      void* q1_dev, void* s1_dev, void* q0_dev, void* s0_dev, uint64_t ldq, float* colsum_dev,
                      void* stream)
{
    return ps_internal::quantize({x_dev, dtype, ld, rows, cols, blocks, fmt, q1_dev, s1_dev, q0_dev, s0_dev, ldq, colsum_dev},
                                 (cudaStream_t)stream);
}

int ps_column_sum(const float* partial_dev, uint32_t blocks, uint32_t cols, void* out_dev, int dtype, void* stream)
{
    if (dtype < PS_DTYPE_F16 || dtype > PS_DTYPE_F32) return PS_ERR_INVALID;
    if (cols == 0) return PS_OK;
    if ((partial_dev == nullptr && blocks > 0) || out_dev == nullptr) return PS_ERR_INVALID;
    const uint32_t grid = (uint32_t)(((uint64_t)cols + 127) / 128);
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == PS_DTYPE_F16)
        launch_behind(column_sum_kernel<__half>, grid, 128, 0, 0, st, partial_dev, blocks, cols, (__half*)out_dev);
    else if (dtype == PS_DTYPE_BF16)
        launch_behind(column_sum_kernel<__nv_bfloat16>, grid, 128, 0, 0, st, partial_dev, blocks, cols, (__nv_bfloat16*)out_dev);
    else
        launch_behind(column_sum_kernel<float>, grid, 128, 0, 0, st, partial_dev, blocks, cols, (float*)out_dev);
    return ps_internal::after_launch();
}

}  // extern "C"
