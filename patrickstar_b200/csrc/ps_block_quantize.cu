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
// flight at once, reduces the magnitudes as integers (an IEEE magnitude orders
// like its bits, two 16-bit ones to a word), and writes every output the caller
// wants from that one read: 2 bytes in and 1 or 2 bytes out per 16-bit element.
// HBM-bound.
#include "ps_b200.h"

#include "ps_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace {

constexpr int kBlock = 128;
constexpr int kThreads = 256;
constexpr int kRowsPerThread = 8;  // 16 threads across 128 columns, 16 down, 8 rows each
constexpr int kWarps = kThreads / 32;

// ---------------------------------------------------------------------------
// eight consecutive elements of a row, as loaded
// ---------------------------------------------------------------------------
template <typename T>
struct Vec8;

template <>
struct Vec8<__half> {
    static constexpr int kWords = 4;  // two magnitudes in each
    static constexpr uint32_t kInf = 0x7c00u;
    uint32_t w[4];
    __device__ __forceinline__ uint32_t key(int i) const { return w[i] & 0x7fff7fffu; }
    __device__ __forceinline__ float value(int j) const
    {
        return __half2float(__ushort_as_half((unsigned short)(w[j >> 1] >> (16 * (j & 1)))));
    }
    __device__ __forceinline__ void set(int j, const __half* p)
    {
        w[j >> 1] |= (uint32_t)__half_as_ushort(*p) << (16 * (j & 1));
    }
};
template <>
struct Vec8<__nv_bfloat16> {
    static constexpr int kWords = 4;
    static constexpr uint32_t kInf = 0x7f80u;
    uint32_t w[4];
    __device__ __forceinline__ uint32_t key(int i) const { return w[i] & 0x7fff7fffu; }
    __device__ __forceinline__ float value(int j) const
    {
        return __uint_as_float((j & 1) ? (w[j >> 1] & 0xffff0000u) : (w[j >> 1] << 16));
    }
    __device__ __forceinline__ void set(int j, const __nv_bfloat16* p)
    {
        w[j >> 1] |= (uint32_t)__bfloat16_as_ushort(*p) << (16 * (j & 1));
    }
};
template <>
struct Vec8<float> {
    static constexpr int kWords = 8;  // one magnitude in each
    static constexpr uint32_t kInf = 0x7f800000u;
    uint32_t w[8];
    __device__ __forceinline__ uint32_t key(int i) const { return w[i] & 0x7fffffffu; }
    __device__ __forceinline__ float value(int j) const { return __uint_as_float(w[j]); }
    __device__ __forceinline__ void set(int j, const float* p) { w[j] = __float_as_uint(*p); }
};

template <typename T>
__device__ __forceinline__ uint32_t key_max(uint32_t a, uint32_t b)
{
    if constexpr (sizeof(T) == 2)
        return __vmaxu2(a, b);
    else
        return a > b ? a : b;
}
template <typename T>
__device__ __forceinline__ uint32_t drop_nonfinite(uint32_t k)
{
    if constexpr (sizeof(T) == 2)
        return k & ~__vcmpgeu2(k, Vec8<T>::kInf * 0x10001u);
    else
        return k >= Vec8<T>::kInf ? 0u : k;
}
// the larger of the magnitudes a word holds
template <typename T>
__device__ __forceinline__ uint32_t key_fold(uint32_t k)
{
    if constexpr (sizeof(T) == 2)
        return max(k & 0xffffu, k >> 16);
    else
        return k;
}
template <typename T>
__device__ __forceinline__ float key_float(uint32_t k)
{
    if constexpr (std::is_same<T, __half>::value)
        return __half2float(__ushort_as_half((unsigned short)k));
    else if constexpr (std::is_same<T, __nv_bfloat16>::value)
        return __uint_as_float(k << 16);
    else
        return __uint_as_float(k);
}

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

struct Shared {
    uint32_t key[kWarps][16][8];
    float sum[kWarps][kBlock];
};

template <typename T, int kMode, int kFmt, bool kSum>
__device__ __forceinline__ void quantize_tile(const QuantArgs& a, uint32_t tile, Shared& sh)
{
    using V = Vec8<T>;
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
    bool odd = false;  // holds an element that is not finite
    {
        uint32_t all = 0;
#pragma unroll
        for (int k = 0; k < V::kWords; ++k) ck[k] = 0;
#pragma unroll
        for (int i = 0; i < kRowsPerThread; ++i) {
            rk[i] = 0;
#pragma unroll
            for (int k = 0; k < V::kWords; ++k) {
                const uint32_t key = v[i].key(k);
                rk[i] = key_max<T>(rk[i], key);
                ck[k] = key_max<T>(ck[k], key);
            }
            all = key_max<T>(all, rk[i]);
        }
        odd = key_fold<T>(all) >= V::kInf;
        if (odd) {
#pragma unroll
            for (int k = 0; k < V::kWords; ++k) ck[k] = 0;
#pragma unroll
            for (int i = 0; i < kRowsPerThread; ++i) {
                rk[i] = 0;
#pragma unroll
                for (int k = 0; k < V::kWords; ++k) {
                    const uint32_t key = drop_nonfinite<T>(v[i].key(k));
                    rk[i] = key_max<T>(rk[i], key);
                    ck[k] = key_max<T>(ck[k], key);
                }
            }
        }
    }

    auto put_row = [&](uint8_t* q, int i, const float* inv, bool one) {
        const uint32_t r = r0 + 16 * i;
        if (r >= a.rows || c0 >= a.cols) return;
        uint32_t out[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int j = 4 * h;
            const uint32_t lo = to_fp8x2<kFmt>(v[i].value(j) * inv[one ? 0 : j], v[i].value(j + 1) * inv[one ? 0 : j + 1]);
            const uint32_t hi = to_fp8x2<kFmt>(v[i].value(j + 2) * inv[one ? 0 : j + 2], v[i].value(j + 3) * inv[one ? 0 : j + 3]);
            out[h] = lo | (hi << 16);
        }
        if (odd) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float f = v[i].value(j);
                if (!(fabsf(f) < __int_as_float(0x7f800000)))
                    out[j >> 2] = (out[j >> 2] & ~(0xffu << (8 * (j & 3)))) | (nonfinite_fp8<kFmt>(f) << (8 * (j & 3)));
            }
        }
        *reinterpret_cast<uint2*>(q + (size_t)r * a.ldq + c0) = make_uint2(out[0], out[1]);
    };

    if constexpr (has_row(kMode)) {
#pragma unroll
        for (int i = 0; i < kRowsPerThread; ++i) {
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) rk[i] = key_max<T>(rk[i], __shfl_xor_sync(0xffffffffu, rk[i], d));
            const uint32_t byte = scale_byte<kFmt>(key_float<T>(key_fold<T>(rk[i])));
            const float inv = scale_inverse(byte);
            put_row(a.q1, i, &inv, true);
            if (cg == 0) {
                const uint32_t r = r0 + 16 * i;
                put_scale(a.s1, r, cb, a.col_blocks, a.row_blocks, r < a.rows ? byte : 0u);
            }
        }
    }

    if constexpr (kSum) {
        float cs[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            cs[j] = 0.f;
#pragma unroll
            for (int i = 0; i < kRowsPerThread; ++i) cs[j] += v[i].value(j);
            cs[j] += __shfl_xor_sync(0xffffffffu, cs[j], 16);
        }
        if (lane < 16) {
#pragma unroll
            for (int j = 0; j < 8; ++j) sh.sum[warp][cg * 8 + j] = cs[j];
        }
    }

    if constexpr (has_col(kMode)) {
#pragma unroll
        for (int k = 0; k < V::kWords; ++k) {
            ck[k] = key_max<T>(ck[k], __shfl_xor_sync(0xffffffffu, ck[k], 16));
            if (lane < 16) sh.key[warp][cg][k] = ck[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < V::kWords; ++k) {
#pragma unroll
            for (int w = 0; w < kWarps; ++w) ck[k] = key_max<T>(ck[k], sh.key[w][cg][k]);
        }
        float inv[8];
        uint32_t byte[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t key = sizeof(T) == 2 ? (ck[j >> 1] >> (16 * (j & 1))) & 0xffffu : ck[j % V::kWords];
            byte[j] = scale_byte<kFmt>(key_float<T>(key));
            inv[j] = scale_inverse(byte[j]);
        }
#pragma unroll
        for (int i = 0; i < kRowsPerThread; ++i) put_row(a.q0, i, inv, false);
        if (rg == 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                put_scale(a.s0, c0 + j, rb, a.row_blocks, a.col_blocks, c0 + j < a.cols ? byte[j] : 0u);
        }
    } else if constexpr (kMode == PS_BLOCKS_TILE) {
        uint32_t key = 0;
#pragma unroll
        for (int k = 0; k < V::kWords; ++k) key = key_max<T>(key, ck[k]);
        key = __reduce_max_sync(0xffffffffu, key_fold<T>(key));
        if (lane == 0) sh.key[warp][0][0] = key;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; ++w) key = max(key, sh.key[w][0][0]);
        const uint32_t byte = scale_byte<kFmt>(key_float<T>(key));
        const float inv = scale_inverse(byte);
#pragma unroll
        for (int i = 0; i < kRowsPerThread; ++i) put_row(a.q1, i, &inv, true);
        if (threadIdx.x < kBlock) {
            const uint32_t r = rb * kBlock + threadIdx.x, c = cb * kBlock + threadIdx.x;
            put_scale(a.s1, r, cb, a.col_blocks, a.row_blocks, r < a.rows ? byte : 0u);
            put_scale(a.s0, c, rb, a.row_blocks, a.col_blocks, c < a.cols ? byte : 0u);
        }
    }

    if constexpr (kSum) {
        if constexpr (!has_col(kMode)) __syncthreads();
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
__global__ void __launch_bounds__(kThreads) block_quantize_kernel(const QuantArgs a)
{
    __shared__ Shared sh;
    cudaTriggerProgrammaticLaunchCompletion();
    quantize_tile<T, kMode, kFmt, kSum>(a, blockIdx.x, sh);
}

// Two matrices in one launch: the input of a layer (kMode) and, behind its `split` tiles, the weight.
template <typename T, int kMode>
__global__ void __launch_bounds__(kThreads) quantize_layer_kernel(const QuantArgs x, const QuantArgs w, uint32_t split)
{
    __shared__ Shared sh;
    cudaTriggerProgrammaticLaunchCompletion();
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
    if (c >= cols) return;
    double t = 0.0;
    for (uint32_t b = 0; b < blocks; ++b) t += (double)partial[(size_t)b * cols + c];
    out[c] = (T)(float)t;
}

template <typename T, int kFmt>
void launch(int mode, const QuantArgs& a, uint32_t tiles, cudaStream_t st)
{
    if (mode == PS_BLOCKS_ROW)
        block_quantize_kernel<T, PS_BLOCKS_ROW, kFmt, false><<<tiles, kThreads, 0, st>>>(a);
    else if (mode == PS_BLOCKS_COL)
        block_quantize_kernel<T, PS_BLOCKS_COL, kFmt, false><<<tiles, kThreads, 0, st>>>(a);
    else if (mode == PS_BLOCKS_TILE)
        block_quantize_kernel<T, PS_BLOCKS_TILE, kFmt, false><<<tiles, kThreads, 0, st>>>(a);
    else if (a.colsum == nullptr)
        block_quantize_kernel<T, PS_BLOCKS_ROW_COL, kFmt, false><<<tiles, kThreads, 0, st>>>(a);
    else
        block_quantize_kernel<T, PS_BLOCKS_ROW_COL, kFmt, true><<<tiles, kThreads, 0, st>>>(a);
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
        quantize_layer_kernel<T, PS_BLOCKS_ROW><<<x_tiles + w_tiles, kThreads, 0, st>>>(x, w, x_tiles);
    else
        quantize_layer_kernel<T, PS_BLOCKS_ROW_COL><<<x_tiles + w_tiles, kThreads, 0, st>>>(x, w, x_tiles);
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
        column_sum_kernel<<<grid, 128, 0, st>>>(partial_dev, blocks, cols, (__half*)out_dev);
    else if (dtype == PS_DTYPE_BF16)
        column_sum_kernel<<<grid, 128, 0, st>>>(partial_dev, blocks, cols, (__nv_bfloat16*)out_dev);
    else
        column_sum_kernel<<<grid, 128, 0, st>>>(partial_dev, blocks, cols, (float*)out_dev);
    return ps_internal::after_launch();
}

}  // extern "C"
