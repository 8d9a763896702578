// Divergence of a student's distribution from the top entries of a teacher's,
// and its gradient with respect to the student's logits.
//
// For a row of logits z over the vocabulary, temperature T and c = log2(e) / T:
//     M = max z,  e_v = 2^((z_v - M) c),  Z = sum e_v,  q_v = e_v / Z
// and for the k listed entries (idx_j, t_j), S the set of listed indices:
//     drop    p = softmax(t / T) over the listed;   p_r = 0
//     bucket  p_j = exp(t_j);   p_r = max(0, 1 - sum p_j),   q_r = sum of q_v, v not in S
//             (p_r = 0 where S is the whole vocabulary: rounding leaves no rest there)
//     loss = T^2 ( sum_j p_j (log p_j - log q_idx_j) + p_r (log p_r - log q_r) )
//     d loss / d z_v = T ( (sum p + p_r) q_v - sum_{j: idx_j = v} p_j - [v not in S] p_r q_v / q_r )
// where sum p + p_r is 1, but for a row that lists nothing (0) or a teacher that gives more than 1.
//
// One CTA takes a row: one pass with a running maximum and sum of its own in
// every thread, joined at the end; and for the gradient a second pass that reads
// the row again, from L2 when it follows the first (148 SMs hold a few rows each,
// 0.1 to 0.5 MB a row).  Subtracting the maximum before scaling keeps every
// finite logit in range (a row of the type's lowest value is a uniform one).
// The listed entries are few: one warp works on them in 64 bits beside the
// others' pass.  Their gradient is written over the row's after it, so the pass
// itself knows nothing of them.  HBM-bound: one read, and one write for the
// gradient; a power of two per element each pass.
#include "ps_b200.h"

#include "ps_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstring>

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;

struct DistillArgs {
    const void* z;
    uint64_t ldz;
    uint32_t rows, vocab, k;
    const void* idx;
    uint64_t ld_idx;
    const void* teacher;
    uint64_t ld_teacher;
    const uint8_t* mask;
    int idx_bytes, teacher_dtype;
    float temperature, weight;
    float* row_loss;
    float4* stats;       // per row: M, factors of e_v in the gradient for v in S and for the others, -
    const float* inv_n;  // 1 / rows that the mask keeps, or NULL: then inv_n_value
    float inv_n_value;
    void* grad;
    uint64_t ldg;
    const ps_scaler_state* scaler;  // gradient in the forward pass: of loss times this scale
    float* used_scale;              // ... which the forward pass leaves here
    const float* grad_out;          // gradient in the backward pass: of loss times this
    uint32_t grad_out_stride;
};

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T>
struct Type;
template <>
struct Type<__half> {
    static constexpr int kVec = 8;
    static __device__ __forceinline__ float load(const __half* p) { return __half2float(*p); }
    static __device__ __forceinline__ __half round(float f) { return __float2half_rn(f); }
    static __device__ __forceinline__ void unpack(const uint4& q, float (&f)[8])
    {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            f[2 * i] = t.x, f[2 * i + 1] = t.y;
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[8])
    {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <>
struct Type<__nv_bfloat16> {
    static constexpr int kVec = 8;
    static __device__ __forceinline__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
    static __device__ __forceinline__ __nv_bfloat16 round(float f) { return __float2bfloat16_rn(f); }
    static __device__ __forceinline__ void unpack(const uint4& q, float (&f)[8])
    {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[8])
    {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <>
struct Type<float> {
    static constexpr int kVec = 4;
    static __device__ __forceinline__ float load(const float* p) { return *p; }
    static __device__ __forceinline__ float round(float f) { return f; }
    static __device__ __forceinline__ void unpack(const uint4& q, float (&f)[4])
    {
        f[0] = __uint_as_float(q.x), f[1] = __uint_as_float(q.y), f[2] = __uint_as_float(q.z), f[3] = __uint_as_float(q.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[4])
    {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
};

__device__ __forceinline__ double teacher_at(const DistillArgs& a, uint64_t i)
{
    if (a.teacher_dtype == PS_DTYPE_F16) return (double)__half2float(reinterpret_cast<const __half*>(a.teacher)[i]);
    if (a.teacher_dtype == PS_DTYPE_BF16)
        return (double)__bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.teacher)[i]);
    return (double)reinterpret_cast<const float*>(a.teacher)[i];
}
__device__ __forceinline__ long long index_at(const DistillArgs& a, uint64_t i)
{
    return a.idx_bytes == 8 ? reinterpret_cast<const long long*>(a.idx)[i]
                            : (long long)reinterpret_cast<const int*>(a.idx)[i];
}
template <typename V>
__device__ __forceinline__ V warp_sum(V v)
{
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
__device__ __forceinline__ double warp_max(double v)
{
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        const double o = __shfl_xor_sync(0xffffffffu, v, d);
        v = (o > v || o != o) ? o : v;  // a NaN stays
    }
    return v;
}

// Where a row's elements lie: `head` of them before the first 16-byte boundary, `vecs` vectors, the rest.
struct RowShape {
    uint32_t head, vecs, tail;
};
template <typename T>
__device__ __forceinline__ RowShape row_shape(const T* p, uint32_t n)
{
    constexpr uint32_t E = Type<T>::kVec;
    RowShape s;
    s.head = (uint32_t)((16u - ((uintptr_t)p & 15u)) & 15u) / (uint32_t)sizeof(T);
    if (s.head > n) s.head = n;
    s.vecs = (n - s.head) / E;
    s.tail = n - s.head - s.vecs * E;
    return s;
}
// Place of element v in the bitmap of listed ones: vectors first, then head and tail.
template <typename T>
__device__ __forceinline__ uint32_t bit_of(const RowShape& s, uint32_t v)
{
    constexpr uint32_t E = Type<T>::kVec;
    if (v < s.head) return s.vecs * E + v;
    const uint32_t u = v - s.head;
    return u < s.vecs * E ? u : u + s.head;
}

// Running maximum and sums of one thread.
struct Running {
    float m = -INFINITY, out = 0.f, in = 0.f;
    __device__ __forceinline__ void raise(float top, float c)
    {
        if (top > m) {
            const float f = ex2((m - top) * c);
            out *= f, in *= f;
            m = top;
        }
    }
    __device__ __forceinline__ float origin() const { return m == -INFINITY ? 0.f : m; }
};

constexpr int kLoss = 1, kGrad = 2;

template <typename T, bool kBucket, int kWhat>
__global__ void __launch_bounds__(kThreads) distill_kernel(const DistillArgs a)
{
    constexpr int E = Type<T>::kVec;
    extern __shared__ uint32_t smem[];
    // listed entries: index (or -1), probability, logit; then the bitmap
    int* const s_idx = reinterpret_cast<int*>(smem);
    float* const s_p = reinterpret_cast<float*>(smem + a.k);
    float* const s_z = reinterpret_cast<float*>(smem + 2 * a.k);
    uint32_t* const s_bits = smem + 3 * a.k;
    __shared__ float s_m[kWarps], s_out[kWarps], s_in[kWarps];
    __shared__ double s_rest, s_mass;  // p_r, and sum p + p_r: 1 unless the teacher gives nothing, or too much
    __shared__ int s_bad;

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float c = (float)(1.4426950408889634 / (double)a.temperature);
    const double inv_t = 1.0 / (double)a.temperature;

    if ((kWhat & kLoss) == 0 && a.used_scale != nullptr && *a.used_scale == *a.grad_out)
        return;  // the forward pass wrote this gradient
    float scale = 1.f;
    if (kWhat & kGrad) {
        if (kWhat & kLoss) {
            scale = a.scaler->dynamic < 0 ? 1.f : (float)a.scaler->cur_scale;
            if (blockIdx.x == 0 && threadIdx.x == 0) *a.used_scale = scale;
        }
    }

    for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* const z = reinterpret_cast<const T*>(a.z) + (uint64_t)row * a.ldz;
        T* const g = reinterpret_cast<T*>(a.grad) + (uint64_t)row * a.ldg;
        const RowShape shape = row_shape(z, a.vocab);
        const bool same_offset = (((uintptr_t)z ^ (uintptr_t)g) & 15u) == 0;
        if (a.mask != nullptr && a.mask[row] == 0) {
            if ((kWhat & kLoss) && threadIdx.x == 0) a.row_loss[row] = 0.f, a.stats[row] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (kWhat & kGrad) {
                const RowShape gs = row_shape(g, a.vocab);
                uint4* gv = reinterpret_cast<uint4*>(g + gs.head);
                for (uint32_t i = threadIdx.x; i < gs.vecs; i += kThreads) gv[i] = make_uint4(0, 0, 0, 0);
                if (threadIdx.x < gs.head) g[threadIdx.x] = Type<T>::round(0.f);
                if (threadIdx.x < gs.tail) g[a.vocab - gs.tail + threadIdx.x] = Type<T>::round(0.f);
            }
            continue;
        }

        __syncthreads();  // the row before is done with shared memory
        if (kBucket && (kWhat & kLoss)) {
            for (uint32_t i = threadIdx.x; i < (a.vocab + 63) / 32; i += kThreads) s_bits[i] = 0;
            __syncthreads();
        }
        // the listed entries, by the first warp
        double tmax = -INFINITY, tsum = 0.0;
        if (warp == 0) {
            bool bad = false;
            for (uint32_t j = lane; j < a.k; j += 32) {
                const long long v = index_at(a, (uint64_t)row * a.ld_idx + j);
                const double t = teacher_at(a, (uint64_t)row * a.ld_teacher + j);
                const bool listed = v >= 0 && v < (long long)a.vocab;
                if (!listed && v != -1) bad = true;
                s_idx[j] = listed ? (int)v : -1;
                if (listed) {
                    s_z[j] = Type<T>::load(z + v);
                    if (kBucket && (kWhat & kLoss)) {
                        const uint32_t bit = bit_of<T>(shape, (uint32_t)v);
                        atomicOr(&s_bits[bit >> 5], 1u << (bit & 31));
                    }
                    tmax = (t > tmax || t != t) ? t : tmax;
                }
            }
            tmax = warp_max(tmax);
            if (!kBucket) {
                const double origin = tmax == -INFINITY ? 0.0 : tmax;
                for (uint32_t j = lane; j < a.k; j += 32)
                    if (s_idx[j] >= 0) tsum += exp((teacher_at(a, (uint64_t)row * a.ld_teacher + j) - origin) * inv_t);
                tsum = warp_sum(tsum);
                for (uint32_t j = lane; j < a.k; j += 32)
                    s_p[j] = s_idx[j] >= 0 && tsum != 0.0
                                 ? (float)(exp((teacher_at(a, (uint64_t)row * a.ld_teacher + j) - origin) * inv_t) / tsum)
                                 : 0.f;
                if (lane == 0) s_mass = tsum == 0.0 ? 0.0 : tsum / tsum;  // a NaN stays
            } else {
                for (uint32_t j = lane; j < a.k; j += 32) {
                    const double p = s_idx[j] >= 0 ? exp(teacher_at(a, (uint64_t)row * a.ld_teacher + j)) : 0.0;
                    s_p[j] = (float)p;
                    tsum += p;
                }
                tsum = warp_sum(tsum);
                bool all = false;  // the whole vocabulary is listed
                if ((kWhat & kLoss) && a.k >= a.vocab) {
                    __syncwarp();
                    uint32_t n = 0;
                    for (uint32_t i = lane; i < (a.vocab + 31) / 32; i += 32) n += __popc(s_bits[i]);
                    all = __reduce_add_sync(0xffffffffu, n) == a.vocab;
                }
                if (lane == 0) {
                    s_rest = tsum != tsum ? tsum : (tsum < 1.0 && !all ? 1.0 - tsum : 0.0);
                    s_mass = tsum + s_rest;
                }
            }
            bad = __any_sync(0xffffffffu, bad);
            if (lane == 0) s_bad = bad;
        }
        if (kBucket && (kWhat & kLoss)) __syncthreads();

        float M, inside, outside;
        if (kWhat & kLoss) {
            Running r;
            const uint4* zv = reinterpret_cast<const uint4*>(z + shape.head);
            const uint8_t* bytes = reinterpret_cast<const uint8_t*>(s_bits);
            for (uint32_t i = threadIdx.x; i < shape.vecs; i += kThreads) {
                float f[E];
                Type<T>::unpack(zv[i], f);
                float top = f[0];
#pragma unroll
                for (int j = 1; j < E; ++j) top = fmaxf(top, f[j]);
                r.raise(top, c);
                const float o = r.origin();
                uint32_t in = 0;
                if (kBucket) in = E == 8 ? bytes[i] : (bytes[i >> 1] >> (4 * (i & 1))) & 15u;
                if (in == 0) {
#pragma unroll
                    for (int j = 0; j < E; ++j) r.out += ex2((f[j] - o) * c);
                } else {
#pragma unroll
                    for (int j = 0; j < E; ++j) {
                        const float e = ex2((f[j] - o) * c);
                        if ((in >> j) & 1)
                            r.in += e;
                        else
                            r.out += e;
                    }
                }
            }
            for (uint32_t i = threadIdx.x; i < shape.head + shape.tail; i += kThreads) {
                const uint32_t v = i < shape.head ? i : i + shape.vecs * E;
                const float f = Type<T>::load(z + v);
                r.raise(f, c);
                const float e = ex2((f - r.origin()) * c);
                bool in = false;
                if (kBucket) {
                    const uint32_t bit = bit_of<T>(shape, v);
                    in = (s_bits[bit >> 5] >> (bit & 31)) & 1;
                }
                if (in)
                    r.in += e;
                else
                    r.out += e;
            }
            // join the threads
            float m = r.m;
#pragma unroll
            for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
            float o = m == -INFINITY ? 0.f : m;
            const float f = r.m == -INFINITY ? 1.f : ex2((r.m - o) * c);  // sums of 0 (or NaN) stay themselves
            const float w_out = warp_sum(r.out * f), w_in = warp_sum(r.in * f);
            if (lane == 0) s_m[warp] = m, s_out[warp] = w_out, s_in[warp] = w_in;
            __syncthreads();
            M = s_m[0];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) M = fmaxf(M, s_m[w]);
            o = M == -INFINITY ? 0.f : M;
            float out = 0.f, in = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float fw = s_m[w] == -INFINITY ? 1.f : ex2((s_m[w] - o) * c);
                out += s_out[w] * fw, in += s_in[w] * fw;
            }
            const float Z = out + in;
            inside = (float)s_mass / Z;
            outside = inside;
            if (kBucket && s_rest > 0.0) outside = inside - (float)(s_rest / (double)out);
            if (warp == 0) {
                const double log_z = log((double)Z);
                double t = 0.0;
                for (uint32_t j = lane; j < a.k; j += 32) {
                    if (s_idx[j] < 0) continue;
                    const double x = teacher_at(a, (uint64_t)row * a.ld_teacher + j);
                    const double log_p = kBucket ? x : (x - tmax) * inv_t - log(tsum);
                    const double p = kBucket ? exp(x) : exp((x - (tmax == -INFINITY ? 0.0 : tmax)) * inv_t) / tsum;
                    const double log_q = ((double)s_z[j] - (double)M) * inv_t - log_z;
                    if (p != 0.0 && (kBucket || tsum != 0.0)) t += p * (log_p - log_q);
                }
                t = warp_sum(t);
                if (kBucket && !(s_rest <= 0.0)) t += s_rest * (log(s_rest) - (log((double)out) - log_z));
                if (s_bad) t = (double)NAN;
                if (lane == 0) {
                    a.row_loss[row] = (float)(t * (double)a.weight * (double)a.temperature * (double)a.temperature);
                    a.stats[row] = make_float4(M, inside, outside, 0.f);
                }
            }
        } else {
            const float4 st = a.stats[row];
            M = st.x, inside = st.y, outside = st.z;
        }

        if (kWhat & kGrad) {
            if (!(kWhat & kLoss)) {
                scale = a.grad_out[(uint64_t)row * a.grad_out_stride];
                __syncthreads();  // the listed entries
            }
            float gf = (float)((double)scale * (double)a.weight * (double)a.temperature *
                               (double)(a.inv_n != nullptr ? *a.inv_n : a.inv_n_value));
            if (s_bad) gf = NAN;
            const float k_out = outside * gf;
            const uint4* zv = reinterpret_cast<const uint4*>(z + shape.head);
            if (same_offset) {
                uint4* gv = reinterpret_cast<uint4*>(g + shape.head);
                for (uint32_t i = threadIdx.x; i < shape.vecs; i += kThreads) {
                    float f[E];
                    Type<T>::unpack(zv[i], f);
#pragma unroll
                    for (int j = 0; j < E; ++j) f[j] = ex2((f[j] - M) * c) * k_out;
                    gv[i] = Type<T>::pack(f);
                }
                for (uint32_t i = threadIdx.x; i < shape.head + shape.tail; i += kThreads) {
                    const uint32_t v = i < shape.head ? i : i + shape.vecs * E;
                    g[v] = Type<T>::round(ex2((Type<T>::load(z + v) - M) * c) * k_out);
                }
            } else {
                for (uint32_t v = threadIdx.x; v < a.vocab; v += kThreads)
                    g[v] = Type<T>::round(ex2((Type<T>::load(z + v) - M) * c) * k_out);
            }
            __syncthreads();  // the row's gradient is written: now the listed elements over it
            for (uint32_t j = threadIdx.x; j < a.k; j += kThreads) {
                const int v = s_idx[j];
                if (v < 0) continue;
                float p = 0.f;
                for (uint32_t i = 0; i < a.k; ++i)
                    if (s_idx[i] == v) p += s_p[i];
                g[v] = Type<T>::round((ex2((s_z[j] - M) * c) * inside - p) * gf);
            }
        }
    }
}

// 1 / max(1, rows kept)
__global__ void distill_count_kernel(const uint8_t* mask, uint32_t rows, float* inv_n)
{
    __shared__ uint32_t s[32];
    uint32_t n = 0;
    for (uint32_t i = threadIdx.x; i < rows; i += blockDim.x) n += mask[i] != 0;
    n = __reduce_add_sync(0xffffffffu, n);
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (uint32_t w = 1; w < blockDim.x / 32; ++w) n += s[w];
        *inv_n = (float)(1.0 / (double)(n ? n : 1));
    }
}

// The rows' losses, summed in 64 bits in a fixed order.
__global__ void distill_sum_kernel(const float* row_loss, uint32_t rows, const float* inv_n, float inv_n_value, float* loss)
{
    __shared__ double s[32];
    double t = 0.0;
    for (uint32_t i = threadIdx.x; i < rows; i += blockDim.x) t += (double)row_loss[i];
    t = warp_sum(t);
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = t;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (uint32_t w = 1; w < blockDim.x / 32; ++w) t += s[w];
        *loss = (float)(t * (double)(inv_n != nullptr ? *inv_n : inv_n_value));
    }
}

template <typename T, bool kBucket, int kWhat>
int launch(const DistillArgs& a, cudaStream_t st)
{
    const int sms = ps_internal::sm_count();
    if (sms < 0) return sms;
    const size_t smem = 12 * (size_t)a.k + (kBucket && (kWhat & kLoss) ? ((size_t)(a.vocab + 63) / 32) * 4 : 0);
    if (smem > 40 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(distill_kernel<T, kBucket, kWhat>,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) {
            ps_internal::set_cuda_error((int)e);
            cudaGetLastError();
            return PS_ERR_CUDA;
        }
    }
    const uint32_t most = (uint32_t)sms * 4;
    distill_kernel<T, kBucket, kWhat><<<a.rows < most ? a.rows : most, kThreads, smem, st>>>(a);
    return ps_internal::after_launch();
}
template <typename T>
int launch(const DistillArgs& a, bool bucket, int what, cudaStream_t st)
{
    if (what == kLoss) return bucket ? launch<T, true, kLoss>(a, st) : launch<T, false, kLoss>(a, st);
    if (what == kGrad) return bucket ? launch<T, true, kGrad>(a, st) : launch<T, false, kGrad>(a, st);
    return bucket ? launch<T, true, kLoss | kGrad>(a, st) : launch<T, false, kLoss | kGrad>(a, st);
}
int launch(const DistillArgs& a, int dtype, bool bucket, int what, cudaStream_t st)
{
    if (dtype == PS_DTYPE_F16) return launch<__half>(a, bucket, what, st);
    if (dtype == PS_DTYPE_BF16) return launch<__nv_bfloat16>(a, bucket, what, st);
    return launch<float>(a, bucket, what, st);
}

int check_problem(const ps_distill_problem* q, const float* inv_n)
{
    if (q == nullptr) return PS_ERR_INVALID;
    if (q->dtype < PS_DTYPE_F16 || q->dtype > PS_DTYPE_F32 || q->teacher_dtype < PS_DTYPE_F16 ||
        q->teacher_dtype > PS_DTYPE_F32)
        return PS_ERR_INVALID;
    if (q->index_bytes != 4 && q->index_bytes != 8) return PS_ERR_INVALID;
    if (q->tail != PS_TAIL_DROP && q->tail != PS_TAIL_BUCKET) return PS_ERR_INVALID;
    if (q->reduction < PS_REDUCE_NONE || q->reduction > PS_REDUCE_MEAN) return PS_ERR_INVALID;
    if (!(q->temperature > 0.f) || !(q->temperature < INFINITY) || !(q->weight < INFINITY) || !(q->weight > -INFINITY))
        return PS_ERR_INVALID;
    if (q->rows == 0) return PS_OK;
    if (q->vocab == 0 || q->k == 0) return PS_ERR_INVALID;
    if (q->vocab > PS_DISTILL_MAX_VOCAB || q->k > PS_DISTILL_MAX_K) return PS_ERR_LIMIT;
    if (q->logits == nullptr || q->indices == nullptr || q->teacher == nullptr) return PS_ERR_INVALID;
    if (q->reduction == PS_REDUCE_MEAN && q->mask != nullptr && inv_n == nullptr) return PS_ERR_INVALID;
    const uint64_t es = q->dtype == PS_DTYPE_F32 ? 4 : 2, ts = q->teacher_dtype == PS_DTYPE_F32 ? 4 : 2;
    if ((uintptr_t)q->logits % es || (uintptr_t)q->teacher % ts || (uintptr_t)q->indices % q->index_bytes)
        return PS_ERR_ALIGN;
    return PS_OK;
}

DistillArgs arguments(const ps_distill_problem* q, const float* inv_n)
{
    DistillArgs a;
    memset(&a, 0, sizeof(a));
    a.z = q->logits, a.ldz = q->ld_logits, a.rows = q->rows, a.vocab = q->vocab, a.k = q->k;
    a.idx = q->indices, a.ld_idx = q->ld_indices, a.idx_bytes = q->index_bytes;
    a.teacher = q->teacher, a.ld_teacher = q->ld_teacher, a.teacher_dtype = q->teacher_dtype;
    a.mask = (const uint8_t*)q->mask;
    a.temperature = q->temperature, a.weight = q->weight;
    const bool mean = q->reduction == PS_REDUCE_MEAN;
    a.inv_n = mean && q->mask != nullptr ? inv_n : nullptr;
    a.inv_n_value = mean && q->rows > 0 ? (float)(1.0 / (double)q->rows) : 1.f;
    return a;
}

}  // namespace

extern "C" {

int ps_distill_forward(const ps_distill_problem* q, float* loss_dev, float* row_loss_dev, void* stats_dev,
                       float* inv_n_dev, const ps_scaler_state* scaler_dev, void* grad_dev, uint64_t ld_grad,
                       float* used_scale_dev, void* stream)
{
    int rc = check_problem(q, inv_n_dev);
    if (rc != PS_OK) return rc;
    const bool grad = grad_dev != nullptr, reduce = q->reduction != PS_REDUCE_NONE;
    if (reduce && loss_dev == nullptr) return PS_ERR_INVALID;
    if (q->rows > 0 && (row_loss_dev == nullptr || stats_dev == nullptr)) return PS_ERR_INVALID;
    if ((uintptr_t)stats_dev % 16) return PS_ERR_ALIGN;
    if (grad && (!reduce || scaler_dev == nullptr || used_scale_dev == nullptr || ld_grad < q->vocab))
        return PS_ERR_INVALID;
    if (grad && (uintptr_t)grad_dev % (q->dtype == PS_DTYPE_F32 ? 4 : 2)) return PS_ERR_ALIGN;
    cudaStream_t st = (cudaStream_t)stream;
    DistillArgs a = arguments(q, inv_n_dev);
    a.row_loss = row_loss_dev, a.stats = (float4*)stats_dev;
    a.grad = grad_dev, a.ldg = ld_grad, a.scaler = scaler_dev, a.used_scale = used_scale_dev;
    if (q->rows > 0) {
        if (a.inv_n != nullptr) {
            distill_count_kernel<<<1, 1024, 0, st>>>(a.mask, q->rows, inv_n_dev);
            rc = ps_internal::after_launch();
            if (rc != PS_OK) return rc;
        }
        rc = launch(a, q->dtype, q->tail == PS_TAIL_BUCKET, grad ? kLoss | kGrad : kLoss, st);
        if (rc != PS_OK) return rc;
    }
    if (!reduce) return PS_OK;
    // no rows: a loss of 0
    distill_sum_kernel<<<1, 1024, 0, st>>>(row_loss_dev, q->rows, q->rows > 0 ? a.inv_n : nullptr, a.inv_n_value, loss_dev);
    return ps_internal::after_launch();
}

int ps_distill_backward(const ps_distill_problem* q, const void* stats_dev, const float* inv_n_dev,
                        const float* grad_out_dev, uint32_t grad_out_stride, const float* used_scale_dev,
                        void* grad_dev, uint64_t ld_grad, void* stream)
{
    const int rc = check_problem(q, inv_n_dev);
    if (rc != PS_OK) return rc;
    if (q->rows == 0) return PS_OK;
    if (stats_dev == nullptr || grad_out_dev == nullptr || grad_dev == nullptr || ld_grad < q->vocab) return PS_ERR_INVALID;
    if (used_scale_dev != nullptr && q->reduction == PS_REDUCE_NONE) return PS_ERR_INVALID;
    if ((uintptr_t)stats_dev % 16 || (uintptr_t)grad_dev % (q->dtype == PS_DTYPE_F32 ? 4 : 2)) return PS_ERR_ALIGN;
    DistillArgs a = arguments(q, inv_n_dev);
    a.stats = (float4*)const_cast<void*>(stats_dev), a.grad_out = grad_out_dev;
    a.grad_out_stride = grad_out_stride, a.used_scale = const_cast<float*>(used_scale_dev);
    a.grad = grad_dev, a.ldg = ld_grad;
    return launch(a, q->dtype, q->tail == PS_TAIL_BUCKET, kGrad, (cudaStream_t)stream);
}

}  // extern "C"
