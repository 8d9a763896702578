// Divergence of a student's distribution from the top entries of a teacher's,
// and its gradient with respect to the student's logits.
//
// For a row of logits z over the vocabulary, temperature T and c = log2(e) / T:
//     M an element near the largest,  e_v = 2^((z_v - M) c),  Z = sum e_v,  q_v = e_v / Z
// and for the k listed entries (idx_j, t_j), S the set of listed indices:
//     drop    p = softmax(t / T) over the listed;   p_r = 0
//     bucket  p_j = exp(t_j);   p_r = max(0, 1 - sum p_j),   q_r = sum of q_v, v not in S
//             (p_r = 0 where S is the whole vocabulary: rounding leaves no rest there)
//     loss = T^2 ( sum_j p_j (log p_j - log q_idx_j) + p_r (log p_r - log q_r) )
//     d loss / d z_v = T ( (sum p + p_r) q_v - sum_{j: idx_j = v} p_j - [v not in S] p_r q_v / q_r )
// where sum p + p_r is 1, but for a row that lists nothing (0) or a teacher that gives more than 1.
// The listed elements may lie so far above the others that relative to M nothing of these is left in 32 bits.  So
// with the bucket the sum over the others is relative to an element M_out near the largest of them,
//     e'_v = 2^((z_v - M_out) c),  Z' = sum of e'_v, v not in S,  q_r = Z' / (Z' + sum of the listed, brought to M_out)
//     d loss / d z_v = T e'_v ((sum p + p_r) q_r - p_r) / Z',  v not in S
// whose every factor is bounded.
//
// One CTA takes a row: one pass with a running maximum and sum of its own in
// every thread, joined at the end; and for the gradient a second pass that reads
// the row again, from L2 when it follows the first (148 SMs hold a few rows each,
// 0.1 to 0.5 MB a row).
// The listed entries are few: one warp works on them in 64 bits beside the
// others' pass.  Their gradient is written over the row's after it, so the pass
// itself knows nothing of them but, for the bucket, one bit per element.
// 4096 x 131073 bf16: loss alone 6.1 TB/s; 8192 x 50257 fp16, k = 64: loss 155 us
// (5.3 TB/s), with the gradient 325 us (5.1 TB/s of one read and one write).  HBM-bound: one read, and one write for the
// gradient; a power of two per element each pass.
#include "ps_b200.h"

#include "ps_internal.h"
#include "ps_launch.cuh"
#include "ps_pair.cuh"
#include "ps_tensor_core.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cfloat>
#include <cstring>
#include <type_traits>

namespace {

constexpr int kMaxThreads = 320;   // 256 of the pass
constexpr int kLongThreads = 576;  // 512 of the pass, for the longest rows
constexpr uint32_t kMaxSlots = 4;
constexpr int kCtas = 3;  // of the largest kind on an SM: 64 registers a thread
// Bytes of rows in work, of 126 MB of L2.  8192 x 50257 fp16 with gradient: 325 us with 64 MB, 386 us with 32 MB (two
// CTAs an SM), 359 us with 128 MB; with the bucket 383, 475 and 383 us.
constexpr uint64_t kRowsInL2 = 64ull << 20;
constexpr uint32_t kMostSmem = 224 * 1024;  // of a CTA: what the layout below may take, beside 3 KB that are static
constexpr int kUnroll = 4;  // vectors of a chunk for each thread of the pass

__device__ unsigned int g_gave_up;  // CTAs that ran into the limit of a wait

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
    float* loss;         // of a single row (else NULL: the rows are summed by a launch of their own)
    float4* stats;       // per row: M, factors of e_v in the gradient for v in S and of e'_v for the others, M_out
    const float* inv_n;  // 1 / rows that the mask keeps, or NULL: then inv_n_value
    float inv_n_value;
    void* grad;
    uint64_t ldg;
    const ps_scaler_state* scaler;  // gradient in the forward pass: of loss times this scale
    float* used_scale;              // ... which the forward pass leaves here
    const float* grad_out;          // gradient in the backward pass: of loss times this
    uint32_t grad_out_stride;
};

__device__ __forceinline__ void prefetch(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
// Four bytes into shared memory, there after a cp.async.wait_all of the same thread.
__device__ __forceinline__ void fetch4(void* dst, const void* src)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(tc::smem_u32(dst)), "l"(src) : "memory");
}
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
    static constexpr uint32_t kNothing = 0xfc00fc00u;  // minus infinities
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b)
    {
        const __half2 h = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float fold(uint32_t a)
    {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a));
        return fmaxf(f.x, f.y);
    }
    static __device__ __forceinline__ float load(const __half* p) { return __half2float(*p); }
    static __device__ __forceinline__ float half_of(uint32_t w, bool upper)
    {
        return __half2float(__ushort_as_half((unsigned short)(upper ? w >> 16 : w)));
    }
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
    static constexpr uint32_t kNothing = 0xff80ff80u;
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b)
    {
        const __nv_bfloat162 h =
            __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float fold(uint32_t a)
    {
        return fmaxf(__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u));
    }
    static __device__ __forceinline__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
    static __device__ __forceinline__ float half_of(uint32_t w, bool upper)
    {
        return __uint_as_float(upper ? w & 0xffff0000u : w << 16);
    }
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
    static constexpr uint32_t kNothing = 0xff800000u;
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b)
    {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }
    static __device__ __forceinline__ float fold(uint32_t a) { return __uint_as_float(a); }
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

// What a row's powers of two are relative to: the exponent of element z is z c - r, one rounding, with
// r = m c rounded and m the largest element.  r itself is the reference, so its rounding does not matter, as
// long as it moves the largest exponent by less than 2^5: |r| < 2^30.  Beyond that (logits near the end of
// their type, or tiny temperatures) the exponent is (z - m) c.
struct Origin {
    float m = -INFINITY, r = 0.f;
    bool far = false;
    __device__ __forceinline__ Origin() {}
    __device__ __forceinline__ Origin(float top, float c) : m(top)
    {
        r = m == -INFINITY ? 0.f : m * c;
        far = fabsf(r) >= 1073741824.f && fabsf(m) < INFINITY;
    }
    __device__ __forceinline__ float exponent(float z, float c) const
    {
        return far ? (z - m) * c : fmaf(z, c, -r);
    }
    // what the exponents are relative to
    __device__ __forceinline__ double reference(float c) const { return far ? (double)m * (double)c : (double)r; }
    // of sums relative to this one, to make them relative to `to` (no smaller)
    __device__ __forceinline__ float factor(const Origin& to, float c) const
    {
        if (m == -INFINITY) return 1.f;  // sums of 0 (or NaN): they stay themselves
        return ex2(far || to.far ? (m - to.m) * c : r - to.r);
    }
};

// Running origin and sums of one thread: of elements outside of S, and of those in it.  The origin is an element,
// not always the largest one: it is raised when an exponent would pass 2^4 (sums of 2^20 such terms are far from
// the end of 32 bits), which after a thread's first elements hardly ever happens.  The listed ones are few; their
// sum is relative to the largest of them itself.
struct Running {
    Origin o;
    Pair out = Pair(0.f, 0.f);
    float m_in = -INFINITY, in = 0.f;
    __device__ __forceinline__ void raise(float top, float c)
    {
        if (o.m == -INFINITY ? top > -INFINITY : o.exponent(top, c) > 16.f) {
            const Origin to(top, c);
            const float f = o.factor(to, c);
            out = mul2(out, Pair(f, f));
            o = to;
        }
    }
    __device__ __forceinline__ void add_listed(float z, float c)
    {
        if (z > m_in)
            in = fmaf(in, ex2((m_in - z) * c), 1.f), m_in = z;
        else if (z != -INFINITY)
            in += ex2((z - m_in) * c);
    }
};

constexpr int kLoss = 1, kGrad = 2;

// One row's listed entries and what the pass over it found; two of them, in turn.
struct RowSlot {
    double rest, mass;  // p_r, and sum p + p_r: 1 unless the teacher gives nothing, or too much
    float M, Z;             // element that exponents are relative to, and the sum of their powers
    float M_out, out;       // the same of the elements outside of S (with the bucket)
    float inside;           // factor of e_v in the gradient, v in S
    float grad;             // factor of the gradient: NaN for a bad row
    int keep, bad, twice;   // the mask keeps the row; an index is outside of the vocabulary; one is listed twice
};
struct Listed {
    double *p, *log_p;  // probabilities and their logarithms
    int* idx;           // or -1
    uint32_t* z;        // logits, or the words that hold them
    uint32_t* bits;     // of every element: is it listed?
    uint32_t* owners;   // of every thread and chunk: has it a listed element?
    uint32_t* seen;     // bits of indices seen, without the bitmap: zeros but while entries are looked at
};
constexpr uint32_t kSeenWords = 1024;
// Threads and shared memory of a CTA: chunks of kUnroll vectors a thread, a ring of them, barriers, listed entries,
// bitmaps.
struct Layout {
    uint32_t chunk_vecs, slots, threads;  // vectors of a chunk, chunks of the ring, threads of the pass (2^shift)
    uint32_t shift;
};
__host__ __device__ __forceinline__ uint32_t bitmap_words(uint32_t vocab) { return (vocab + 63) / 64 * 2; }
// a vector has four elements at least
__host__ __device__ __forceinline__ uint32_t owner_words(const Layout& l, uint32_t vocab)
{
    return ((vocab / 4 + l.chunk_vecs - 1) / l.chunk_vecs * (l.threads / 32) + 1) / 2 * 2;
}
__host__ __device__ __forceinline__ size_t smem_bytes(const Layout& l, uint32_t k, uint32_t vocab, bool bits, bool seen)
{
    return (size_t)l.slots * l.chunk_vecs * 16 + 48 * (size_t)k +
           (bits ? 8 * (size_t)(bitmap_words(vocab) + owner_words(l, vocab)) : seen ? 4 * kSeenWords : 0);
}
// Word of `owners` for element v of the vectors (bit: thread % 32)
template <typename T>
__device__ __forceinline__ uint32_t owner_of(const Layout& lay, const RowShape& s, uint32_t v, uint32_t* bit)
{
    static_assert(kUnroll == 4, "a chunk is four vectors a thread");
    const uint32_t i = (v - s.head) / Type<T>::kVec, t = i & (lay.threads - 1);
    *bit = t & 31;
    return ((i >> (lay.shift + 2)) << (lay.shift - 5)) + (t >> 5);
}

__device__ __forceinline__ float grad_factor(const DistillArgs& a, float scale)
{
    return (float)((double)scale * (double)a.weight * (double)a.temperature *
                   (double)(a.inv_n != nullptr ? *a.inv_n : a.inv_n_value));
}

// The listed entries of a row, by one warp, before the pass over it.
template <typename T, bool kBucket, int kWhat>
__device__ void entries_before(const DistillArgs& a, const Layout& lay, uint32_t row, RowSlot& slot, const Listed& l,
                               float scale)
{
    const uint32_t lane = threadIdx.x & 31;
    const bool keep = a.mask == nullptr || a.mask[row] != 0;
    if (lane == 0) slot.keep = keep, slot.bad = 0;
    if (!keep) return;
    const T* const z = reinterpret_cast<const T*>(a.z) + (uint64_t)row * a.ldz;
    const RowShape shape = row_shape(z, a.vocab);
    const double inv_t = 1.0 / (double)a.temperature;
    bool bad = false;
    bool twice = false;
    double tmax = -INFINITY, tsum = 0.0;
    if (row + gridDim.x < a.rows) {  // the entries of the row after are fetched by the time they are wanted
        const char* const i = reinterpret_cast<const char*>(a.idx) + (uint64_t)(row + gridDim.x) * a.ld_idx * a.idx_bytes;
        const uint32_t ts = a.teacher_dtype == PS_DTYPE_F32 ? 4 : 2;
        const char* const t = reinterpret_cast<const char*>(a.teacher) + (uint64_t)(row + gridDim.x) * a.ld_teacher * ts;
        for (uint32_t at = lane * 128; at < a.k * a.idx_bytes; at += 32 * 128) prefetch(i + at);
        for (uint32_t at = lane * 128; at < a.k * ts; at += 32 * 128) prefetch(t + at);
    }
#pragma unroll 4
    for (uint32_t j = lane; j < a.k; j += 32) {
        const long long v = index_at(a, (uint64_t)row * a.ld_idx + j);
        const bool is = v >= 0 && v < (long long)a.vocab;
        if (!is && v != -1) bad = true;
        l.idx[j] = is ? (int)v : -1;
        l.log_p[j] = teacher_at(a, (uint64_t)row * a.ld_teacher + j);
    }
    // the logits of the listed entries are on their way until the pass over the row is done; of 16-bit types the
    // aligned word that holds them
    for (uint32_t j = lane; j < a.k; j += 32)
        if (l.idx[j] >= 0) fetch4(&l.z[j], reinterpret_cast<const void*>((uintptr_t)(z + l.idx[j]) & ~(uintptr_t)3));
    for (uint32_t j = lane; j < a.k; j += 32) {
        const int v = l.idx[j];
        const double t = l.log_p[j];
        if (v < 0) continue;
        if (kBucket && (kWhat & kLoss)) {
            const uint32_t bit = bit_of<T>(shape, (uint32_t)v), one = 1u << (bit & 31);
            if (atomicOr(&l.bits[bit >> 5], one) & one) twice = true;
            if ((uint32_t)v - shape.head < shape.vecs * Type<T>::kVec) {
                uint32_t of;
                const uint32_t w = owner_of<T>(lay, shape, (uint32_t)v, &of);
                atomicOr(&l.owners[w], 1u << of);
            }
        } else if (kWhat & kGrad) {  // two of an index share a bit (so may others: then it is looked up in vain)
            const uint32_t bit = (uint32_t)v & (32 * kSeenWords - 1), one = 1u << (bit & 31);
            if (atomicOr(&l.seen[bit >> 5], one) & one) twice = true;
        }
        tmax = (t > tmax || t != t) ? t : tmax;
    }
    if (kWhat & kGrad) {
        twice = __any_sync(0xffffffffu, twice);
        __syncwarp();
        if (!(kBucket && (kWhat & kLoss)))
            for (uint32_t j = lane; j < a.k; j += 32)
                if (l.idx[j] >= 0) l.seen[((uint32_t)l.idx[j] & (32 * kSeenWords - 1)) >> 5] = 0;
    }
    if (!kBucket) tmax = warp_max(tmax);
    const double origin = kBucket || tmax == -INFINITY ? 0.0 : tmax;
    for (uint32_t j = lane; j < a.k; j += 32) {
        const double x = kBucket ? l.log_p[j] : (l.log_p[j] - origin) * inv_t;
        const double p = l.idx[j] >= 0 ? exp(x) : 0.0;
        l.log_p[j] = x, l.p[j] = p;
        tsum += p;
    }
    tsum = warp_sum(tsum);
    double rest = 0.0, mass = tsum;
    if (!kBucket) {
        mass = tsum == 0.0 ? 0.0 : tsum / tsum;  // a NaN stays
        const double inv = tsum == 0.0 ? 0.0 : 1.0 / tsum, log_sum = (kWhat & kLoss) ? log(tsum) : 0.0;
        for (uint32_t j = lane; j < a.k; j += 32) l.p[j] *= inv, l.log_p[j] -= log_sum;
    } else if (kWhat & kLoss) {
        bool all = false;  // the whole vocabulary is listed
        if (a.k >= a.vocab) {
            __syncwarp();
            uint32_t n = 0;
            for (uint32_t i = lane; i < (a.vocab + 31) / 32; i += 32) n += __popc(l.bits[i]);
            all = __reduce_add_sync(0xffffffffu, n) == a.vocab;
        }
        rest = tsum != tsum ? tsum : (tsum < 1.0 && !all ? 1.0 - tsum : 0.0);
        mass = tsum + rest;
    }
    bad = __any_sync(0xffffffffu, bad);
    if (kWhat == kGrad) scale = a.grad_out[(uint64_t)row * a.grad_out_stride];
    if (lane == 0) {
        slot.rest = rest, slot.mass = mass, slot.bad = bad, slot.twice = twice;
        if (kWhat & kGrad) slot.grad = bad ? NAN : grad_factor(a, scale);
    }
}

// ... and after it: the row's loss, and the gradient of the listed elements over what the pass wrote there.
template <typename T, bool kBucket, int kWhat>
__device__ void entries_after(const DistillArgs& a, const Layout& lay, uint32_t row, const RowSlot& slot, const Listed& l,
                              float c)
{
    const uint32_t lane = threadIdx.x & 31;
    if (!slot.keep) return;
    const Origin o(slot.M, c);
    const T* const zr = reinterpret_cast<const T*>(a.z) + (uint64_t)row * a.ldz;
    asm volatile("cp.async.wait_all;" ::: "memory");
    auto logit = [&](uint32_t j, int v) {  // every lane looks at what it has fetched itself
        const uint32_t w = l.z[j];
        if constexpr (sizeof(T) == 4)
            return __uint_as_float(w);
        else
            return Type<T>::half_of(w, ((uintptr_t)(zr + v) >> 1) & 1);
    };
    if (kWhat & kLoss) {
        const double log_z = log((double)slot.Z);
        double t = 0.0;
        for (uint32_t j = lane; j < a.k; j += 32) {
            const int v = l.idx[j];
            const double p = l.p[j];
            if (v < 0 || p == 0.0) continue;
            const double z = (double)logit(j, v);
            const double x = o.far ? (z - (double)slot.M) * (double)c : z * (double)c - (double)o.r;
            t += p * (l.log_p[j] - (x * 0.6931471805599453 - log_z));
        }
        t = warp_sum(t);
        if (kBucket && !(slot.rest <= 0.0)) {
            const double apart = Origin(slot.M_out, c).reference(c) - o.reference(c);
            t += slot.rest * (log(slot.rest) - (apart * 0.6931471805599453 + log((double)slot.out) - log_z));
        }
        if (slot.bad) t = (double)NAN;
        if (lane == 0) {
            const float f = (float)(t * (double)a.weight * (double)a.temperature * (double)a.temperature);
            a.row_loss[row] = f;
            if (a.loss != nullptr) *a.loss = f;  // a mean over one row, too
        }
    }
    if (kWhat & kGrad) {
        T* const g = reinterpret_cast<T*>(a.grad) + (uint64_t)row * a.ldg;
        for (uint32_t j = lane; j < a.k; j += 32) {
            const int v = l.idx[j];
            if (v < 0) continue;
            float p = (float)l.p[j];
            if (slot.twice) {
                p = 0.f;
                for (uint32_t i = 0; i < a.k; ++i)
                    if (l.idx[i] == v) p += (float)l.p[i];
            }
            g[v] = Type<T>::round((ex2(o.exponent(logit(j, v), c)) * slot.inside - p) * slot.grad);
        }
    }
    if (kBucket && (kWhat & kLoss)) {  // the bitmap is zeros again
        __syncwarp();
        const RowShape shape = row_shape(zr, a.vocab);
        for (uint32_t j = lane; j < a.k; j += 32)
            if (l.idx[j] >= 0) {
                const uint32_t v = (uint32_t)l.idx[j];
                uint32_t of;
                l.bits[bit_of<T>(shape, v) >> 5] = 0;
                if (v - shape.head < shape.vecs * Type<T>::kVec) l.owners[owner_of<T>(lay, shape, v, &of)] = 0;
            }
        __syncwarp();
    }
}

// One warp fetches a row's vectors in chunks, ahead of their use, with bulk copies into a ring (for the
// gradient the same ones again behind them).  One warp works on the listed entries of the row before and of
// the row after meanwhile, so that their chains of 64-bit logarithms and scattered loads hide behind the
// pass.  The other warps pass over the chunks.
template <typename T, bool kBucket, int kWhat, bool kLong>
__global__ void __launch_bounds__(kLong ? kLongThreads : kMaxThreads, kLong ? 2 : kCtas)
distill_kernel(const DistillArgs a, const Layout lay)
{
    constexpr int E = Type<T>::kVec;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ RowSlot slots[2];
    __shared__ float s_m[kLongThreads / 32], s_out[kLongThreads / 32], s_m_in[kLongThreads / 32], s_in[kLongThreads / 32];
    __shared__ uint64_t full[kMaxSlots], empty[kMaxSlots];
    __shared__ volatile int gave_up;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t threads = lay.threads, warps = threads >> 5;
    const float c = (float)(1.4426950408889634 / (double)a.temperature);
    Listed listed[2];
    {
        double* const d = reinterpret_cast<double*>(smem + (size_t)lay.slots * lay.chunk_vecs * 16);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            listed[i].p = d + 2 * i * a.k;
            listed[i].log_p = d + (2 * i + 1) * a.k;
            listed[i].idx = reinterpret_cast<int*>(d + 4 * a.k) + 2 * i * a.k;
            listed[i].z = reinterpret_cast<uint32_t*>(d + 4 * a.k) + (2 * i + 1) * a.k;
            listed[i].bits = reinterpret_cast<uint32_t*>(d + 6 * a.k) + i * bitmap_words(a.vocab);
            listed[i].seen = reinterpret_cast<uint32_t*>(d + 6 * a.k);
            listed[i].owners = reinterpret_cast<uint32_t*>(d + 6 * a.k) + 2 * bitmap_words(a.vocab) + i * owner_words(lay, a.vocab);
        }
    }

    cudaTriggerProgrammaticLaunchCompletion();
    cudaGridDependencySynchronize();
    if ((kWhat & kLoss) == 0 && a.used_scale != nullptr && *a.used_scale == *a.grad_out)
        return;  // the forward pass wrote this gradient
    float scale = 1.f;
    if ((kWhat & kGrad) && (kWhat & kLoss)) {
        scale = a.scaler->dynamic < 0 ? 1.f : (float)a.scaler->cur_scale;
        if (blockIdx.x == 0 && threadIdx.x == 0) *a.used_scale = scale;
    }
    if (kBucket && (kWhat & kLoss))
        for (uint32_t i = threadIdx.x; i < 2 * (bitmap_words(a.vocab) + owner_words(lay, a.vocab)); i += blockDim.x)
            listed[0].bits[i] = 0;
    else if (kWhat & kGrad)
        for (uint32_t i = threadIdx.x; i < kSeenWords; i += blockDim.x) listed[0].seen[i] = 0;
    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < lay.slots; ++s) tc::bar_init(&full[s], 1), tc::bar_init(&empty[s], warps);
        gave_up = 0;
        tc::bar_init_fence();
    }
    __syncthreads();

    constexpr int kPasses = kWhat == (kLoss | kGrad) ? 2 : 1;
    if (warp == warps + 1) {
        if (tc::elect_one()) {
            const uint64_t once = tc::evict_first_policy();
            uint32_t n = 0, at = 0, phase = 1;  // of the place's barrier `empty`: the first round waits for nothing
            bool ok = true;
            for (uint32_t row = blockIdx.x; row < a.rows && ok; row += gridDim.x) {
                if (a.mask != nullptr && a.mask[row] == 0) continue;
                const T* const z = reinterpret_cast<const T*>(a.z) + (uint64_t)row * a.ldz;
                const RowShape shape = row_shape(z, a.vocab);
                const uint4* const zv = reinterpret_cast<const uint4*>(z + shape.head);
                for (int pass = 0; pass < kPasses && ok; ++pass)
                    for (uint32_t v0 = 0; v0 < shape.vecs; v0 += lay.chunk_vecs, ++n) {
                        if (n >= lay.slots && !tc::bar_wait(&empty[at], phase, &gave_up)) {
                            ok = false;
                            break;
                        }
                        const uint32_t bytes = min(lay.chunk_vecs, shape.vecs - v0) * 16;
                        tc::bar_expect(&full[at], bytes);
                        void* const dst = smem + (size_t)at * lay.chunk_vecs * 16;
                        if (pass + 1 < kPasses)  // read again soon
                            tc::load_bulk(dst, zv + v0, bytes, &full[at]);
                        else
                            tc::load_bulk(dst, zv + v0, bytes, &full[at], once);
                        if (++at == lay.slots) at = 0, phase ^= 1;
                    }
            }
            if (gave_up) {
                // copies may still be landing in this CTA's memory
                int ignore = 0;
                for (uint32_t i = n < lay.slots ? 0 : n - lay.slots; i < n; ++i)
                    tc::bar_wait(&full[i % lay.slots], (i / lay.slots) & 1, &ignore);
            }
        }
    } else if (warp == warps) {
        entries_before<T, kBucket, kWhat>(a, lay, blockIdx.x, slots[0], listed[0], scale);
        uint32_t it = 0;
        for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x, ++it) {
            asm volatile("bar.sync 2, %0;" ::"r"(threads + 32) : "memory");  // see below
            const uint32_t other = (it + 1) & 1;
            if (it > 0) entries_after<T, kBucket, kWhat>(a, lay, row - gridDim.x, slots[other], listed[other], c);
            __syncwarp();
            if (row + gridDim.x < a.rows)
                entries_before<T, kBucket, kWhat>(a, lay, row + gridDim.x, slots[other], listed[other], scale);
        }
        asm volatile("bar.sync 2, %0;" ::"r"(threads + 32) : "memory");
        entries_after<T, kBucket, kWhat>(a, lay, blockIdx.x + (it - 1) * gridDim.x, slots[(it - 1) & 1], listed[(it - 1) & 1], c);
    } else {
        uint32_t it = 0, at = 0, phase = 0;
        bool lost = false;  // a chunk did not come
        for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x, ++it) {
            // this row's entries are there, the row before is written
            asm volatile("bar.sync 2, %0;" ::"r"(threads + 32) : "memory");
            RowSlot& slot = slots[it & 1];
            const T* const z = reinterpret_cast<const T*>(a.z) + (uint64_t)row * a.ldz;
            T* const g = reinterpret_cast<T*>(a.grad) + (uint64_t)row * a.ldg;
            if (!slot.keep) {
                if ((kWhat & kLoss) && threadIdx.x == 0) {
                    a.row_loss[row] = 0.f, a.stats[row] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (a.loss != nullptr) *a.loss = 0.f;
                }
                if (kWhat & kGrad) {
                    const RowShape gs = row_shape(g, a.vocab);
                    uint4* gv = reinterpret_cast<uint4*>(g + gs.head);
                    for (uint32_t i = threadIdx.x; i < gs.vecs; i += threads) __stcs(gv + i, make_uint4(0, 0, 0, 0));
                    if (threadIdx.x < gs.head) g[threadIdx.x] = Type<T>::round(0.f);
                    if (threadIdx.x < gs.tail) g[a.vocab - gs.tail + threadIdx.x] = Type<T>::round(0.f);
                }
                continue;
            }
            const RowShape shape = row_shape(z, a.vocab);
            const uint32_t edge = shape.head + shape.tail;  // elements outside of the vectors: one for each thread
            const uint32_t v_edge = threadIdx.x < shape.head ? threadIdx.x : threadIdx.x + shape.vecs * E;
            float f_edge = -INFINITY;
            if (threadIdx.x < edge) f_edge = Type<T>::load(z + v_edge);

            // the next chunk's vectors of this thread into q, of `count` that the row has left, after `look` saw them
            auto take = [&](uint4(&q)[kUnroll], uint32_t count, auto whole, auto&& look) {
                if (!tc::bar_wait(&full[at], phase, &gave_up)) lost = true;
                uint4* const from = reinterpret_cast<uint4*>(smem) + at * lay.chunk_vecs + threadIdx.x;
                look(from);
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) {
                    if constexpr (!decltype(whole)::value) {
                        q[u] = make_uint4(Type<T>::kNothing, Type<T>::kNothing, Type<T>::kNothing, Type<T>::kNothing);
                        if (threadIdx.x + u * threads >= count) continue;
                    }
                    q[u] = from[u * threads];
                }
                __syncwarp();
                if (lane == 0) tc::bar_arrive(&empty[at]);  // read: the chunk's place may be filled again
                if (++at == lay.slots) at = 0, phase ^= 1;
            };
            const uint32_t whole_vecs = shape.vecs / lay.chunk_vecs * lay.chunk_vecs;

            float M_out, outside;  // what the pass writes in the gradient is relative to
            if (kWhat & kLoss) {
                Running run;
                const uint32_t* const bits = listed[it & 1].bits;
                const uint8_t* const bytes = reinterpret_cast<const uint8_t*>(bits);
                const uint32_t* owners = listed[it & 1].owners + warp;
                auto add = [&](uint32_t v0, auto whole) {
                    const uint32_t count = shape.vecs - v0;
                    uint4 q[kUnroll];
                    take(q, count, whole, [&](uint4* from) {
                        if (!kBucket) return;
                        const bool some = (*owners >> lane) & 1;
                        owners += warps;
                        if (!some) return;
                        // the listed elements of this thread are summed apart, and taken out of the chunk
                        uint32_t in = 0;
#pragma unroll
                        for (uint32_t u = 0; u < kUnroll; ++u) {
                            const uint32_t i = v0 + threadIdx.x + u * threads;
                            if (i < shape.vecs)
                                in |= (E == 8 ? (uint32_t)bytes[i] : (bytes[i >> 1] >> (4 * (i & 1))) & 15u) << (8 * u);
                        }
                        for (; in != 0; in &= in - 1) {
                            const uint32_t bit = __ffs(in) - 1;
                            T* const e = reinterpret_cast<T*>(from + (bit >> 3) * threads) + (bit & 7);
                            run.add_listed(Type<T>::load(e), c);
                            *e = Type<T>::round(-INFINITY);
                        }
                        tc::fence_to_async();  // the next copy into this place comes after these writes
                    });
                    uint32_t top = Type<T>::kNothing;
#pragma unroll
                    for (int u = 0; u < kUnroll; ++u)
                        top = Type<T>::larger(
                            top, Type<T>::larger(Type<T>::larger(q[u].x, q[u].y), Type<T>::larger(q[u].z, q[u].w)));
                    run.raise(Type<T>::fold(top), c);
                    if (!run.o.far) {
                        const Pair c2(c, c), r2(-run.o.r, -run.o.r);
#pragma unroll
                        for (int u = 0; u < kUnroll; ++u) {
                            if (!decltype(whole)::value && u * threads >= count) break;
                            float f[E];
                            Type<T>::unpack(q[u], f);
#pragma unroll
                            for (int j = 0; j < E; j += 2) {
                                const float2 x = fma2(Pair(f[j], f[j + 1]), c2, r2).get();
                                run.out = add2(run.out, Pair(ex2(x.x), ex2(x.y)));
                            }
                        }
                    } else {
                        float out = 0.f;
#pragma unroll
                        for (int u = 0; u < kUnroll; ++u) {
                            float f[E];
                            Type<T>::unpack(q[u], f);
#pragma unroll
                            for (int j = 0; j < E; ++j) out += ex2(run.o.exponent(f[j], c));
                        }
                        run.out = add2(run.out, Pair(out, 0.f));
                    }
                };
                for (uint32_t v0 = 0; v0 < whole_vecs; v0 += lay.chunk_vecs) add(v0, std::true_type());
                if (whole_vecs < shape.vecs) add(whole_vecs, std::false_type());
                if (threadIdx.x < edge) {
                    bool in = false;
                    if (kBucket) {
                        const uint32_t bit = bit_of<T>(shape, v_edge);
                        in = (bits[bit >> 5] >> (bit & 31)) & 1;
                    }
                    if (in) {
                        run.add_listed(f_edge, c);
                    } else {
                        run.raise(f_edge, c);
                        run.out = add2(run.out, Pair(ex2(run.o.exponent(f_edge, c)), 0.f));
                    }
                }
                // join the threads
                float m = run.o.m;
#pragma unroll
                for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
                const float f = lost ? NAN : run.o.factor(Origin(m, c), c);
                const float2 two = run.out.get();
                const float w_out = warp_sum((two.x + two.y) * f);
                if (lane == 0) s_m[warp] = m, s_out[warp] = w_out;
                // the listed ones' sum, from `from` to the largest of them
                auto bring = [c](float from, float to) { return from == -INFINITY ? 1.f : ex2((from - to) * c); };
                if (kBucket) {
                    float m_in = run.m_in;
#pragma unroll
                    for (int d = 16; d; d >>= 1) m_in = fmaxf(m_in, __shfl_xor_sync(0xffffffffu, m_in, d));
                    const float w_in = warp_sum(run.in * bring(run.m_in, m_in));
                    if (lane == 0) s_m_in[warp] = m_in, s_in[warp] = w_in;
                }
                asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory");  // the warps of the pass
                M_out = lane < warps ? s_m[lane] : -INFINITY;
                float out = lane < warps ? s_out[lane] : 0.f;
                const Origin mine(M_out, c);
#pragma unroll
                for (int d = 16; d; d >>= 1) M_out = fmaxf(M_out, __shfl_xor_sync(0xffffffffu, M_out, d));
                out = warp_sum(out * mine.factor(Origin(M_out, c), c));
                float M = M_out, Z = out, inside;
                if (kBucket) {
                    float m_in = lane < warps ? s_m_in[lane] : -INFINITY, in = lane < warps ? s_in[lane] : 0.f;
                    const float from = m_in;
#pragma unroll
                    for (int d = 16; d; d >>= 1) m_in = fmaxf(m_in, __shfl_xor_sync(0xffffffffu, m_in, d));
                    in = warp_sum(in * bring(from, m_in));
                    // both relative to M_out, unless a listed element is far above it: one approximate power less
                    const Origin others(M_out, c);
                    float rest = out;
                    if (M_out == -INFINITY ? m_in > -INFINITY : others.exponent(m_in, c) > 16.f)
                        M = m_in, rest *= others.factor(Origin(M, c), c);
                    if (m_in != -INFINITY) in *= ex2(Origin(M, c).exponent(m_in, c));
                    Z = rest + in;
                    inside = (float)slot.mass / Z;
                    outside = (float)((slot.mass * (double)(rest / Z) - slot.rest) / (double)out);
                    if (out == 0.f && Z > 0.f && slot.rest <= 0.0) outside = 0.f;  // nothing there, and nothing wanted
                } else {
                    inside = outside = (float)slot.mass / Z;
                }
                if (threadIdx.x == 0) {
                    slot.M = M, slot.Z = Z, slot.M_out = M_out, slot.out = out, slot.inside = inside;
                    a.stats[row] = make_float4(M, inside, outside, M_out);
                }
            } else {
                const float4 st = a.stats[row];
                M_out = st.w, outside = st.z;
                if (threadIdx.x == 0) slot.M = st.x, slot.inside = st.y;
            }

            if (kWhat & kGrad) {
                const float k_out = outside * slot.grad;
                const Origin o(M_out, c);
                const bool same_offset = (((uintptr_t)z ^ (uintptr_t)g) & 15u) == 0;
                auto write = [&](uint32_t v0, auto whole, auto plain) {
                    const Pair c2(c, c), r2(-o.r, -o.r), k2(k_out, k_out);
                    const uint32_t count = shape.vecs - v0;
                    uint4 q[kUnroll];
                    take(q, count, whole, [](uint4*) {});
                    T* const to = g + shape.head + ((uint64_t)v0 + threadIdx.x) * E;
#pragma unroll
                    for (int u = 0; u < kUnroll; ++u) {
                        if (!decltype(whole)::value && threadIdx.x + u * threads >= count) break;
                        float f[E];
                        Type<T>::unpack(q[u], f);
                        if constexpr (decltype(plain)::value) {
#pragma unroll
                            for (int j = 0; j < E; j += 2) {
                                const float2 x = fma2(Pair(f[j], f[j + 1]), c2, r2).get();
                                const float2 y = mul2(Pair(ex2(x.x), ex2(x.y)), k2).get();
                                f[j] = y.x, f[j + 1] = y.y;
                            }
                            __stcs(reinterpret_cast<uint4*>(to) + u * threads, Type<T>::pack(f));
                        } else {
#pragma unroll
                            for (int j = 0; j < E; ++j)
                                to[(uint64_t)u * threads * E + j] = Type<T>::round(ex2(o.exponent(f[j], c)) * k_out);
                        }
                    }
                };
                if (same_offset && !o.far) {
                    for (uint32_t v0 = 0; v0 < whole_vecs; v0 += lay.chunk_vecs) write(v0, std::true_type(), std::true_type());
                    if (whole_vecs < shape.vecs) write(whole_vecs, std::false_type(), std::true_type());
                } else {
                    for (uint32_t v0 = 0; v0 < shape.vecs; v0 += lay.chunk_vecs) write(v0, std::false_type(), std::false_type());
                }
                if (lost && shape.vecs > 0) g[shape.head] = Type<T>::round(NAN);
                if (threadIdx.x < edge) g[v_edge] = Type<T>::round(ex2(o.exponent(f_edge, c)) * k_out);
            }
        }
        asm volatile("bar.sync 2, %0;" ::"r"(threads + 32) : "memory");
    }
    __syncwarp();
    __syncthreads();
    if (threadIdx.x == 0 && gave_up) atomicAdd(&g_gave_up, 1u);
}

// 1 / max(1, rows kept)
__global__ void distill_count_kernel(const uint8_t* mask, uint32_t rows, float* inv_n)
{
    __shared__ uint32_t s[32];
    cudaGridDependencySynchronize();
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
    cudaGridDependencySynchronize();
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

template <typename T, bool kBucket, int kWhat, bool kLong>
int launch(const DistillArgs& a, const Layout& lay, size_t smem, uint32_t grid, cudaStream_t st)
{
    if (smem > kMostSmem) return PS_ERR_LIMIT;
    static std::atomic<uint64_t> seen{0};
    const int rc = allow_smem(distill_kernel<T, kBucket, kWhat, kLong>, kMostSmem, seen);
    if (rc != PS_OK) return rc;
    launch_behind(distill_kernel<T, kBucket, kWhat, kLong>, grid, lay.threads + 64, (uint32_t)smem, 0, st, a, lay);
    return ps_internal::after_launch();
}

template <typename T, bool kBucket, int kWhat>
int launch(const DistillArgs& a, cudaStream_t st)
{
    const int sms = ps_internal::sm_count();
    if (sms < 0) return sms;
    // Threads for a row by its size: four vectors a thread and chunk, four chunks.  Small CTAs, since each brings a
    // warp for listed entries and rows' own latencies overlap (8192 x 50257 fp16, loss: 158 us with 128 threads,
    // 167 us with 256; with the gradient and 8, 64 or 128 entries 308, 329 and 388 us, not 321, 343 and 448 us; with the
    // bucket and 64 entries 385 us, not 404 us; 4096 x 70000 bf16 222 us, not 230 us).  512 threads for the longest rows,
    // of which L2 keeps two an SM for the second pass, and where there is no more than one row for an SM.
    const uint64_t bytes = (uint64_t)a.vocab * sizeof(T);
    const bool few = a.rows <= (uint32_t)sms;
    const bool bits = kBucket && (kWhat & kLoss), seen = kWhat & kGrad;
    Layout lay;
    if (bytes <= 16 * 1024)
        lay.shift = 6;
    else if (!few && bytes <= 160 * 1024)
        lay.shift = 7;
    else
        lay.shift = bytes <= 32 * 1024 ? 8 : 9;
    size_t smem;
    for (;; --lay.shift) {
        lay.threads = 1u << lay.shift;
        lay.chunk_vecs = kUnroll * lay.threads;
        const size_t limit = (lay.shift == 9 ? 108 : 200) * 1024;  // two CTAs an SM
        for (lay.slots = kMaxSlots; lay.slots > 2 && smem_bytes(lay, a.k, a.vocab, bits, seen) > limit; --lay.slots) {}
        smem = smem_bytes(lay, a.k, a.vocab, bits, seen);
        if (smem <= kMostSmem || lay.shift == 6) break;  // the longest bitmaps leave room for small chunks only
    }
    const bool is_long = lay.shift == 9;
    // As many rows in work as SMs hold, but for the gradient no more than L2 keeps until the second pass.
    uint64_t most = 227 * 1024 / (smem + 2048);
    const uint64_t by_threads = is_long ? 2 : (uint64_t)kMaxThreads * kCtas / (lay.threads + 64);
    most = most < 1 ? 1 : most < by_threads ? most : by_threads;
    if ((kWhat & kLoss) && (kWhat & kGrad)) {
        const uint64_t fit = kRowsInL2 / ((uint64_t)sms * bytes);
        most = fit >= most ? most : fit < 2 ? (most < 2 ? most : 2) : fit;
    }
    most *= (uint64_t)sms;
    const uint32_t grid = a.rows < most ? a.rows : (uint32_t)most;
    return is_long ? launch<T, kBucket, kWhat, true>(a, lay, smem, grid, st)
                   : launch<T, kBucket, kWhat, false>(a, lay, smem, grid, st);
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
    // below the normal numbers log2(e) / temperature is not finite any more
    if (!(q->temperature >= FLT_MIN) || !(q->temperature < INFINITY) || !(q->weight < INFINITY) || !(q->weight > -INFINITY))
        return PS_ERR_INVALID;
    if (q->rows == 0) return PS_OK;
    if (q->vocab == 0 || q->k == 0) return PS_ERR_INVALID;
    if (q->vocab > (q->tail == PS_TAIL_BUCKET ? PS_DISTILL_MAX_VOCAB / 2 : PS_DISTILL_MAX_VOCAB) ||
        q->k > PS_DISTILL_MAX_K || q->rows > 0x7fffffffu)
        return PS_ERR_LIMIT;
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
    a.loss = reduce && q->rows == 1 ? loss_dev : nullptr;
    if (q->rows > 0) {
        if (a.inv_n != nullptr) {
            launch_behind(distill_count_kernel, 1, 1024, 0, 0, st, a.mask, q->rows, inv_n_dev);
            rc = ps_internal::after_launch();
            if (rc != PS_OK) return rc;
        }
        rc = launch(a, q->dtype, q->tail == PS_TAIL_BUCKET, grad ? kLoss | kGrad : kLoss, st);
        if (rc != PS_OK) return rc;
    }
    if (!reduce || a.loss != nullptr) return PS_OK;
    // no rows: a loss of 0
    launch_behind(distill_sum_kernel, 1, 1024, 0, 0, st, (const float*)row_loss_dev, q->rows,
                  q->rows > 0 ? a.inv_n : (const float*)nullptr, a.inv_n_value, loss_dev);
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

int ps_distill_gave_up(uint32_t* count)
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
