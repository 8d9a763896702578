// The linear layer on the 8-bit path: one call for the forward pass and one for
// the backward pass, so that a step spends its host time on two calls and not
// on nine.  What is kept between them is one buffer: the quantized input for the
// weight's gradient, the quantized weight for the input's.
#include "ps_b200.h"

#include "ps_internal.h"

namespace {

uint64_t round_up(uint64_t n, uint64_t to) { return (n + to - 1) / to * to; }
uint64_t row_bytes(uint32_t cols) { return round_up(cols, 16); }
uint64_t scale_bytes(uint64_t outer, uint64_t contracted)
{
    return (contracted + 511) / 512 * ((outer + 127) / 128) * 512;
}

// Takes pieces of a buffer, each from a 256-byte boundary on; with a null base it counts.
struct Pieces {
    char* base;
    uint64_t used = 0;
    void* take(uint64_t bytes)
    {
        void* p = base == nullptr ? nullptr : base + used;
        used += round_up(bytes, 256);
        return p;
    }
};

struct Saved {
    void *w, *ws0, *x, *xs0;
    Saved(Pieces& p, const ps_fp8_linear* q, int keep)
    {
        const bool own_w = (keep & PS_KEEP_WEIGHT) && q->kept_data == nullptr;
        w = own_w ? p.take(q->n * row_bytes(q->k)) : nullptr;
        ws0 = own_w ? p.take(scale_bytes(q->k, q->n)) : nullptr;
        x = (keep & PS_KEEP_INPUT) ? p.take(q->tokens * row_bytes(q->k)) : nullptr;
        xs0 = (keep & PS_KEEP_INPUT) ? p.take(scale_bytes(q->k, q->tokens)) : nullptr;
    }
};
struct ForwardScratch {
    void *x, *xs1, *w = nullptr, *ws1 = nullptr, *ws0 = nullptr;
    ForwardScratch(Pieces& p, const ps_fp8_linear* q, int keep)
    {
        x = p.take(q->tokens * row_bytes(q->k));
        xs1 = p.take(scale_bytes(q->tokens, q->k));
        if (q->kept_data != nullptr) return;
        ws1 = p.take(scale_bytes(q->n, q->k));
        if (keep & PS_KEEP_WEIGHT) return;
        w = p.take(q->n * row_bytes(q->k));
        ws0 = p.take(scale_bytes(q->k, q->n));
    }
};
struct BackwardScratch {
    void *g1, *s1, *g0, *s0;
    float* sums;
    BackwardScratch(Pieces& p, const ps_fp8_linear* q)
    {
        g1 = p.take(q->tokens * row_bytes(q->n));
        s1 = p.take(scale_bytes(q->tokens, q->n));
        g0 = p.take(q->tokens * row_bytes(q->n));
        s0 = p.take(scale_bytes(q->n, q->tokens));
        sums = (float*)p.take(((uint64_t)q->tokens + 127) / 128 * q->n * sizeof(float));
    }
};

int check_layer(const ps_fp8_linear* q)
{
    if (q == nullptr) return PS_ERR_INVALID;
    if (q->x_dtype < PS_DTYPE_F16 || q->x_dtype > PS_DTYPE_F32) return PS_ERR_INVALID;
    if (q->tokens > 0x7fffff00u || q->k > 0x7fffff00u || q->n > 0x7fffff00u) return PS_ERR_LIMIT;
    if (q->kept_data != nullptr && (q->kept_fmt != PS_FP8_E4M3 && q->kept_fmt != PS_FP8_E5M2)) return PS_ERR_INVALID;
    return PS_OK;
}

}  // namespace

extern "C" {

int ps_fp8_linear_sizes(const ps_fp8_linear* q, int keep, uint64_t* sizes)
{
    const int rc = check_layer(q);
    if (rc != PS_OK) return rc;
    if (sizes == nullptr) return PS_ERR_INVALID;
    Pieces saved{nullptr}, forward{nullptr}, backward{nullptr};
    Saved(saved, q, keep), ForwardScratch(forward, q, keep), BackwardScratch(backward, q);
    sizes[0] = saved.used, sizes[1] = forward.used, sizes[2] = backward.used;
    return PS_OK;
}

int ps_fp8_linear_forward(const ps_fp8_linear* q, int keep, void* y_dev, uint64_t ld_y, void* saved_dev,
                          void* scratch_dev, void* stream)
{
    int rc = check_layer(q);
    if (rc != PS_OK) return rc;
    if (q->tokens == 0 || q->n == 0) return PS_OK;
    if (scratch_dev == nullptr && q->k > 0) return PS_ERR_INVALID;
    if (((uintptr_t)saved_dev | (uintptr_t)scratch_dev) % 256) return PS_ERR_ALIGN;
    Pieces saved{(char*)saved_dev}, scratch{(char*)scratch_dev};
    const Saved kept(saved, q, keep);
    const ForwardScratch tmp(scratch, q, keep);
    if (saved.used > 0 && saved_dev == nullptr) return PS_ERR_INVALID;
    const bool both = keep & PS_KEEP_INPUT;
    const ps_internal::QuantizeJob x = {q->x, q->x_dtype, q->ld_x, q->tokens, q->k,
                                        both ? PS_BLOCKS_ROW_COL : PS_BLOCKS_ROW, PS_FP8_E4M3, tmp.x, tmp.xs1,
                                        kept.x, kept.xs0, row_bytes(q->k), nullptr};
    ps_block_operand a = {tmp.x, tmp.xs1, row_bytes(q->k), PS_FP8_E4M3, 1}, b;
    if (q->kept_data != nullptr) {
        rc = ps_internal::quantize(x, (cudaStream_t)stream);
        b = {q->kept_data, q->kept_scales1, q->ld_kept, q->kept_fmt, 1};
    } else {
        void* const w = kept.w != nullptr ? kept.w : tmp.w;
        const ps_internal::QuantizeJob job = {q->weight, q->weight_dtype, q->ld_weight, q->n, q->k, PS_BLOCKS_TILE,
                                              PS_FP8_E4M3, w, tmp.ws1, nullptr, kept.w != nullptr ? kept.ws0 : tmp.ws0,
                                              row_bytes(q->k), nullptr};
        rc = ps_internal::quantize_layer(x, job, (cudaStream_t)stream);
        b = {w, tmp.ws1, row_bytes(q->k), PS_FP8_E4M3, 1};
    }
    if (rc != PS_OK) return rc;
    return ps_block_matmul(&a, &b, q->tokens, q->n, q->k, q->bias, q->bias_dtype, y_dev, q->x_dtype, ld_y, stream);
}

int ps_fp8_linear_backward(const ps_fp8_linear* q, int keep, const void* saved_dev, const void* dy_dev, uint64_t ld_dy,
                           int grad_fmt, void* dx_dev, uint64_t ld_dx, void* dw_dev, void* db_dev, void* scratch_dev,
                           void* stream)
{
    int rc = check_layer(q);
    if (rc != PS_OK) return rc;
    if (grad_fmt != PS_FP8_E4M3 && grad_fmt != PS_FP8_E5M2) return PS_ERR_INVALID;
    if ((dx_dev != nullptr && !(keep & PS_KEEP_WEIGHT)) || (dw_dev != nullptr && !(keep & PS_KEEP_INPUT)))
        return PS_ERR_INVALID;
    if (((uintptr_t)saved_dev | (uintptr_t)scratch_dev) % 256) return PS_ERR_ALIGN;
    Pieces saved{(char*)const_cast<void*>(saved_dev)}, scratch{(char*)scratch_dev};
    const Saved kept(saved, q, keep);
    const BackwardScratch tmp(scratch, q);
    if ((saved.used > 0 && saved_dev == nullptr) || (scratch.used > 0 && scratch_dev == nullptr)) return PS_ERR_INVALID;
    const bool row = dx_dev != nullptr || db_dev != nullptr, col = dw_dev != nullptr || db_dev != nullptr;
    if (!row && !col) return PS_OK;
    rc = ps_internal::quantize({dy_dev, q->x_dtype, ld_dy, q->tokens, q->n,
                                row && col ? PS_BLOCKS_ROW_COL : row ? PS_BLOCKS_ROW : PS_BLOCKS_COL, grad_fmt, tmp.g1,
                                tmp.s1, tmp.g0, tmp.s0, row_bytes(q->n), db_dev != nullptr ? tmp.sums : nullptr},
                               (cudaStream_t)stream);
    if (rc == PS_OK && dx_dev != nullptr) {
        const ps_block_operand a = {tmp.g1, tmp.s1, row_bytes(q->n), grad_fmt, 1};
        const ps_block_operand b = q->kept_data != nullptr
                                       ? ps_block_operand{q->kept_data, q->kept_scales0, q->ld_kept, q->kept_fmt, 0}
                                       : ps_block_operand{kept.w, kept.ws0, row_bytes(q->k), PS_FP8_E4M3, 0};
        rc = ps_block_matmul(&a, &b, q->tokens, q->k, q->n, nullptr, 0, dx_dev, q->x_dtype, ld_dx, stream);
    }
    if (rc == PS_OK && dw_dev != nullptr) {
        const ps_block_operand a = {tmp.g0, tmp.s0, row_bytes(q->n), grad_fmt, 0};
        const ps_block_operand b = {kept.x, kept.xs0, row_bytes(q->k), PS_FP8_E4M3, 0};
        rc = ps_block_matmul(&a, &b, q->n, q->k, q->tokens, nullptr, 0, dw_dev, q->weight_dtype, q->k, stream);
    }
    if (rc == PS_OK && db_dev != nullptr)
        rc = ps_column_sum(tmp.sums, (uint32_t)(((uint64_t)q->tokens + 127) / 128), q->n, db_dev, q->bias_dtype, stream);
    return rc;
}

}  // extern "C"
