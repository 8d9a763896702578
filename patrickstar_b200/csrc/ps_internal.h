// What the translation units of the library share and do not export.
#ifndef PS_B200_INTERNAL_H
#define PS_B200_INTERNAL_H

#include <cuda_runtime.h>

#include <cstdint>

namespace ps_internal {

// Records a failed CUDA call for ps_last_cuda_error() of the calling thread.
__attribute__((visibility("hidden"))) void set_cuda_error(int e);
// Counts one launch of ps_launch_count() and reports the launch's own status.
__attribute__((visibility("hidden"))) int after_launch();
// SM count of the current device (kept after the first question), or a PS_ERR_* code.
__attribute__((visibility("hidden"))) int sm_count();

// One matrix of ps_block_quantize.
struct QuantizeJob {
    const void* x;
    int dtype;
    uint64_t ld;
    uint32_t rows, cols;
    int blocks, fmt;
    void *q1, *s1, *q0, *s0;
    uint64_t ldq;
    float* colsum;
};
__attribute__((visibility("hidden"))) int quantize(const QuantizeJob& j, cudaStream_t st);
// A layer's input (row or row and column blocks) and weight (tiles), both to e4m3, in one launch where
// their types agree.
__attribute__((visibility("hidden"))) int quantize_layer(const QuantizeJob& x, const QuantizeJob& w, cudaStream_t st);

}  // namespace ps_internal

#endif
