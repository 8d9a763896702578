// What the translation units of the library share and do not export.
#ifndef PS_B200_INTERNAL_H
#define PS_B200_INTERNAL_H

#include <cuda_runtime.h>

namespace ps_internal {

// Records a failed CUDA call for ps_last_cuda_error() of the calling thread.
__attribute__((visibility("hidden"))) void set_cuda_error(int e);
// Counts one launch of ps_launch_count() and reports the launch's own status.
__attribute__((visibility("hidden"))) int after_launch();
// SM count of the current device (kept after the first question), or a PS_ERR_* code.
__attribute__((visibility("hidden"))) int sm_count();

}  // namespace ps_internal

#endif
