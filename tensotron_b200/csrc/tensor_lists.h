// Host entries of the kernels over lists of tensors (tensor_lists.cu), called by tt_clip_grad_norm_list and
// tt_adam_step_list.  The arrays of pointers and sizes are host memory, read during the call.
#pragma once
#include <cuda_runtime.h>

namespace tt {
namespace lists {

// Bytes of workspace launch_norm needs (partial sums), whatever the list.
constexpr int MAX_PARTIALS = 16384;
constexpr size_t WORKSPACE_BYTES = sizeof(double) * MAX_PARTIALS + 256;

// norm = sqrt(sum of squares over the list), coef = clamp(max_norm / (norm + eps), 0, 1) (NaN stays NaN); each is
// stored when its pointer is not null; scale: every element of the list is multiplied by coef.  `ticket` is a device
// word that is zero between launches.  *launches is increased by the kernels enqueued.
cudaError_t launch_clip(cudaStream_t st, int count, float* const* grads, const long long* sizes, float max_norm, float eps,
                        bool scale, float* norm_out, float* coef_out, void* workspace, unsigned int* ticket, int num_sms,
                        long long* launches);

// Adam over the list with the arguments of tt_adam_step; *grad_scale (device, optional) multiplies every gradient first.
cudaError_t launch_adam(cudaStream_t st, int count, float* const* p, const float* const* g, float* const* m,
                        float* const* v, const long long* sizes, float* adv, const float* grad_scale, float b1, float b2,
                        float lr, float eps, float cwd, float dfac, bool advance, unsigned int* ticket, int num_sms,
                        long long* launches);

// Loads the kernels, once per context (called from tt_create), so that a first call may be inside a capture.
cudaError_t init_lists();

}  // namespace lists
}  // namespace tt
