// Attention kernel of launch_kernels_diff for int8 caches (see launch_kernels_diff.cu).
#include "differential_attention.cuh"

namespace pa {
int read_status_diff_int8(int *v) { return read_and_clear_device_status(v); }
int enqueue_diff_int8(const pa_params *p, cudaStream_t stream) { return dispatch_diff<KV_I8>(p, stream); }
} // namespace pa

PA_TIMELINE_ACCESSOR(pa_debug_timeline_diff_int8)
PA_BOUNDS_ACCESSOR(pa_debug_bounds_diff_int8)
