// launch_kernels_int8_reduce: 8-bit integer KV cache, split-context decode attention (no reference
// counterpart; the form, the checks and the scales are those of launch_kernels_fp8_reduce).
//
// Partial rows are fp32 where the caller's scratch is.  In fp16 their rounding is as large as that of the result
// (the weights, in two parts, no longer show beside them): 2.9e-4 instead of 2.1e-4 against fp64.
#include "launch_common.cuh"

namespace pa {
int read_status_int8_reduce(int *v) { return read_and_clear_device_status(v); }
} // namespace pa

PA_TIMELINE_ACCESSOR(pa_debug_timeline_int8_reduce)
PA_BOUNDS_ACCESSOR(pa_debug_bounds_int8_reduce)

extern "C" PA_API int launch_kernels_int8_reduce(const pa_params *p, void *stream, float *us_out) {
  using namespace pa;
  if (int rc = validate_params(p, /*fp8_entry=*/true, /*needs_scratch=*/true, /*int8_entry=*/true)) return rc;
  if (us_out) us_out[0] = us_out[1] = 0.f;
  if (p->num_seqs == 0) return PA_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return run_timed(
      s, us_out, [&] { return dispatch_head_size<KV_I8, MODE_SPLIT>(p, s); },
      [&] { return p->tmp_out_f32 != 0 ? dispatch_merge<float>(p, s) : dispatch_merge(p, s); }, true);
}
