// launch_kernels_int8_loop: 8-bit integer KV cache, single-pass decode attention (no reference
// counterpart; the form, the checks and the scales are those of launch_kernels_fp8_loop).
#include "launch_common.cuh"

namespace pa {
int read_status_int8_loop(int *v) { return read_and_clear_device_status(v); }
} // namespace pa

PA_TIMELINE_ACCESSOR(pa_debug_timeline_int8_loop)
PA_BOUNDS_ACCESSOR(pa_debug_bounds_int8_loop)

extern "C" PA_API int launch_kernels_int8_loop(const pa_params *p, void *stream, float *us_out) {
  using namespace pa;
  if (int rc = validate_params(p, /*fp8_entry=*/true, /*needs_scratch=*/false, /*int8_entry=*/true)) return rc;
  if (us_out) us_out[0] = 0.f;
  if (p->num_seqs == 0) return PA_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return run_timed(
      s, us_out, [&] { return dispatch_head_size<KV_I8, MODE_LOOP>(p, s); }, [] { return 0; }, false);
}
