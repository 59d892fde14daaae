// Differential attention over the paged cache (no reference counterpart): launch of the attention
// kernel with two V heads per K head (paged_attention_kernel with VH = 2), shared by the units that
// instantiate it per cache type.  See launch_kernels_diff.cu for the mathematics and the second kernel.
#pragma once

#include "launch_common.cuh"

namespace pa {

// Partition size in tokens: the longest context spread evenly over the partitions that the scratch has
// room for, in steps of 64.  The last partition is open-ended, so a context beyond the caller's hint is
// still attended to its end.
inline uint32_t diff_partition_tokens(const pa_params *p) {
  const uint32_t longest = std::min(context_hint(p) != 0u ? context_hint(p) : context_limit(p), 1u << 30);
  const uint32_t even = divide_round_up(std::max(longest, 1u), p->max_num_partitions);
  return divide_round_up(even, 64u) * 64u;
}

template <int D, int KV, int TILES>
static int enqueue_diff(const pa_params *p, cudaStream_t stream, uint32_t hpc) {
  using L = SmemLayout<D, KV, 4, TILES, 2>;
  using policy = typename L::policy;
  DeviceInfo dev{};
  if (int rc = get_device_info(&dev)) return rc;
  if (dev.cc_major < 10) return fail(PA_ERR_CUDA, "this library needs an sm_100a device");
  AttnArgs args = make_attn_args<D, KV, 4, TILES>(p, hpc);
  args.partition_tokens = diff_partition_tokens(p);
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  if (stream != nullptr && stream != cudaStreamLegacy) PA_CUDA_TRY(cudaStreamIsCapturing(stream, &capture));
  args.sched_slot = next_sched_slot(capture != cudaStreamCaptureStatusNone);
  CUtensorMap map_k, map_v;
  if (int rc = encode_cache_map<D, KV>(&map_k, p->key_cache, p, args.rows_per_box, args.heads_per_box)) return rc;
  if (int rc = encode_cache_map<D, KV>(&map_v, p->value_cache, p, args.rows_per_box, args.heads_per_box)) return rc;
  auto kernel = paged_attention_kernel<D, KV, MODE_SPLIT, 4, TILES, 2>;
  static thread_local int configured_device = -1;
  int device = 0;
  PA_CUDA_TRY(cudaGetDevice(&device));
  if (configured_device != device) {
    PA_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::DYN_SMEM));
    configured_device = device;
  }
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  cfg.blockDim = dim3(policy::threads_per_cta, 1, 1);
  cfg.dynamicSmemBytes = L::DYN_SMEM;
  cfg.stream = stream;
  const uint64_t items = static_cast<uint64_t>(p->num_kv_heads / args.hpc) * p->max_num_partitions * p->num_seqs;
  const uint64_t resident = static_cast<uint64_t>(policy::ctas_per_sm) * static_cast<uint64_t>(dev.sm_count);
  cfg.gridDim = dim3(static_cast<unsigned>(std::min(items, resident)), 1, 1);
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  PA_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, map_k, map_v, args));
  return PA_OK;
}

// KV heads per CTA (whole pairs) and tiles per stage, by the rules of ordinary attention.  (CTAs of 8 warps and 8
// KV heads brought nothing here: 60 against 59 us on 2 x 65536 tokens of e4m3, weights in one part.)
template <int D, int KV>
static int dispatch_diff_tiles(const pa_params *p, cudaStream_t stream) {
  const uint32_t hpc = p->num_kv_heads % 4u == 0u ? 4u : 2u;
  const uint32_t tiles = choose_stage_tiles<D, KV>(p, hpc, 4u);
  if constexpr (max_stage_tiles<D, KV>() >= 4u) {
    if (tiles == 4u) return enqueue_diff<D, KV, 4>(p, stream, hpc);
  }
  if constexpr (max_stage_tiles<D, KV>() >= 2u) {
    if (tiles >= 2u) return enqueue_diff<D, KV, 2>(p, stream, hpc);
  }
  return enqueue_diff<D, KV, 1>(p, stream, hpc);
}

template <int KV>
static int dispatch_diff(const pa_params *p, cudaStream_t stream) {
  if (p->head_size == 128) return dispatch_diff_tiles<128, KV>(p, stream);
  return dispatch_diff_tiles<64, KV>(p, stream);
}

// one per unit: the kernel's tables exist once per translation unit
int enqueue_diff_f16(const pa_params *p, cudaStream_t stream);
int enqueue_diff_e5m2(const pa_params *p, cudaStream_t stream);
int enqueue_diff_e4m3(const pa_params *p, cudaStream_t stream);
int enqueue_diff_int8(const pa_params *p, cudaStream_t stream);

} // namespace pa
