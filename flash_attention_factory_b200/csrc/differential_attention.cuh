// Differential attention over the paged cache (no reference counterpart): launch of the attention
// kernel with two V heads per K head (paged_attention_kernel with VH = 2), shared by the units that
// instantiate it per cache type.  See launch_kernels_diff.cu for the mathematics and the second kernel.
#pragma once

#include "launch_common.cuh"

namespace pa {

// KV heads per CTA: whole pairs, by the rule of ordinary attention.
inline uint32_t diff_heads_per_cta(const pa_params *p) { return p->num_kv_heads % 4u == 0u ? 4u : 2u; }

// Tiles per warp and stage, by the rule of ordinary attention.
template <int D, int KV>
uint32_t diff_stage_tiles(const pa_params *p) {
  return choose_stage_tiles<D, KV>(p, diff_heads_per_cta(p), 4u);
}

// Rows of a head that one TMA box copies (AttnArgs::rows_per_box of the launch).
inline uint32_t diff_box_rows(const pa_params *p) {
  const bool f16 = p->kv_dtype == PA_KV_F16; // the 8-bit types share their geometry
  const uint32_t tiles = p->head_size == 128 ? (f16 ? diff_stage_tiles<128, KV_F16>(p) : diff_stage_tiles<128, KV_E5M2>(p))
                                             : (f16 ? diff_stage_tiles<64, KV_F16>(p) : diff_stage_tiles<64, KV_E5M2>(p));
  return std::min(p->block_size, 64u / diff_heads_per_cta(p) * tiles);
}

// Partition size in tokens: the longest context spread evenly over the partitions that the scratch has
// room for, in steps of 64, or of a box where that has 128 rows (8-bit caches, head size 64, blocks of 128, an odd number
// of pairs): a box is copied out of one block, so a partition may only begin where a box does.  The last partition is
// open-ended, so a context beyond the caller's hint is still attended to its end.
inline uint32_t diff_partition_tokens(const pa_params *p) {
  const uint32_t longest = std::min(context_hint(p) != 0u ? context_hint(p) : context_limit(p), 1u << 30);
  const uint32_t even = divide_round_up(std::max(longest, 1u), p->max_num_partitions);
  const uint32_t step = std::max(64u, diff_box_rows(p));
  return divide_round_up(even, step) * step;
}

template <int D, int KV, int TILES>
static int enqueue_diff(const pa_params *p, cudaStream_t stream) {
  using L = SmemLayout<D, KV, 4, TILES, 2>;
  using policy = typename L::policy;
  DeviceInfo dev{};
  if (int rc = get_device_info(&dev)) return rc;
  if (dev.cc_major < 10) return fail(PA_ERR_CUDA, "this library needs an sm_100a device");
  AttnArgs args = make_attn_args<D, KV, 4, TILES>(p, diff_heads_per_cta(p));
  args.partition_tokens = diff_partition_tokens(p);
  if (args.partition_tokens % args.rows_per_box != 0u)
    return fail(PA_ERR_BAD_ARG, "partitions of %u tokens would begin inside a box of %u rows", args.partition_tokens,
                args.rows_per_box);
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

// (CTAs of 8 warps and 8 KV heads brought nothing here: 60 against 59 us on 2 x 65536 tokens of e4m3, weights in one
// part.)
template <int D, int KV>
static int dispatch_diff_tiles(const pa_params *p, cudaStream_t stream) {
  const uint32_t tiles = diff_stage_tiles<D, KV>(p);
  if constexpr (max_stage_tiles<D, KV>() >= 4u) {
    if (tiles == 4u) return enqueue_diff<D, KV, 4>(p, stream);
  }
  if constexpr (max_stage_tiles<D, KV>() >= 2u) {
    if (tiles >= 2u) return enqueue_diff<D, KV, 2>(p, stream);
  }
  return enqueue_diff<D, KV, 1>(p, stream);
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
