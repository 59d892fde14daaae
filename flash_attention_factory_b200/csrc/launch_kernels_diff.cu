// launch_kernels_diff: differential attention over the paged cache, one decode token per sequence (no
// reference counterpart).
//
//   o[h] = (softmax(s q[2h] K[2k]^T) - lambda[h] softmax(s q[2h+1] K[2k+1]^T)) [V[2k] V[2k+1]]
//
// The value product is linear in the weights, so the two maps never meet before the end: the attention
// kernel treats them as two query heads of one KV pair, each with its own K head, online softmax and
// partial rows over the pair's two V heads, and the second kernel merges the partitions of both maps,
// subtracts, and applies the norm of the row.
// Bound by HBM like ordinary attention: K and V of a pair are streamed once for both maps of all its
// query heads.
#include "differential_attention.cuh"

namespace pa {

int read_status_diff(int *v) { return read_and_clear_device_status(v); }
int enqueue_diff_f16(const pa_params *p, cudaStream_t stream) { return dispatch_diff<KV_F16>(p, stream); }

namespace {

struct DiffMergeArgs {
  __half *out;          // [S, H, 2 D]
  const float *tmp_out; // [S, 2 H, NP, 2 D]
  const float *max_logits, *exp_sums;
  const uint32_t *context_lens, *seq_indices, *table_offsets;
  const float *lambdas, *norm_weight;
  uint32_t num_heads; // H
  uint32_t max_num_partitions, partition_tokens, ctx_limit, block_shift;
  float norm_eps, norm_scale;
};

// One CTA per (sequence, head), half of its threads per map.  A thread owns 4 of the row's 2 D dims and every
// CLASSES-th partition; the first rows are requested before the weights are known, so a context of up
// to UNROLL * CLASSES partitions costs one round trip to memory behind the context length.  Partitions
// are added in increasing order per class, classes in increasing order: the result does not depend on
// timing.
constexpr uint32_t kMergeWeights = 1024; // partitions whose weights are kept in shared memory

template <int D, int THREADS>
__global__ void __launch_bounds__(THREADS) merge_difference_kernel(const DiffMergeArgs a) {
  constexpr uint32_t ROW = 2 * D;
  constexpr uint32_t HALF_CTA = THREADS / 2;
  constexpr uint32_t LANES_PER_ROW = ROW / 4;               // 64 or 32 threads
  constexpr uint32_t CLASSES = HALF_CTA / LANES_PER_ROW;    // partitions that a map takes at a time
  constexpr uint32_t UNROLL = 8;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const uint32_t head = blockIdx.x;
  const uint32_t seq = (a.seq_indices != nullptr) ? __ldg(a.seq_indices + blockIdx.y) : blockIdx.y;
  const uint32_t map = tid / HALF_CTA;
  const uint32_t cls = (tid % HALF_CTA) / LANES_PER_ROW;
  const uint32_t col = (tid % LANES_PER_ROW) * 4u;
  const uint32_t NP = a.max_num_partitions;
  const size_t base = ((static_cast<size_t>(seq) * a.num_heads + head) * 2u + map) * NP;

  __shared__ float weights[2][kMergeWeights];
  __shared__ float top[2], inverse[2];
  __shared__ float part[2][CLASSES][ROW];
  __shared__ float squares[2];

  float4 rows[UNROLL];
#pragma unroll
  for (uint32_t u = 0; u < UNROLL; ++u) {
    const uint32_t p = cls + u * CLASSES;
    rows[u] = (p < NP) ? __ldcg(reinterpret_cast<const float4 *>(a.tmp_out + (base + p) * ROW + col))
                       : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const uint32_t ctx = merge_context(a.context_lens, seq, a.ctx_limit, a.table_offsets, a.block_shift);
  const uint32_t np = min(divide_round_up(ctx, a.partition_tokens), NP); // as the first kernel counts
  // one warp per map: largest logit, weights and total weight of its partitions
  if (tid % HALF_CTA < 32u) {
    float m = neg_infinity();
    for (uint32_t p = lane; p < np; p += 32) m = fmaxf(m, a.max_logits[base + p]);
#pragma unroll
    for (uint32_t o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float total = 0.f;
    for (uint32_t p = lane; p < np; p += 32) {
      const float w = a.exp_sums[base + p] * __expf(a.max_logits[base + p] - m);
      if (p < kMergeWeights) weights[map][p] = w;
      total += w;
    }
#pragma unroll
    for (uint32_t o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (lane == 0) {
      top[map] = m;
      inverse[map] = (total > 0.f) ? 1.f / total : 0.f;
    }
  }
  __syncthreads();
  const float m = top[map], inv = inverse[map];
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float4 v, uint32_t p) {
    const float w =
        ((p < kMergeWeights) ? weights[map][p] : a.exp_sums[base + p] * __expf(a.max_logits[base + p] - m)) * inv;
    sum.x += w * v.x;
    sum.y += w * v.y;
    sum.z += w * v.z;
    sum.w += w * v.w;
  };
#pragma unroll
  for (uint32_t u = 0; u < UNROLL; ++u) {
    const uint32_t p = cls + u * CLASSES;
    if (p < np) add(rows[u], p);
  }
  for (uint32_t p0 = cls + UNROLL * CLASSES; p0 < np; p0 += UNROLL * CLASSES) {
#pragma unroll
    for (uint32_t u = 0; u < UNROLL; ++u) {
      const uint32_t p = p0 + u * CLASSES;
      if (p < np) rows[u] = __ldcg(reinterpret_cast<const float4 *>(a.tmp_out + (base + p) * ROW + col));
    }
#pragma unroll
    for (uint32_t u = 0; u < UNROLL; ++u) {
      const uint32_t p = p0 + u * CLASSES;
      if (p < np) add(rows[u], p);
    }
  }
  *reinterpret_cast<float4 *>(&part[map][cls][col]) = sum;
  __syncthreads();
  // the first ROW / 4 threads: difference of the maps, norm, store
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  const bool active = tid < LANES_PER_ROW;
  if (active) {
    const float lambda = __ldg(a.lambdas + head);
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      float o0 = 0.f, o1 = 0.f;
#pragma unroll
      for (uint32_t k = 0; k < CLASSES; ++k) {
        o0 += part[0][k][col + j];
        o1 += part[1][k][col + j];
      }
      x[j] = o0 - lambda * o1;
    }
    if (a.norm_weight != nullptr) {
      float q = x[0] * x[0] + x[1] * x[1] + x[2] * x[2] + x[3] * x[3];
#pragma unroll
      for (uint32_t o = 16; o > 0; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
      if (lane == 0) squares[warp] = q;
    }
  }
  if (a.norm_weight != nullptr) {
    __syncthreads();
    if (active) {
      float q = squares[0];
      if (LANES_PER_ROW == 64) q += squares[1];
      const float r = rsqrtf(q / static_cast<float>(ROW) + a.norm_eps) * a.norm_scale;
      const float4 w = __ldg(reinterpret_cast<const float4 *>(a.norm_weight + col));
      x[0] *= r * w.x;
      x[1] *= r * w.y;
      x[2] *= r * w.z;
      x[3] *= r * w.w;
    }
  }
  if (active)
    *reinterpret_cast<uint2 *>(a.out + (static_cast<size_t>(seq) * a.num_heads + head) * ROW + col) =
        make_uint2(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]));
}

template <int D>
int enqueue_difference(const pa_diff_params *d, cudaStream_t stream) {
  const pa_params *p = &d->attn;
  DiffMergeArgs a{};
  a.out = static_cast<__half *>(p->out);
  a.tmp_out = static_cast<const float *>(p->tmp_out);
  a.max_logits = p->max_logits;
  a.exp_sums = p->exp_sums;
  a.context_lens = p->context_lens;
  a.seq_indices = p->seq_indices;
  a.table_offsets = p->block_table_offsets;
  a.lambdas = d->lambdas;
  a.norm_weight = d->norm_weight;
  a.num_heads = p->num_heads / 2u;
  a.max_num_partitions = p->max_num_partitions;
  a.partition_tokens = diff_partition_tokens(p);
  a.ctx_limit = context_limit(p);
  a.block_shift = log2_pow2(p->block_size);
  a.norm_eps = d->norm_eps;
  a.norm_scale = d->norm_scale;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(a.num_heads, p->num_seqs, 1);
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // Many partitions of few rows: more threads take more of them at a time (64 rows of 74 partitions: 10 us
  // instead of 15).  With more rows than the GPU holds CTAs of 1024 threads the small ones win (768 rows of 48:
  // 11 us instead of 25).
  if (p->max_num_partitions > 32u && static_cast<uint64_t>(a.num_heads) * p->num_seqs <= 296u) {
    cfg.blockDim = dim3(1024, 1, 1);
    PA_CUDA_TRY(cudaLaunchKernelEx(&cfg, merge_difference_kernel<D, 1024>, a));
  } else {
    cfg.blockDim = dim3(256, 1, 1);
    PA_CUDA_TRY(cudaLaunchKernelEx(&cfg, merge_difference_kernel<D, 256>, a));
  }
  return PA_OK;
}

int validate_diff(const pa_diff_params *d) {
  if (d == nullptr) return fail(PA_ERR_BAD_ARG, "params is null");
  const pa_params *p = &d->attn;
  const int32_t kv = p->kv_dtype;
  if (kv != PA_KV_F16 && kv != PA_KV_FP8_E5M2 && kv != PA_KV_FP8_E4M3 && kv != PA_KV_INT8)
    return fail(PA_ERR_BAD_ARG, "unknown kv_dtype %d", kv);
  if (int rc = validate_params(p, kv != PA_KV_F16, /*needs_scratch=*/true, kv == PA_KV_INT8)) return rc;
  if (p->sinks != nullptr || p->alibi_slopes != nullptr || p->softcap > 0.f)
    return fail(PA_ERR_UNSUPPORTED, "differential attention takes no sinks, alibi_slopes or softcap");
  if (p->num_seqs == 0) return PA_OK;
  if (p->num_kv_heads % 2u != 0u)
    return fail(PA_ERR_BAD_ARG, "differential attention needs KV heads in pairs, got %u", p->num_kv_heads);
  if (d->lambdas == nullptr) return fail(PA_ERR_BAD_ARG, "lambdas is null");
  if (d->norm_weight != nullptr) {
    if (!(d->norm_eps > 0.f)) return fail(PA_ERR_BAD_ARG, "norm_eps must be positive");
    if (!aligned16(d->norm_weight)) return fail(PA_ERR_BAD_ARG, "norm_weight must be 16-byte aligned");
  }
  return PA_OK;
}

} // namespace
} // namespace pa

PA_TIMELINE_ACCESSOR(pa_debug_timeline_diff)
PA_BOUNDS_ACCESSOR(pa_debug_bounds_diff)

extern "C" PA_API uint32_t pa_diff_num_partitions(uint32_t num_seqs, uint32_t num_kv_heads, uint32_t head_size,
                                                  uint32_t max_context_len, int32_t kv_dtype) {
  using namespace pa;
  if ((head_size != 128 && head_size != 64) || num_kv_heads == 0 || num_kv_heads % 2u != 0u) return 0;
  if (kv_dtype != PA_KV_F16 && kv_dtype != PA_KV_FP8_E5M2 && kv_dtype != PA_KV_FP8_E4M3 && kv_dtype != PA_KV_INT8) return 0;
  if (max_context_len == 0 || num_seqs == 0) return 1;
  // An item (a partition of the 4 or 2 heads of a CTA) of 512 KB: smaller ones show the cost of an item, larger
  // ones leave CTAs idle at the end of a ragged batch (48 sequences up to 8192 tokens, fp16, 8 KV heads of 128:
  // 127 us with 256 tokens, 138 with 512, 167 with 1024, 149 with 171).
  const uint32_t hpc = num_kv_heads % 4u == 0u ? 4u : 2u;
  const uint32_t token_bytes = hpc * head_size * 2u * (kv_dtype == PA_KV_F16 ? 2u : 1u);
  const uint64_t longest = max_context_len; // 64 bits: rounding a hint of nearly 2^32 up passes 32
  const uint32_t usual_tokens = (512u << 10) / token_bytes;
  const uint64_t usual = (longest + usual_tokens - 1u) / usual_tokens;
  const uint64_t units = static_cast<uint64_t>(num_seqs) * (num_kv_heads / hpc);
  const uint64_t items = units * usual, slots = 296u; // CTAs resident on 148 SMs
  uint64_t parts = usual;
  // With few items the last round of CTAs counts: the contexts are cut so that whole rounds are full, in
  // partitions of at least 64 tokens (2 sequences of 65536 tokens, e4m3: 58 us with 74 partitions, one item for
  // every CTA, 68 us with 128, 81 us with 111).
  if (items < 4u * slots) {
    const uint64_t rounds = std::max<uint64_t>(1u, items / slots);
    parts = std::max<uint64_t>(1u, rounds * slots / units);
    parts = std::min<uint64_t>(parts, (longest + 63u) / 64u);
  }
  return static_cast<uint32_t>(std::min<uint64_t>(65535u, parts)); // the kernel's index arithmetic
}

extern "C" PA_API int launch_kernels_diff(const pa_diff_params *p, void *stream, float *us_out) {
  using namespace pa;
  if (int rc = validate_diff(p)) return rc;
  if (us_out) us_out[0] = us_out[1] = 0.f;
  const pa_params *q = &p->attn;
  if (q->num_seqs == 0) return PA_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto attention = [&] {
    switch (q->kv_dtype) {
    case PA_KV_F16: return enqueue_diff_f16(q, s);
    case PA_KV_FP8_E5M2: return enqueue_diff_e5m2(q, s);
    case PA_KV_FP8_E4M3: return enqueue_diff_e4m3(q, s);
    default: return enqueue_diff_int8(q, s);
    }
  };
  return run_timed(
      s, us_out, attention,
      [&] { return q->head_size == 128 ? enqueue_difference<128>(p, s) : enqueue_difference<64>(p, s); }, true);
}
