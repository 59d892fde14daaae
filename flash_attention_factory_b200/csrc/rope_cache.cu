// pa_rope_and_cache: the cache append of pa_reshape_and_cache with the rotary position embedding
// applied to K, and to the step's queries, on the way (no reference counterpart).
//
//   a' = a cos_i(p) - b sin_i(p),  b' = b cos_i(p) + a sin_i(p)     for every pair i of a head
//
// in fp32 from the fp16 inputs, rounded once: to fp16 (queries, fp16 caches) or, over the scale, to
// the 8-bit code.  Bound by HBM: every element is read once and written once, and one launch stands
// for the two rotations and the append.
#include "cache_codes.cuh"
#include "launch_common.cuh"

namespace pa {
namespace {

constexpr uint32_t kRopeThreads = 128;
constexpr uint32_t kRopeBatch = 3; // heads whose rows a thread requests together

struct RopeArgs {
  const __half *query, *key, *value;
  __half *query_out;
  void *key_cache, *value_cache;
  const int64_t *slots, *positions;
  const float *cos_sin;
  const float *k_scales, *v_scales; // per head or per block and head; unused for a scalar
  uint64_t num_slots, max_position, query_stride, key_stride, value_stride;
  uint32_t num_heads, num_kv_heads, head_size, block_size, rotary_dim;
  float scale;
};

template <int KV>
__device__ __forceinline__ void store_piece(void *row, uint32_t elem, const float (&x)[8], const Divider &by) {
  if constexpr (KV == KV_F16) {
    *reinterpret_cast<uint4 *>(static_cast<__half *>(row) + elem) = pack_half8(x);
  } else {
    float q[8] = {x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]};
    divide8(q, by);
    *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(row) + elem) =
        make_uint2(pack_codes<KV>(q[0], q[1], q[2], q[3]), pack_codes<KV>(q[4], q[5], q[6], q[7]));
  }
}

// One CTA per token.  A thread keeps one item of 16 elements (see rotary_item) for all the heads it
// visits, so the eight cosines and sines it needs are fetched once: lanes_per_head = head_size / 16
// neighbouring threads share a head, the CTA walks the rows query heads, K heads, V heads.
template <int KV, int SCALES, bool INTERLEAVED, bool CHAINED>
__global__ void __launch_bounds__(kRopeThreads) rope_and_cache_kernel(const RopeArgs a) {
  // decode-sized calls join the chain of programmatic launches, as the plain writer does
  if constexpr (CHAINED) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
  }
  const uint32_t token = blockIdx.x;
  const int64_t slot = __ldg(a.slots + token);
  const int64_t position = __ldg(a.positions + token);
  const uint32_t D = a.head_size;
  const uint32_t lanes_per_head = D / 16u;
  const uint32_t heads_per_pass = kRopeThreads / lanes_per_head;
  const uint32_t item = threadIdx.x % lanes_per_head;
  const uint32_t head0 = threadIdx.x / lanes_per_head;
  if (head0 >= heads_per_pass) return;
  const RotaryItem rot = rotary_item(item, a.rotary_dim, INTERLEAVED);
  const uint32_t rotated_heads = a.num_heads + a.num_kv_heads;
  const uint32_t total = rotated_heads + a.num_kv_heads;
  // the rows of kRopeBatch heads at a time; the first ones are on their way before the slot and the position
  // are known (the rows of a skipped token are read in vain)
  uint4 raw[kRopeBatch][2];
  auto load = [&](uint32_t first) {
#pragma unroll
    for (uint32_t i = 0; i < kRopeBatch; ++i) {
      const uint32_t head = first + i * heads_per_pass;
      if (head < total) {
        const bool is_v = head >= rotated_heads;
        const __half *src =
            (head < a.num_heads) ? a.query + static_cast<size_t>(token) * a.query_stride + static_cast<size_t>(head) * D
            : is_v ? a.value + static_cast<size_t>(token) * a.value_stride + static_cast<size_t>(head - rotated_heads) * D
                   : a.key + static_cast<size_t>(token) * a.key_stride + static_cast<size_t>(head - a.num_heads) * D;
        raw[i][0] = __ldg(reinterpret_cast<const uint4 *>(src + rot.first));
        raw[i][1] = __ldg(reinterpret_cast<const uint4 *>(src + rot.second));
      }
    }
  };
  load(head0);
  if (slot < 0 || static_cast<uint64_t>(slot) >= a.num_slots) return; // padding token / out of range
  if (position < 0 || static_cast<uint64_t>(position) >= a.max_position) return;
  float c[8], s[8];
  if (rot.rotated) load_cos_sin(a.cos_sin + static_cast<size_t>(position) * a.rotary_dim, item, a.rotary_dim, c, s);

  __half *qo = a.query_out + static_cast<size_t>(token) * a.num_heads * D;
  constexpr uint32_t ELT = (KV == KV_F16) ? 2u : 1u;
  const size_t row_bytes = static_cast<size_t>(a.num_kv_heads) * D * ELT;
  uint8_t *kc = static_cast<uint8_t *>(a.key_cache) + static_cast<size_t>(slot) * row_bytes;
  uint8_t *vc = static_cast<uint8_t *>(a.value_cache) + static_cast<size_t>(slot) * row_bytes;
  for (uint32_t first = head0; first < total; first += kRopeBatch * heads_per_pass) {
    if (first != head0) load(first);
#pragma unroll
    for (uint32_t i = 0; i < kRopeBatch; ++i) {
      const uint32_t head = first + i * heads_per_pass;
      if (head >= total) break;
      const bool is_v = head >= rotated_heads;
      const bool is_q = head < a.num_heads;
      const uint32_t kv_head = is_v ? head - rotated_heads : head - a.num_heads; // of K and V rows
      float x[8], y[8];
      unpack_half8(raw[i][0], x);
      unpack_half8(raw[i][1], y);
      if (rot.rotated && !is_v) rotate_item(x, y, c, s, INTERLEAVED); // V rows take the same two pieces
      if (is_q) {
        __half *dst = qo + static_cast<size_t>(head) * D;
        *reinterpret_cast<uint4 *>(dst + rot.first) = pack_half8(x);
        *reinterpret_cast<uint4 *>(dst + rot.second) = pack_half8(y);
      } else {
        uint8_t *dst = (is_v ? vc : kc) + static_cast<size_t>(kv_head) * D * ELT;
        float scale = a.scale;
        if constexpr (KV != KV_F16 && SCALES != SCALE_SCALAR) {
          const size_t si = (SCALES == SCALE_PER_HEAD)
                                ? kv_head
                                : static_cast<size_t>(slot / a.block_size) * a.num_kv_heads + kv_head;
          scale = __ldg((is_v ? a.v_scales : a.k_scales) + si);
        }
        const Divider by(scale);
        store_piece<KV>(dst, rot.first, x, by);
        store_piece<KV>(dst, rot.second, y, by);
      }
    }
  }
}

template <int KV, int SCALES>
int launch_rope(const RopeArgs &a, uint32_t num_tokens, bool interleaved, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(num_tokens, 1, 1);
  cfg.blockDim = dim3(kRopeThreads, 1, 1);
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  const bool chained = num_tokens <= 4096u; // the plain writer's rule
  cfg.numAttrs = chained ? 1 : 0;
  auto kernel = interleaved
                    ? (chained ? rope_and_cache_kernel<KV, SCALES, true, true> : rope_and_cache_kernel<KV, SCALES, true, false>)
                    : (chained ? rope_and_cache_kernel<KV, SCALES, false, true> : rope_and_cache_kernel<KV, SCALES, false, false>);
  PA_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a));
  return PA_OK;
}

template <int KV>
int dispatch_rope(const RopeArgs &a, const pa_cache_write_params &c, bool interleaved, cudaStream_t stream) {
  if constexpr (KV != KV_F16) {
    if (c.k_scale_per_head != nullptr) return launch_rope<KV, SCALE_PER_HEAD>(a, c.num_tokens, interleaved, stream);
    if (c.k_scale_per_block != nullptr) return launch_rope<KV, SCALE_PER_BLOCK>(a, c.num_tokens, interleaved, stream);
  }
  return launch_rope<KV, SCALE_SCALAR>(a, c.num_tokens, interleaved, stream);
}

} // namespace
} // namespace pa

extern "C" PA_API int pa_rope_and_cache(const pa_rope_cache_params *p, void *stream) {
  using namespace pa;
  if (p == nullptr) return fail(PA_ERR_BAD_ARG, "params is null");
  const pa_cache_write_params &c = p->cache;
  if (int rc = validate_cache_write(&c)) return rc;
  if (c.num_tokens == 0) return PA_OK;
  if (int rc = validate_rotation(c.head_size, p->rotary_dim, p->cos_sin, p->max_position, p->num_heads, p->query,
                                 p->query_out, p->query_token_stride, p->key_token_stride, p->value_token_stride))
    return rc;
  if (p->positions == nullptr || p->cos_sin == nullptr || p->rotary_dim == 0)
    return fail(PA_ERR_BAD_ARG, "positions, cos_sin and rotary_dim are required");
  RopeArgs a{};
  a.query = static_cast<const __half *>(p->query);
  a.key = static_cast<const __half *>(c.key);
  a.value = static_cast<const __half *>(c.value);
  a.query_out = static_cast<__half *>(p->query_out);
  a.key_cache = c.key_cache;
  a.value_cache = c.value_cache;
  a.slots = c.slot_mapping;
  a.positions = p->positions;
  a.cos_sin = p->cos_sin;
  a.k_scales = c.k_scale_per_head != nullptr ? c.k_scale_per_head : c.k_scale_per_block;
  a.v_scales = c.v_scale_per_head != nullptr ? c.v_scale_per_head : c.v_scale_per_block;
  a.num_slots = c.num_blocks * c.block_size;
  a.max_position = p->max_position;
  a.query_stride = p->query_token_stride;
  a.key_stride = p->key_token_stride;
  a.value_stride = p->value_token_stride;
  a.num_heads = p->query != nullptr ? p->num_heads : 0u;
  a.num_kv_heads = c.num_kv_heads;
  a.head_size = c.head_size;
  a.block_size = c.block_size;
  a.rotary_dim = p->rotary_dim;
  a.scale = c.fp8_scale;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool interleaved = p->interleaved != 0u;
  switch (c.kv_dtype) {
  case PA_KV_F16: return dispatch_rope<KV_F16>(a, c, interleaved, s);
  case PA_KV_FP8_E5M2: return dispatch_rope<KV_E5M2>(a, c, interleaved, s);
  case PA_KV_FP8_E4M3: return dispatch_rope<KV_E4M3>(a, c, interleaved, s);
  default: return dispatch_rope<KV_I8>(a, c, interleaved, s);
  }
}
