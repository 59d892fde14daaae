// pa_append_block_scaled: appends new K/V tokens to an 8-bit cache that keeps one scale for each block of
// tokens and KV head, and keeps those scales (no reference counterpart).
//
// For every block and head that new rows reach, K and V each, with s the scale so far (0 for a block
// that starts with a new row) and q the largest code (127, 448, 57344):
//   s' = max(s, max|new rows| / q)
//   rows held before:  code' = round(code * s / s')   (only where s' > s)
//   new rows:          code  = round(x / s')
// x is the fp32 value of the row, rotated on the way if the call asks for it (see rope_cache.cu).
// Bound by HBM on prompts (every new element is read once from memory and its code written once)
// and by latency on decode steps: context length -> block id -> scale and rows -> codes.
#include "cache_codes.cuh"
#include "launch_common.cuh"

namespace pa {
namespace {

struct AppendArgs {
  const __half *query, *key, *value;
  __half *query_out;
  void *key_cache, *value_cache;
  float *k_scales, *v_scales;
  const uint32_t *block_tables, *context_lens, *cu_tokens;
  const float *cos_sin;
  uint64_t position_limit; // tokens at or behind it are skipped (table row, rotation table)
  uint64_t query_stride, key_stride, value_stride;
  uint64_t num_blocks;
  uint32_t num_seqs, num_tokens, num_heads, num_kv_heads, head_size, block_shift, block_size, max_blocks_per_seq;
  uint32_t rotary_dim;
  uint32_t tokens_per_cta; // 1..32
};

template <int KV>
__device__ __forceinline__ float largest_code() {
  return (KV == KV_I8) ? 127.f : (KV == KV_E4M3) ? 448.f : 57344.f;
}

// Where one new token goes.
struct TokenPlace {
  uint32_t position;
  uint32_t block;
  uint32_t rows_here; // new rows of the call that land in the same block from this token on
  bool valid;
  bool leads;         // first new token of its block
};

// Sequence of a token by bisection of the row offsets, then its position, block and neighbours.
__device__ __forceinline__ TokenPlace place_token(const AppendArgs &a, uint32_t token) {
  TokenPlace t{};
  if (token >= a.num_tokens) return t;
  uint32_t seq = token, begin = token, end = token + 1;
  if (a.cu_tokens != nullptr) {
    uint32_t lo = 0, hi = a.num_seqs + 1; // first offset beyond the token
    while (lo < hi) {
      const uint32_t mid = (lo + hi) >> 1;
      if (__ldg(a.cu_tokens + mid) <= token) lo = mid + 1;
      else hi = mid;
    }
    if (lo == 0 || lo > a.num_seqs) return t; // before the first or behind the last sequence
    seq = lo - 1;
    begin = __ldg(a.cu_tokens + seq);
    end = min(__ldg(a.cu_tokens + lo), a.num_tokens);
  }
  const int64_t position = static_cast<int64_t>(__ldg(a.context_lens + seq)) - (end - token);
  if (position < 0 || static_cast<uint64_t>(position) >= a.position_limit) return t;
  t.position = static_cast<uint32_t>(position);
  t.block = __ldg(a.block_tables + static_cast<size_t>(seq) * a.max_blocks_per_seq + (t.position >> a.block_shift));
  if (t.block >= a.num_blocks) return t;
  const uint32_t row = t.position & (a.block_size - 1u);
  t.leads = row == 0 || token == begin || t.position == 0;
  const uint64_t room = min(static_cast<uint64_t>(a.block_size - row), a.position_limit - t.position);
  t.rows_here = static_cast<uint32_t>(min(room, static_cast<uint64_t>(end - token)));
  t.valid = true;
  return t;
}

// One warp: K or V rows [0, rows) of one (block, head), rows laid over the lanes in items of 16 elements.
template <int KV, bool INTERLEAVED>
__device__ void append_rows(const AppendArgs &a, const __half *src, uint64_t stride, bool rotate, uint32_t position,
                            uint8_t *block_rows, float *scale_at, uint32_t first_row, uint32_t rows, uint32_t lane) {
  const uint32_t D = a.head_size;
  const uint32_t lanes_per_row = D / 16u;
  const uint32_t rows_per_pass = 32u / lanes_per_row;
  const uint32_t item = lane % lanes_per_row, lane_row = lane / lanes_per_row;
  const bool active = lane_row < rows_per_pass;
  const RotaryItem rot = rotate ? rotary_item(item, a.rotary_dim, INTERLEAVED) : rotary_item(item, 0u, false);
  const size_t pitch = static_cast<size_t>(a.num_kv_heads) * D; // bytes between two rows of the block

  auto load_row = [&](uint32_t r, float (&x)[8], float (&y)[8]) {
    const __half *row = src + static_cast<size_t>(r) * stride;
    unpack_half8(__ldg(reinterpret_cast<const uint4 *>(row + rot.first)), x);
    unpack_half8(__ldg(reinterpret_cast<const uint4 *>(row + rot.second)), y);
    // infinities count as the largest fp16 value, so that one of them does not take the block's scale
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (isinf(x[j])) x[j] = copysignf(65504.f, x[j]);
      if (isinf(y[j])) y[j] = copysignf(65504.f, y[j]);
    }
    if (rot.rotated) {
      float c[8], s[8];
      load_cos_sin(a.cos_sin + static_cast<size_t>(position + r) * a.rotary_dim, item, a.rotary_dim, c, s);
      rotate_item(x, y, c, s, INTERLEAVED);
    }
  };

  const float held = (first_row == 0u) ? 0.f : *scale_at;
  float top = 0.f; // NaNs drop out of fmaxf
  for (uint32_t r = lane_row; active && r < rows; r += rows_per_pass) {
    float x[8], y[8];
    load_row(r, x, y);
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, fmaxf(fabsf(x[j]), fabsf(y[j])));
  }
#pragma unroll
  for (uint32_t o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float scale = fmaxf(held, __fdiv_rn(top, largest_code<KV>()));
  const float by = (scale > 0.f) ? scale : 1.f; // a block of zeros keeps scale 0 and codes 0

  if (scale > held && active) {
    // the rows held before, under the new scale
    for (uint32_t r = lane_row; r < first_row; r += rows_per_pass) {
      uint4 *at = reinterpret_cast<uint4 *>(block_rows + r * pitch + item * 16u);
      uint4 v = *at;
      uint32_t *w = reinterpret_cast<uint32_t *>(&v);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x[4];
        unpack_codes<KV>(w[i], x);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = __fdiv_rn(__fmul_rn(x[j], held), by);
        w[i] = pack_codes<KV>(x[0], x[1], x[2], x[3]);
      }
      *at = v;
    }
  }
  for (uint32_t r = lane_row; active && r < rows; r += rows_per_pass) {
    float x[8], y[8];
    load_row(r, x, y);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = __fdiv_rn(x[j], by);
      y[j] = __fdiv_rn(y[j], by);
    }
    uint8_t *row = block_rows + (first_row + r) * pitch;
    *reinterpret_cast<uint2 *>(row + rot.first) =
        make_uint2(pack_codes<KV>(x[0], x[1], x[2], x[3]), pack_codes<KV>(x[4], x[5], x[6], x[7]));
    *reinterpret_cast<uint2 *>(row + rot.second) =
        make_uint2(pack_codes<KV>(y[0], y[1], y[2], y[3]), pack_codes<KV>(y[4], y[5], y[6], y[7]));
  }
  __syncwarp(); // every lane has read the old scale
  if (lane == 0) *scale_at = scale;
}

// A CTA owns tokens_per_cta consecutive new tokens: it appends the blocks whose first new token is among
// them (a block belongs to exactly one CTA whatever its later tokens) and rotates the tokens' queries.
// Every warp works out the places of the tokens for itself, a token per lane, and takes every n-th
// (head, K or V) of a block.
template <int KV, bool INTERLEAVED>
__global__ void __launch_bounds__(512) append_block_scaled_kernel(const AppendArgs a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const uint32_t token0 = blockIdx.x * a.tokens_per_cta;
  TokenPlace mine{};
  if (lane < a.tokens_per_cta) mine = place_token(a, token0 + lane);
  const uint32_t D = a.head_size;
  const uint32_t heads = a.num_kv_heads;

  uint32_t leaders = __ballot_sync(0xffffffffu, mine.valid && mine.leads);
  while (leaders != 0u) {
    const uint32_t src = __ffs(leaders) - 1u;
    leaders &= leaders - 1u;
    const uint32_t position = __shfl_sync(0xffffffffu, mine.position, src);
    const uint32_t block = __shfl_sync(0xffffffffu, mine.block, src);
    const uint32_t rows = __shfl_sync(0xffffffffu, mine.rows_here, src);
    const uint32_t first_row = position & (a.block_size - 1u);
    const size_t token = token0 + src;
    for (uint32_t job = warp; job < 2u * heads; job += warps) {
      const bool is_v = job >= heads;
      const uint32_t head = is_v ? job - heads : job;
      const uint64_t stride = is_v ? a.value_stride : a.key_stride;
      const __half *rows_src = (is_v ? a.value : a.key) + token * stride + static_cast<size_t>(head) * D;
      uint8_t *block_rows = static_cast<uint8_t *>(is_v ? a.value_cache : a.key_cache) +
                            (static_cast<size_t>(block) * a.block_size * heads + head) * D;
      float *scale_at = (is_v ? a.v_scales : a.k_scales) + static_cast<size_t>(block) * heads + head;
      append_rows<KV, INTERLEAVED>(a, rows_src, stride, !is_v && a.cos_sin != nullptr, position, block_rows, scale_at,
                                   first_row, rows, lane);
    }
  }

  if (a.query == nullptr) return;
  uint32_t live = __ballot_sync(0xffffffffu, mine.valid);
  const uint32_t lanes_per_head = D / 16u;
  const uint32_t heads_per_pass = blockDim.x / lanes_per_head;
  const uint32_t item = threadIdx.x % lanes_per_head, head0 = threadIdx.x / lanes_per_head;
  const RotaryItem rot = rotary_item(item, a.cos_sin != nullptr ? a.rotary_dim : 0u, INTERLEAVED);
  while (live != 0u) {
    const uint32_t src = __ffs(live) - 1u;
    live &= live - 1u;
    const uint32_t position = __shfl_sync(0xffffffffu, mine.position, src);
    const size_t token = token0 + src;
    if (head0 >= heads_per_pass) continue;
    float c[8], s[8];
    if (rot.rotated) load_cos_sin(a.cos_sin + static_cast<size_t>(position) * a.rotary_dim, item, a.rotary_dim, c, s);
    for (uint32_t head = head0; head < a.num_heads; head += heads_per_pass) {
      const __half *row = a.query + token * a.query_stride + static_cast<size_t>(head) * D;
      __half *dst = a.query_out + (token * a.num_heads + head) * D;
      float x[8], y[8];
      unpack_half8(__ldg(reinterpret_cast<const uint4 *>(row + rot.first)), x);
      unpack_half8(__ldg(reinterpret_cast<const uint4 *>(row + rot.second)), y);
      if (rot.rotated) rotate_item(x, y, c, s, INTERLEAVED);
      *reinterpret_cast<uint4 *>(dst + rot.first) = pack_half8(x);
      *reinterpret_cast<uint4 *>(dst + rot.second) = pack_half8(y);
    }
  }
}

template <int KV>
int launch_append(const AppendArgs &a, bool interleaved, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(divide_round_up(a.num_tokens, a.tokens_per_cta), 1, 1);
  cfg.blockDim = dim3(32u * std::min(16u, std::max(4u, 2u * a.num_kv_heads)), 1, 1);
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto kernel = interleaved ? append_block_scaled_kernel<KV, true> : append_block_scaled_kernel<KV, false>;
  PA_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a));
  return PA_OK;
}

} // namespace
} // namespace pa

extern "C" PA_API int pa_append_block_scaled(const pa_block_scaled_params *p, void *stream) {
  using namespace pa;
  if (p == nullptr) return fail(PA_ERR_BAD_ARG, "params is null");
  if (p->kv_dtype != PA_KV_INT8 && p->kv_dtype != PA_KV_FP8_E4M3 && p->kv_dtype != PA_KV_FP8_E5M2)
    return fail(PA_ERR_BAD_ARG, "block scales need an int8, e4m3 or e5m2 cache, got kv_dtype %d", p->kv_dtype);
  if (int rc = validate_rotation(p->head_size, p->rotary_dim, p->cos_sin, p->max_position, p->num_heads, p->query,
                                 p->query_out, p->query_token_stride, p->key_token_stride, p->value_token_stride))
    return rc;
  if (p->block_size == 0 || !is_pow2(p->block_size) || p->block_size > 1024u)
    return fail(PA_ERR_UNSUPPORTED, "block_size must be a power of two, at most 1024");
  if (p->num_kv_heads == 0 || p->num_kv_heads > 65535u) return fail(PA_ERR_BAD_ARG, "num_kv_heads must be in 1..65535");
  if (p->num_tokens == 0 || p->num_seqs == 0) return PA_OK;
  if (!p->key || !p->value || !p->key_cache || !p->value_cache || !p->k_scale_per_block || !p->v_scale_per_block ||
      !p->block_tables || !p->context_lens)
    return fail(PA_ERR_BAD_ARG, "a required pointer is null");
  if (p->num_blocks == 0 || p->max_blocks_per_seq == 0) return fail(PA_ERR_BAD_ARG, "empty cache");
  if (p->cu_tokens == nullptr && p->num_tokens != p->num_seqs)
    return fail(PA_ERR_BAD_ARG, "without cu_tokens every sequence has one new token: num_tokens must equal num_seqs");
  if (p->num_tokens > (1u << 30) || p->num_seqs > (1u << 30))
    return fail(PA_ERR_BAD_ARG, "num_tokens and num_seqs are limited to 2^30");
  if (!aligned16(p->key) || !aligned16(p->value) || !aligned16(p->key_cache) || !aligned16(p->value_cache))
    return fail(PA_ERR_BAD_ARG, "key / value / caches must be 16-byte aligned");
  AppendArgs a{};
  a.query = static_cast<const __half *>(p->query);
  a.key = static_cast<const __half *>(p->key);
  a.value = static_cast<const __half *>(p->value);
  a.query_out = static_cast<__half *>(p->query_out);
  a.key_cache = p->key_cache;
  a.value_cache = p->value_cache;
  a.k_scales = p->k_scale_per_block;
  a.v_scales = p->v_scale_per_block;
  a.block_tables = p->block_tables;
  a.context_lens = p->context_lens;
  a.cu_tokens = p->cu_tokens;
  a.cos_sin = p->cos_sin;
  a.position_limit = std::min<uint64_t>(static_cast<uint64_t>(p->max_blocks_per_seq) * p->block_size, 0xffffffffull);
  if (p->cos_sin != nullptr) a.position_limit = std::min<uint64_t>(a.position_limit, p->max_position);
  a.query_stride = p->query_token_stride;
  a.key_stride = p->key_token_stride;
  a.value_stride = p->value_token_stride;
  a.num_blocks = p->num_blocks;
  a.num_seqs = p->num_seqs;
  a.num_tokens = p->num_tokens;
  a.num_heads = p->num_heads;
  a.num_kv_heads = p->num_kv_heads;
  a.head_size = p->head_size;
  a.block_shift = log2_pow2(p->block_size);
  a.block_size = p->block_size;
  a.max_blocks_per_seq = p->max_blocks_per_seq;
  a.rotary_dim = p->cos_sin != nullptr ? p->rotary_dim : 0u;
  // as many tokens per CTA as a sequence has on average, up to a block: about one block per CTA
  // on prompts, one token on decode steps
  uint32_t per_cta = 1;
  if (p->cu_tokens != nullptr)
    while (per_cta < 32u && per_cta < p->block_size && per_cta * 2u <= p->num_tokens / p->num_seqs) per_cta *= 2u;
  a.tokens_per_cta = per_cta;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool interleaved = p->interleaved != 0u;
  if (p->kv_dtype == PA_KV_INT8) return launch_append<KV_I8>(a, interleaved, s);
  if (p->kv_dtype == PA_KV_FP8_E4M3) return launch_append<KV_E4M3>(a, interleaved, s);
  return launch_append<KV_E5M2>(a, interleaved, s);
}
