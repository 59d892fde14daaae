// pa_append_block_scaled: appends new K/V tokens to an 8-bit cache that keeps one scale for each block of
// tokens and KV head, and keeps those scales (no reference counterpart).
//
// For every block and head that new rows reach, K and V each, with s the scale so far (0 for a block
// that starts with a new row) and q the largest code (127, 448, 57344):
//   s' = max(s, max|new rows| / q)
//   rows held before:  code' = round(code * s / s')   (only where s' > s)
//   new rows:          code  = round(x / s')
// x is the fp32 value of the row, rotated on the way if the call asks for it (see rope_cache.cu).
// Every new element is read once from memory and its code written once.  Bound on prompts by the instructions per
// value and, where K is rotated, by the fetches of its angles from the L1 cache (twice the time of the bytes); on
// decode steps by latency: context length -> block id -> scale and rows -> codes.
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
  uint32_t warps_per_job;  // 1, 2, 4 or 8
  uint32_t append_ctas;    // CTAs of a column that append; the others rotate queries
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

// Sequence of this lane's token: the last entry of the row offsets that is not beyond it.  The warp holds every
// step-th offset in registers and bisects those with shuffles; what is left of the search (nothing up to
// 31 sequences) goes to memory.  Returns num_seqs for a token of no sequence.  Called by all lanes.
__device__ __forceinline__ uint32_t find_sequence(const AppendArgs &a, uint32_t token, uint32_t lane) {
  const uint32_t n = a.num_seqs + 1u;
  const uint32_t step = (n + 31u) / 32u;
  const uint32_t sample = (lane * step < n) ? __ldg(a.cu_tokens + lane * step) : 0xffffffffu;
  uint32_t k = 0; // samples that are not beyond the token, at most 31
#pragma unroll
  for (uint32_t b = 16; b > 0; b >>= 1)
    if (__shfl_sync(0xffffffffu, sample, k + b - 1u) <= token) k += b;
  if (__shfl_sync(0xffffffffu, sample, 31) <= token) k = 32;
  if (k == 0) return a.num_seqs;
  uint32_t lo = (k - 1u) * step, hi = min(lo + step, n); // the entry lies in [lo, hi)
  while (hi - lo > 1u) {
    const uint32_t mid = (lo + hi) >> 1;
    if (__ldg(a.cu_tokens + mid) <= token) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Place of this lane's token: sequence, position, block and the tokens that follow it there.  Called by all lanes.
__device__ __forceinline__ TokenPlace place_token(const AppendArgs &a, uint32_t token, bool mine, uint32_t lane) {
  TokenPlace t{};
  uint32_t seq = token, begin = token, end = token + 1;
  if (a.cu_tokens != nullptr) seq = find_sequence(a, token, lane);
  if (!mine || token >= a.num_tokens || seq >= a.num_seqs) return t;
  if (a.cu_tokens != nullptr) {
    begin = __ldg(a.cu_tokens + seq);
    end = min(__ldg(a.cu_tokens + seq + 1), a.num_tokens);
  }
  const int64_t position = static_cast<int64_t>(__ldg(a.context_lens + seq)) - (end - token);
  if (position < 0 || static_cast<uint64_t>(position) >= a.position_limit) return t;
  t.position = static_cast<uint32_t>(position);
  t.block = __ldg(a.block_tables + static_cast<size_t>(seq) * a.max_blocks_per_seq + (t.position >> a.block_shift));
  if (t.block >= a.num_blocks) return t;
  const uint32_t row = t.position & (a.block_size - 1u);
  t.leads = row == 0 || token == begin;
  const uint64_t room = min(static_cast<uint64_t>(a.block_size - row), a.position_limit - t.position);
  t.rows_here = static_cast<uint32_t>(min(room, static_cast<uint64_t>(end - token)));
  t.valid = true;
  return t;
}

constexpr uint32_t kAppendThreads = 256;
constexpr uint32_t kAppendWarps = kAppendThreads / 32;
constexpr uint32_t kQueryBatch = 4; // query rows that a thread requests together

// What a lane does of every row group: the lanes of a warp hold rows_per_pass rows side by side, 16 elements
// each (see rotary_item).
struct LaneShare {
  uint32_t item, row, rows_per_pass;
  bool active;
  __device__ __forceinline__ LaneShare(uint32_t head_size, uint32_t lane) {
    const uint32_t lanes_per_row = head_size / 16u;
    rows_per_pass = 32u / lanes_per_row;
    item = lane % lanes_per_row;
    row = lane / lanes_per_row;
    active = row < rows_per_pass;
  }
};

// An item of a row that is not rotated: eight elements of each half, so that the lanes of a row make one run of
// addresses with every piece (16 elements in a row would touch half of every 32-byte sector, twice).
__device__ __forceinline__ RotaryItem plain_item(uint32_t item, uint32_t head_size) {
  return RotaryItem{item * 8u, head_size / 2u + item * 8u, false};
}

// What one warp does for K or V of one (block, head): some of its new rows.
struct RowJob {
  const __half *src;   // the warp's first row
  uint64_t stride;     // elements between two rows
  const float *angles; // rotation table row of that row; null: not rotated
  uint8_t *dst;        // where that row goes
  uint8_t *block_rows; // row 0 of the head in the block
  float *scale_at;
  size_t pitch;        // bytes between two rows of the block
  uint32_t rows;
  uint32_t first_row;  // of the block, the first new one: those before it are held
  uint32_t rotary_dim;
  float held;          // scale so far
  bool live;           // false: nothing to do, but the other warps of the CTA may wait for this one
  bool is_v;
  bool in_stage;       // the rows fit the warp's stage of shared memory
};

// The general way, row by row from memory: rows with infinities or NaNs (an infinity counts as the largest fp16
// value, so that it does not take the block's scale; NaNs drop out of fmaxf), and more rows than a warp's corner of
// shared memory holds.
template <bool INTERLEAVED>
__device__ __forceinline__ void load_row_with_care(const RowJob &job, const LaneShare &l, const RotaryItem &rot, uint32_t r,
                                                   float (&x)[8], float (&y)[8]) {
  const __half *row = job.src + static_cast<size_t>(r) * job.stride;
  unpack_half8(__ldg(reinterpret_cast<const uint4 *>(row + rot.first)), x);
  unpack_half8(__ldg(reinterpret_cast<const uint4 *>(row + rot.second)), y);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (isinf(x[j])) x[j] = copysignf(65504.f, x[j]);
    if (isinf(y[j])) y[j] = copysignf(65504.f, y[j]);
  }
  if (rot.rotated) {
    float c[8], s[8];
    load_cos_sin(job.angles + static_cast<size_t>(r) * job.rotary_dim, l.item, job.rotary_dim, c, s);
    rotate_item(x, y, c, s, INTERLEAVED);
  }
}

template <bool INTERLEAVED>
__device__ __forceinline__ float largest_with_care(const RowJob &job, const LaneShare &l, const RotaryItem &rot) {
  float top = 0.f;
#pragma unroll 1
  for (uint32_t r = l.row; l.active && r < job.rows; r += l.rows_per_pass) {
    float x[8], y[8];
    load_row_with_care<INTERLEAVED>(job, l, rot, r, x, y);
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, fmaxf(fabsf(x[j]), fabsf(y[j])));
  }
  return top;
}

template <int KV, bool INTERLEAVED>
__device__ __forceinline__ void store_with_care(const RowJob &job, const LaneShare &l, const RotaryItem &rot, float scale) {
  const Divider by(scale);
#pragma unroll 1
  for (uint32_t r = l.row; l.active && r < job.rows; r += l.rows_per_pass) {
    float x[8], y[8];
    load_row_with_care<INTERLEAVED>(job, l, rot, r, x, y);
    divide8(x, by);
    divide8(y, by);
    uint8_t *row = job.dst + r * job.pitch;
    *reinterpret_cast<uint2 *>(row + rot.first) =
        make_uint2(pack_codes<KV>(x[0], x[1], x[2], x[3]), pack_codes<KV>(x[4], x[5], x[6], x[7]));
    *reinterpret_cast<uint2 *>(row + rot.second) =
        make_uint2(pack_codes<KV>(y[0], y[1], y[2], y[3]), pack_codes<KV>(y[4], y[5], y[6], y[7]));
  }
}

// Rows that a block held before, under its new scale; 16 codes of every row for this lane.
template <int KV>
__device__ __forceinline__ void requantise_rows(uint8_t *at, size_t step, uint32_t rows, float held, float scale) {
#pragma unroll 1
  for (uint32_t r = 0; r < rows; ++r, at += step) {
    uint4 v = *reinterpret_cast<uint4 *>(at);
    uint32_t *w = reinterpret_cast<uint32_t *>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float c[4];
      unpack_codes<KV>(w[i], c);
#pragma unroll
      for (int j = 0; j < 4; ++j) c[j] = __fdiv_rn(__fmul_rn(c[j], held), scale);
      w[i] = pack_codes<KV>(c[0], c[1], c[2], c[3]);
    }
    *reinterpret_cast<uint4 *>(at) = v;
  }
}

__device__ __forceinline__ float max_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ void copy_async_16(uint32_t dst_smem, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst_smem), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { // all groups but the N newest have landed
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 load_shared_16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

template <int PASSES>
constexpr uint32_t kStageBytes = PASSES * 2 * 32 * 16; // one job's rows of a warp

// The usual way: up to PASSES row groups of the warp are copied to its own corner of shared memory while the job before
// is worked on, and are gone through there twice, for the maximum and for the codes.  (K is rotated both times: the
// rotated rows as fp32 in registers cost the SM a third of its warps.)  Every lane reads back what it copied itself, so
// nothing but its own copies has to be waited for.  The maximum of V is taken two fp16 values at a time.  The
// maxima propagate NaNs, so an infinity or a NaN among the inputs shows in the result.  A lane without a row of its
// own in a group takes the last row over again: it changes no maximum and is not stored.
// Measured on 37 364 prompt tokens (8 KV heads of 128, e4m3, rotated): rows in registers, read when their job comes,
// 79 us; with the copies ahead, pairs of values per instruction and whole runs of addresses per piece 72 us (51 us
// without the rotation, whose angles come from the L1 cache twice for every head; 38 us is what the bytes take).
// Layout: [row group][piece][lane], 16 bytes each.
template <int PASSES, bool ROTATE, bool INTERLEAVED>
struct HeldRows {
  const RowJob &job;
  const LaneShare &l;
  const RotaryItem &rot;
  uint32_t at; // this lane's 16 bytes of row group 0, piece 0

  __device__ __forceinline__ void values(int i, Item2 &v) const {
    unpack_item(load_shared_16(at + i * 1024u), load_shared_16(at + i * 1024u + 512u), v);
    if constexpr (ROTATE) {
      if (rot.rotated) {
        const float *angles = job.angles + min(l.row + i * l.rows_per_pass, job.rows - 1u) * job.rotary_dim + l.item * 8u;
        rotate_item2(v, angles, angles + job.rotary_dim / 2u, INTERLEAVED);
      }
    }
  }

  __device__ __forceinline__ float largest() const {
    if constexpr (ROTATE) {
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < PASSES; ++i) {
        Item2 v;
        values(i, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          top = max_or_nan(top, max_or_nan(fabsf(v.x[j].x), fabsf(v.x[j].y)));
          top = max_or_nan(top, max_or_nan(fabsf(v.y[j].x), fabsf(v.y[j].y)));
        }
      }
      return top;
    } else {
      __half2 top = __half2half2(__ushort_as_half(0));
#pragma unroll
      for (int i = 0; i < 2 * PASSES; ++i) {
        const uint4 raw = load_shared_16(at + i * 512u);
        const __half2 *h = reinterpret_cast<const __half2 *>(&raw);
#pragma unroll
        for (int j = 0; j < 4; ++j) top = __hmax2_nan(top, __habs2(h[j]));
      }
      const float2 t = __half22float2(top);
      return max_or_nan(t.x, t.y);
    }
  }

  template <int KV>
  __device__ __forceinline__ void store(float scale) const {
    const Divider by(scale); // the caller has made sure of its range
    const float2 minus_s = make_float2(-by.s, -by.s), r = make_float2(by.r, by.r);
    const uint32_t distance = rot.second - rot.first;
    uint8_t *to = job.dst + l.row * job.pitch + rot.first;
    const size_t step = l.rows_per_pass * job.pitch;
#pragma unroll
    for (int i = 0; i < PASSES; ++i, to += step) {
      Item2 v;
      values(i, v);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v.x[j] = divide2(v.x[j], minus_s, r);
        v.y[j] = divide2(v.y[j], minus_s, r);
      }
      if (l.active && l.row + i * l.rows_per_pass < job.rows) {
        *reinterpret_cast<uint2 *>(to) = make_uint2(pack_small_codes<KV>(v.x[0].x, v.x[0].y, v.x[1].x, v.x[1].y),
                                                    pack_small_codes<KV>(v.x[2].x, v.x[2].y, v.x[3].x, v.x[3].y));
        *reinterpret_cast<uint2 *>(to + distance) = make_uint2(pack_small_codes<KV>(v.y[0].x, v.y[0].y, v.y[1].x, v.y[1].y),
                                                               pack_small_codes<KV>(v.y[2].x, v.y[2].y, v.y[3].x, v.y[3].y));
      }
    }
  }
};

// Starts the copies of a job's rows; the table rows of their angles are called into the L1 cache.
template <int PASSES>
__device__ __forceinline__ void fetch_rows(const RowJob &job, const LaneShare &l, const RotaryItem &rot, uint32_t at) {
  if (job.in_stage) {
    const uint8_t *src = reinterpret_cast<const uint8_t *>(job.src + rot.first);
    const uint32_t distance = (rot.second - rot.first) * 2u;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const uint32_t r = min(l.row + i * l.rows_per_pass, job.rows - 1u);
      const uint8_t *row = src + r * (job.stride * 2u);
      copy_async_16(at + i * 1024u, row);
      copy_async_16(at + i * 1024u + 512u, row + distance);
      if (rot.rotated) {
        const float *angles = job.angles + r * job.rotary_dim + l.item * 8u;
        asm volatile("prefetch.global.L1 [%0];" ::"l"(angles));
        asm volatile("prefetch.global.L1 [%0];" ::"l"(angles + job.rotary_dim / 2u));
      }
    }
  }
  copies_commit();
}

// Largest magnitude among a job's rows of this warp, in all lanes; `careful` if infinities or NaNs or their number call
// for the general way.
template <bool INTERLEAVED, int PASSES, bool ROTATE>
__device__ __forceinline__ float largest_of_rows(const RowJob &job, const LaneShare &l, const RotaryItem &rot, uint32_t at,
                                                 bool &careful) {
  careful = true;
  float top = 0.f;
  if (job.in_stage) {
    top = HeldRows<PASSES, ROTATE, INTERLEAVED>{job, l, rot, at}.largest();
    careful = __any_sync(0xffffffffu, !(top <= 1e30f)) != 0;
  }
  if (careful && job.live) top = largest_with_care<INTERLEAVED>(job, l, rot);
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top))); // magnitudes order like their bits
}

// The rest of a live job, once `top`, the largest magnitude among the rows of all its `parts` warps, is known: new
// codes by this one, number `part`, and its share of the held rows.
template <int KV, bool INTERLEAVED, int PASSES, bool ROTATE>
__device__ __forceinline__ void store_rows(const RowJob &job, const LaneShare &l, const RotaryItem &rot, uint32_t at,
                                           bool careful, float top, uint32_t part, uint32_t parts, uint32_t lane) {
  const float grown = fmaxf(job.held, __fdiv_rn(top, largest_code<KV>()));
  const float scale = (grown > 0.f) ? grown : 1.f; // a block of zeros keeps scale 0 and codes 0
  if (!careful && !Divider(scale).plain) HeldRows<PASSES, ROTATE, INTERLEAVED>{job, l, rot, at}.template store<KV>(scale);
  else store_with_care<KV, INTERLEAVED>(job, l, rot, scale);
  if (grown > job.held && l.active) {
    const uint32_t r = part * l.rows_per_pass + l.row, step = parts * l.rows_per_pass;
    if (r < job.first_row)
      requantise_rows<KV>(job.block_rows + r * job.pitch + l.item * 16u, step * job.pitch,
                          divide_round_up(job.first_row - r, step), job.held, scale);
  }
  // every lane of the job's warps has read the old scale: this warp's before its copies were waited for, the others'
  // before the barrier between the two functions
  if (lane == 0 && part == 0u) *job.scale_at = grown;
}

// A column of CTAs (blockIdx.x) owns tokens_per_cta consecutive new tokens: it appends the blocks whose first new
// token is among them (a block belongs to exactly one column whatever its later tokens) and rotates the tokens'
// queries.  The jobs of a block (K and V of each head) go round the warps of the first append_ctas CTAs of the
// column, parts warps to a job; the other CTAs take the queries.  Every warp works out the places of the tokens
// for itself, a token per lane.
template <int KV, bool INTERLEAVED, int PASSES>
__global__ void __launch_bounds__(kAppendThreads, 3) append_block_scaled_kernel(const AppendArgs a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  extern __shared__ __align__(16) uint8_t stages[]; // [warp][2][kStageBytes]
  __shared__ float tops[2][kAppendWarps];
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
  const uint32_t token0 = blockIdx.x * a.tokens_per_cta;
  const TokenPlace mine = place_token(a, token0 + lane, lane < a.tokens_per_cta, lane);
  const uint32_t D = a.head_size;
  if (blockIdx.y < a.append_ctas) {
    const uint32_t heads = a.num_kv_heads;
    const LaneShare lane_share(D, lane);
    const RotaryItem rot_k = a.rotary_dim != 0u ? rotary_item(lane_share.item, a.rotary_dim, INTERLEAVED)
                                                : plain_item(lane_share.item, D);
    const RotaryItem rot_v = plain_item(lane_share.item, D);
    const uint32_t parts = a.warps_per_job, part = warp % parts;
    const uint32_t jobs_at_once = kAppendWarps / parts;
    const uint32_t own_stage = smem_u32(stages) + warp * 2u * kStageBytes<PASSES> + lane * 16u;
    const uint32_t j_first = blockIdx.y * jobs_at_once + warp / parts, j_step = a.append_ctas * jobs_at_once;
    const uint32_t rounds = divide_round_up(2u * heads, j_step); // of every block: the same for all warps

    // the jobs of this warp, block after block
    uint32_t leaders = __ballot_sync(0xffffffffu, mine.valid && mine.leads);
    uint32_t left = 0, j = 0, position = 0, block = 0, new_rows = 0;
    size_t token = 0;
    auto next_job = [&](RowJob &job) -> bool {
      if (left == 0u) {
        if (leaders == 0u) return false;
        const uint32_t src = __ffs(leaders) - 1u;
        leaders &= leaders - 1u;
        position = __shfl_sync(0xffffffffu, mine.position, src);
        block = __shfl_sync(0xffffffffu, mine.block, src);
        new_rows = __shfl_sync(0xffffffffu, mine.rows_here, src);
        token = token0 + src;
        left = rounds;
        j = j_first;
      }
      // a job's rows go to its warps in runs of whole row groups
      const uint32_t run = divide_round_up(divide_round_up(new_rows, parts), lane_share.rows_per_pass) * lane_share.rows_per_pass;
      const uint32_t run0 = min(new_rows, part * run);
      job.live = j < 2u * heads; // the others have nothing to do, but the CTA's warps may wait for them
      job.is_v = job.live && j >= heads;
      const uint32_t head = !job.live ? 0u : job.is_v ? j - heads : j;
      job.rows = min(new_rows - run0, run);
      job.in_stage = job.live && job.rows != 0u && job.rows <= PASSES * lane_share.rows_per_pass;
      job.first_row = position & (a.block_size - 1u);
      job.pitch = static_cast<size_t>(heads) * D;
      job.rotary_dim = a.rotary_dim;
      job.stride = job.is_v ? a.value_stride : a.key_stride;
      job.src = (job.is_v ? a.value : a.key) + (token + run0) * job.stride + static_cast<size_t>(head) * D;
      job.block_rows = static_cast<uint8_t *>(job.is_v ? a.value_cache : a.key_cache) +
                       (static_cast<size_t>(block) * a.block_size * heads + head) * D;
      job.dst = job.block_rows + (job.first_row + run0) * job.pitch;
      job.scale_at = (job.is_v ? a.v_scales : a.k_scales) + static_cast<size_t>(block) * heads + head;
      job.angles = (job.is_v || a.rotary_dim == 0u) ? nullptr : a.cos_sin + static_cast<size_t>(position + run0) * a.rotary_dim;
      job.held = (job.live && job.first_row != 0u) ? *job.scale_at : 0.f;
      j += j_step;
      --left;
      return true;
    };

    uint32_t round = 0;
    RowJob next;
    bool more = next_job(next);
    if (more) fetch_rows<PASSES>(next, lane_share, next.is_v ? rot_v : rot_k, own_stage);
    while (more) {
      const RowJob job = next;
      const uint32_t at = own_stage + (round & 1u) * kStageBytes<PASSES>;
      more = next_job(next);
      if (more) {
        fetch_rows<PASSES>(next, lane_share, next.is_v ? rot_v : rot_k, own_stage + ((round + 1u) & 1u) * kStageBytes<PASSES>);
        copies_wait<1>();
      } else {
        copies_wait<0>();
      }
      const bool rotated = job.angles != nullptr;
      bool careful;
      float top = rotated ? largest_of_rows<INTERLEAVED, PASSES, true>(job, lane_share, rot_k, at, careful)
                          : largest_of_rows<INTERLEAVED, PASSES, false>(job, lane_share, rot_v, at, careful);
      if (parts > 1u) {
        // The largest value of the job's warps.  Warps with K and with V jobs, or with none, meet at this one barrier: all
        // warps of the CTA make the same number of rounds.  Two rows of the table in turn: a warp may be a round ahead
        // of another.
        float *const row = tops[round & 1u];
        if (lane == 0) row[warp] = top;
        __syncthreads();
        for (uint32_t k = 0; k < parts; ++k) top = fmaxf(top, row[warp - part + k]);
      }
      if (job.live) {
        if (rotated) store_rows<KV, INTERLEAVED, PASSES, true>(job, lane_share, rot_k, at, careful, top, part, parts, lane);
        else store_rows<KV, INTERLEAVED, PASSES, false>(job, lane_share, rot_v, at, careful, top, part, parts, lane);
      }
      ++round;
    }
    return;
  }

  // queries: (token, head) pairs go round groups of head_size / 16 lanes
  const uint32_t lanes_per_head = D / 16u;
  const uint32_t pairs_at_once = kAppendThreads / lanes_per_head;
  const uint32_t item = threadIdx.x % lanes_per_head, pair0 = threadIdx.x / lanes_per_head;
  const RotaryItem rot = rotary_item(item, a.rotary_dim, INTERLEAVED);
  const uint32_t pairs = a.tokens_per_cta * a.num_heads;
  const uint32_t step = (gridDim.y - a.append_ctas) * pairs_at_once;
  // the same trips for all lanes: they shuffle
  for (uint32_t p0 = (blockIdx.y - a.append_ctas) * pairs_at_once; p0 < pairs; p0 += kQueryBatch * step) {
    uint4 raw[kQueryBatch][2];
    uint32_t position[kQueryBatch];
    size_t row[kQueryBatch]; // token * num_heads + head
    bool take[kQueryBatch];
#pragma unroll
    for (uint32_t k = 0; k < kQueryBatch; ++k) {
      const uint32_t pair = p0 + k * step + pair0;
      const uint32_t t = pair / a.num_heads, head = pair - t * a.num_heads;
      position[k] = __shfl_sync(0xffffffffu, mine.position, t & 31u);
      take[k] = __shfl_sync(0xffffffffu, mine.valid ? 1 : 0, t & 31u) != 0 && pair0 < pairs_at_once && pair < pairs;
      row[k] = static_cast<size_t>(token0 + t) * a.num_heads + head;
      if (take[k]) {
        const __half *src = a.query + static_cast<size_t>(token0 + t) * a.query_stride + static_cast<size_t>(head) * D;
        raw[k][0] = __ldg(reinterpret_cast<const uint4 *>(src + rot.first));
        raw[k][1] = __ldg(reinterpret_cast<const uint4 *>(src + rot.second));
      }
    }
#pragma unroll
    for (uint32_t k = 0; k < kQueryBatch; ++k) {
      if (!take[k]) continue;
      Item2 v;
      unpack_item(raw[k][0], raw[k][1], v);
      if (rot.rotated) {
        const float *angles = a.cos_sin + static_cast<size_t>(position[k]) * a.rotary_dim + item * 8u;
        rotate_item2(v, angles, angles + a.rotary_dim / 2u, INTERLEAVED);
      }
      __half *dst = a.query_out + row[k] * D;
      *reinterpret_cast<uint4 *>(dst + rot.first) = make_uint4(pack_half2(v.x[0].x, v.x[0].y), pack_half2(v.x[1].x, v.x[1].y),
                                                               pack_half2(v.x[2].x, v.x[2].y), pack_half2(v.x[3].x, v.x[3].y));
      *reinterpret_cast<uint4 *>(dst + rot.second) = make_uint4(pack_half2(v.y[0].x, v.y[0].y), pack_half2(v.y[1].x, v.y[1].y),
                                                                pack_half2(v.y[2].x, v.y[2].y), pack_half2(v.y[3].x, v.y[3].y));
    }
  }
}

template <int KV, int PASSES>
int launch_append(const AppendArgs &a, uint32_t query_ctas, bool interleaved, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(divide_round_up(a.num_tokens, a.tokens_per_cta), a.append_ctas + query_ctas, 1);
  cfg.blockDim = dim3(kAppendThreads, 1, 1);
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.dynamicSmemBytes = kAppendWarps * 2u * kStageBytes<PASSES>;
  auto kernel = interleaved ? append_block_scaled_kernel<KV, true, PASSES> : append_block_scaled_kernel<KV, false, PASSES>;
  static thread_local int configured_device[2] = {-1, -1};
  int device = 0;
  PA_CUDA_TRY(cudaGetDevice(&device));
  if (configured_device[interleaved ? 1 : 0] != device) {
    PA_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(cfg.dynamicSmemBytes)));
    configured_device[interleaved ? 1 : 0] = device;
  }
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
  // On prompts a CTA takes 32 tokens (two blocks of 16), so that finding their places is paid for once; on decode
  // steps one, and in between as many as a sequence has on average.
  const uint32_t average = p->cu_tokens != nullptr ? std::max(1u, p->num_tokens / p->num_seqs) : 1u;
  uint32_t per_cta = 1;
  while (per_cta < 32u && per_cta * 2u <= average) per_cta *= 2u;
  a.tokens_per_cta = per_cta;
  // A few new rows per block (decode steps): one group of rows per warp, and twice the CTAs on an SM.  Otherwise four
  // groups, and as many warps to a job as hold a block's new rows in shared memory.  (By the average: where many decode
  // tokens come with a prompt chunk, the chunk's rows take the general way, right but slow: 255 tokens and a chunk
  // of 2048, int8, 8 KV heads of 128, 24 us instead of the 9 that the chunk takes alone.)
  const uint32_t rows = std::min(p->block_size, average);
  const uint32_t rows_per_pass = 32u / (p->head_size / 16u);
  const bool few = rows <= rows_per_pass;
  uint32_t parts = 1;
  while (parts < kAppendWarps && parts * (few ? 1u : 4u) * rows_per_pass < rows) parts *= 2u;
  a.warps_per_job = parts;
  // CTAs in a column: enough to fill the 444 places of the GPU twice or so, no more than there is work for.  (9 163
  // tokens of 37 sequences, 8 KV heads of 64, blocks of 64: without queries 19.2 us with 4 CTAs, 24 with 2; with 40
  // query heads 34.8 us with 2 + 3, 36.8 with 4 + 3, 40 with 4 + 1, 38 with 4 + 6.)
  const uint32_t columns = divide_round_up(p->num_tokens, per_cta);
  auto ctas = [&](uint32_t aimed_at, uint32_t useful) { return std::min(std::max(1u, aimed_at / columns), useful); };
  a.append_ctas = ctas(p->query != nullptr ? 592u : 1184u, divide_round_up(2u * p->num_kv_heads * parts, kAppendWarps));
  uint32_t query_ctas = 0;
  if (p->query != nullptr)
    query_ctas = ctas(888u, divide_round_up(per_cta * p->num_heads * (p->head_size / 16u), kQueryBatch * kAppendThreads));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool interleaved = p->interleaved != 0u;
  auto launch = [&](auto few_rows, auto many_rows) {
    return few ? few_rows(a, query_ctas, interleaved, s) : many_rows(a, query_ctas, interleaved, s);
  };
  if (p->kv_dtype == PA_KV_INT8) return launch(launch_append<KV_I8, 1>, launch_append<KV_I8, 4>);
  if (p->kv_dtype == PA_KV_FP8_E4M3) return launch(launch_append<KV_E4M3, 1>, launch_append<KV_E4M3, 4>);
  return launch(launch_append<KV_E5M2, 1>, launch_append<KV_E5M2, 4>);
}
