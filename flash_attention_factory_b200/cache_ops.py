"""Writing new tokens into the paged KV cache (the step before decode attention).

`reshape_and_cache` scatters this step's K/V rows into the cache the attention operators read
([num_blocks, block_size, num_kv_heads, head_size]) and casts them to the cache type on the
way.  The reference builds its caches on the host with torch casts
(test_paged_fp8cache.py:180-203); this is the device-side counterpart of that fixture code.

`rope_and_cache` does the same with the rotary position embedding applied to K, and to the
step's queries, in the same launch.  `append_block_scaled` appends to an 8-bit cache that keeps a scale
for each block of tokens and KV head, and keeps those scales.
"""
from __future__ import annotations

import ctypes

import torch

from . import _cabi, _launch

_F16, _F32, _I64 = torch.float16, torch.float32, torch.int64


def _kv_dtype(cache: torch.Tensor) -> int:
    if cache.dtype == torch.float16:
        return _cabi.KV_F16
    if cache.dtype == torch.float8_e4m3fn:
        return _cabi.KV_FP8_E4M3
    if cache.dtype in (torch.float8_e5m2, torch.uint8):
        return _cabi.KV_FP8_E5M2
    if cache.dtype == torch.int8:
        return _cabi.KV_INT8
    raise RuntimeError(f"unsupported cache dtype {cache.dtype}")


def _set_scales(p, num_blocks: int, kv_heads: int, index: int, k_scale_per_head, v_scale_per_head, k_scale_per_block,
                v_scale_per_block) -> None:
    """Fills the scale arrays of a cache-write argument block from those that are given."""
    if k_scale_per_head is not None:
        p.k_scale_per_head = _scale_pointer(k_scale_per_head, "k_scale_per_head", (kv_heads,), index)
    if v_scale_per_head is not None:
        p.v_scale_per_head = _scale_pointer(v_scale_per_head, "v_scale_per_head", (kv_heads,), index)
    if k_scale_per_block is not None:
        p.k_scale_per_block = _scale_pointer(k_scale_per_block, "k_scale_per_block", (num_blocks, kv_heads), index)
    if v_scale_per_block is not None:
        p.v_scale_per_block = _scale_pointer(v_scale_per_block, "v_scale_per_block", (num_blocks, kv_heads), index)


def _scale_pointer(t: torch.Tensor, name: str, shape, index: int) -> int:
    if t.dtype is not _F32 or t.shape != shape or t.get_device() != index or not t.is_contiguous():
        raise RuntimeError(f"{name} must be a contiguous float32 tensor of shape {shape} on the cache's device")
    return t.data_ptr()


def reshape_and_cache(key: torch.Tensor, value: torch.Tensor, key_cache: torch.Tensor,
                      value_cache: torch.Tensor, slot_mapping: torch.Tensor, fp8_scale: float = 1.0, *,
                      k_scale_per_head=None, v_scale_per_head=None,
                      k_scale_per_block=None, v_scale_per_block=None) -> None:
    """key/value fp16 [T, HK, D] -> caches at slot_mapping[t] = block_id * block_size + row.

    Negative slots are skipped.  FP8 and int8 caches store round-to-nearest-even(x / scale),
    saturating (int8: to -127 .. 127), where scale is `fp8_scale` or, when given, the entry of the token's KV head
    in `k_scale_per_head` / `v_scale_per_head` (float32 [HK]) or of its block and KV head in
    `k_scale_per_block` / `v_scale_per_block` (float32 [num_blocks, HK]); the attention
    operators take the same scale arguments.  Asynchronous on torch's current stream.
    """
    if not key.is_cuda:
        raise RuntimeError("reshape_and_cache needs CUDA tensors (no CPU fallback exists)")
    for t in (key, value, key_cache, value_cache, slot_mapping):
        if not t.is_contiguous() or t.device != key.device:
            raise RuntimeError("all tensors must be contiguous and on the same device")
    if key.dtype != torch.float16 or value.dtype != torch.float16 or key.shape != value.shape:
        raise RuntimeError("key and value must be float16 tensors of the same shape")
    if slot_mapping.dtype != torch.int64 or slot_mapping.numel() != key.size(0):
        raise RuntimeError("slot_mapping must be int64 with one entry per token")
    if key_cache.shape != value_cache.shape or key_cache.dtype != value_cache.dtype:
        raise RuntimeError("key_cache and value_cache must match")
    if key_cache.dim() != 4 or tuple(key_cache.shape[2:]) != tuple(key.shape[1:]):
        raise RuntimeError("cache must be [num_blocks, block_size, num_kv_heads, head_size]")
    p = _cabi.PaCacheWriteParams()
    p.key, p.value = key.data_ptr(), value.data_ptr()
    p.key_cache, p.value_cache = key_cache.data_ptr(), value_cache.data_ptr()
    p.slot_mapping = slot_mapping.data_ptr()
    p.num_tokens, p.num_kv_heads, p.head_size = key.size(0), key.size(1), key.size(2)
    p.block_size, p.num_blocks = key_cache.size(1), key_cache.size(0)
    p.fp8_scale = float(fp8_scale)
    p.kv_dtype = _kv_dtype(key_cache)
    _set_scales(p, key_cache.size(0), key.size(1), key.get_device(), k_scale_per_head, v_scale_per_head,
                k_scale_per_block, v_scale_per_block)
    lib = _cabi.load_library()
    with torch.cuda.device(key.device):
        stream = torch.cuda.current_stream(key.device).cuda_stream
        _cabi.check(lib.pa_reshape_and_cache(ctypes.byref(p), ctypes.c_void_p(stream)))


def _token_rows(t: torch.Tensor, shape, name: str, index: int) -> int:
    """Checks fp16 rows [T, heads, D] whose tokens may lie any stride apart (slices of one projection's
    output); returns that stride in elements."""
    if t.dtype is not _F16 or len(shape) != 3 or t.get_device() != index:
        raise RuntimeError(f"{name} must be a float16 tensor [tokens, heads, head_size] on the cache's device")
    tokens, heads, d = shape
    stride, head_stride, last = t.stride()
    if last != 1 or (head_stride != d and heads != 1):
        raise RuntimeError(f"the heads of a token of {name} must be contiguous")
    if tokens <= 1:
        return heads * d
    if stride % 8 != 0 or stride < 0:
        raise RuntimeError(f"the token stride of {name} must be a multiple of 8 elements")
    return stride


def _check_caches(rows, value, key_cache, value_cache, shape) -> int:
    """Checks the caches (of `shape`) against the rows of key and value; returns the device index."""
    index = key_cache.get_device()
    if index < 0 or value_cache.get_device() != index or not (key_cache.is_contiguous() and value_cache.is_contiguous()):
        raise RuntimeError("the caches must be contiguous CUDA tensors on one device (no CPU fallback exists)")
    if len(shape) != 4 or shape != value_cache.shape or key_cache.dtype is not value_cache.dtype:
        raise RuntimeError("key_cache and value_cache must match")
    if len(rows) != 3 or rows != value.shape or rows[1] != shape[2] or rows[2] != shape[3]:
        raise RuntimeError("cache must be [num_blocks, block_size, num_kv_heads, head_size]")
    return index


def _check_rotation(cos_sin, index: int) -> None:
    if (cos_sin.dtype is not _F32 or cos_sin.dim() != 2 or not cos_sin.is_contiguous()
            or cos_sin.get_device() != index):
        raise RuntimeError("cos_sin must be a contiguous float32 tensor [max_position, rotary_dim] on the cache's device")


def _check_queries(p, query, query_out, rows, index: int) -> None:
    """Fills the query part of an argument block."""
    if query is None and query_out is None:
        return
    if query is None or query_out is None:
        raise RuntimeError("query and query_out must be given together")
    shape = query.shape
    p.query_token_stride = _token_rows(query, shape, "query", index)
    if shape[0] != rows[0] or shape[2] != rows[2]:
        raise RuntimeError("query and key must have the same tokens and head_size")
    if (query_out.shape != shape or query_out.dtype is not _F16 or not query_out.is_contiguous()
            or query_out.get_device() != index):
        raise RuntimeError("query_out must be a contiguous float16 tensor of query's shape")
    p.num_heads, p.query, p.query_out = shape[1], query.data_ptr(), query_out.data_ptr()


def rope_and_cache(query, key: torch.Tensor, value: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor,
                   query_out, key_cache: torch.Tensor, value_cache: torch.Tensor, slot_mapping: torch.Tensor,
                   fp8_scale: float = 1.0, *, interleaved: bool = False, k_scale_per_head=None, v_scale_per_head=None,
                   k_scale_per_block=None, v_scale_per_block=None) -> None:
    """`reshape_and_cache` with the rotary position embedding applied to K and to the step's queries.

    query fp16 [T, H, D] and key / value fp16 [T, HK, D] may be slices of one projection's output (the
    heads of a token contiguous, tokens any multiple of 8 elements apart); query and query_out
    (contiguous, or query itself if that is contiguous) may both be None.  positions int64 [T];
    cos_sin float32 [max_position, R]: R / 2 cosines, then the sines, of a position's angles; the first R
    dims of a head (a multiple of 16) are rotated, as pairs (i, i + R / 2), or (2 i, 2 i + 1) with
    `interleaved`.  The rotation runs in fp32 and is rounded once, to fp16 or to the cache's code.

    Slots, cache types and scales are those of `reshape_and_cache`.  A token with a negative slot (padding),
    or whose slot or position is out of range, is skipped: its cache and query_out rows stay as they
    were.  Asynchronous on torch's current stream.
    """
    shape, rows = key_cache.shape, key.shape
    index = _check_caches(rows, value, key_cache, value_cache, shape)
    p = _cabi.PaRopeCacheParams()
    p.key_token_stride = _token_rows(key, rows, "key", index)
    p.value_token_stride = _token_rows(value, rows, "value", index)
    num_blocks, block_size, kv_heads, head_size = shape
    tokens = rows[0]
    for x in (slot_mapping, positions):
        if x.dtype is not _I64 or x.numel() != tokens or not x.is_contiguous() or x.get_device() != index:
            raise RuntimeError("slot_mapping and positions must be int64 with one entry per token on the cache's device")
    _check_rotation(cos_sin, index)
    _check_queries(p, query, query_out, rows, index)
    c = p.cache
    c.key, c.value = key.data_ptr(), value.data_ptr()
    c.key_cache, c.value_cache = key_cache.data_ptr(), value_cache.data_ptr()
    c.slot_mapping = slot_mapping.data_ptr()
    c.num_tokens, c.num_kv_heads, c.head_size = tokens, kv_heads, head_size
    c.block_size, c.num_blocks = block_size, num_blocks
    c.fp8_scale, c.kv_dtype = float(fp8_scale), _kv_dtype(key_cache)
    if not (k_scale_per_head is v_scale_per_head is k_scale_per_block is v_scale_per_block is None):
        _set_scales(c, num_blocks, kv_heads, index, k_scale_per_head, v_scale_per_head, k_scale_per_block, v_scale_per_block)
    p.positions, p.cos_sin = positions.data_ptr(), cos_sin.data_ptr()
    p.max_position, p.rotary_dim = cos_sin.shape
    p.interleaved = int(interleaved)
    _launch.call(_cabi.load_library().pa_rope_and_cache, p, index)


def append_block_scaled(key: torch.Tensor, value: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                        k_scale_per_block: torch.Tensor, v_scale_per_block: torch.Tensor, block_tables: torch.Tensor,
                        context_lens: torch.Tensor, *, cu_tokens=None, query=None, query_out=None, cos_sin=None,
                        interleaved: bool = False) -> None:
    """Appends new tokens to an int8 or FP8 cache with one scale per block of tokens and KV head.

    Sequence i's new tokens are rows cu_tokens[i] .. cu_tokens[i + 1] - 1 of key / value fp16 [T, HK, D]
    (int32 [S + 1]; None: one token per sequence) and take its positions context_lens[i] - n ..
    context_lens[i] - 1: context_lens [S] already counts them, as the attention call that follows reads it.
    k_scale_per_block / v_scale_per_block (float32 [num_blocks, HK]) are read and written: a block's scale
    grows to max|row| / q of its new rows where that is more (q = 127, 448 or 57344 for int8, e4m3, e5m2), the
    rows held before are then stored again under the new scale, and a block whose first row is new starts
    afresh.  A block of zeros has scale 0.  Infinities count as the largest fp16 value, NaNs do not count.

    With `cos_sin` (see `rope_and_cache`) K is rotated by its position on the way, and query -> query_out too
    if given.  The blocks a call writes must belong to one sequence each (full blocks may be shared).  Rows
    behind the last sequence, and tokens whose position lies outside the table row or the rotation table, are
    skipped.  Asynchronous on torch's current stream.
    """
    shape, rows = key_cache.shape, key.shape
    index = _check_caches(rows, value, key_cache, value_cache, shape)
    p = _cabi.PaBlockScaledParams()
    p.key_token_stride = _token_rows(key, rows, "key", index)
    p.value_token_stride = _token_rows(value, rows, "value", index)
    num_blocks, block_size, kv_heads, head_size = shape
    for t in (k_scale_per_block, v_scale_per_block):
        if (t.dtype is not _F32 or t.shape != (num_blocks, kv_heads) or not t.is_contiguous()
                or t.get_device() != index):
            raise RuntimeError("k_scale_per_block and v_scale_per_block must be contiguous float32 tensors "
                               "[num_blocks, num_kv_heads] on the cache's device")
    seqs = context_lens.numel()
    if block_tables.dim() != 2 or block_tables.shape[0] != seqs:
        raise RuntimeError("block_tables must be [num_seqs, max_blocks_per_seq] with one context length per row")
    for t in (block_tables, context_lens, cu_tokens):
        if t is not None and (t.dtype is not torch.int32 or not t.is_contiguous() or t.get_device() != index):
            raise RuntimeError("block_tables, context_lens and cu_tokens must be contiguous int32 on the cache's device")
    if cu_tokens is not None:
        if cu_tokens.numel() != seqs + 1:
            raise RuntimeError("cu_tokens must have num_seqs + 1 entries")
        p.cu_tokens = cu_tokens.data_ptr()
    if cos_sin is not None:
        _check_rotation(cos_sin, index)
        p.cos_sin = cos_sin.data_ptr()
        p.max_position, p.rotary_dim = cos_sin.shape
    elif query is not None:
        raise RuntimeError("queries are only taken to be rotated: cos_sin is missing")
    _check_queries(p, query, query_out, rows, index)
    p.key, p.value = key.data_ptr(), value.data_ptr()
    p.key_cache, p.value_cache = key_cache.data_ptr(), value_cache.data_ptr()
    p.k_scale_per_block, p.v_scale_per_block = k_scale_per_block.data_ptr(), v_scale_per_block.data_ptr()
    p.block_tables, p.context_lens = block_tables.data_ptr(), context_lens.data_ptr()
    p.num_seqs, p.num_tokens, p.num_kv_heads, p.head_size = seqs, rows[0], kv_heads, head_size
    p.block_size, p.max_blocks_per_seq, p.num_blocks = block_size, block_tables.shape[1], num_blocks
    p.kv_dtype, p.interleaved = _kv_dtype(key_cache), int(interleaved)
    _launch.call(_cabi.load_library().pa_append_block_scaled, p, index)
