"""Shared body of the four ``run`` functions.

Unpacks torch tensors exactly as the reference's pybind shims do
(paged_attention_loop/paged_attention_loop.cpp:44-79,
paged_attention_fp8_loop/paged_attention_fp8_loop.cpp:44-81): sizes come from
the tensor shapes, pointers from ``data_ptr()``, int32 tables are read as
uint32.  torch is used for device memory and the current stream only.
"""
from __future__ import annotations

import torch

from .. import _cabi, _launch

_F16, _F32, _I32 = torch.float16, torch.float32, torch.int32


def _require(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def _kv_dtype_of(cache: torch.Tensor, fp8: bool, int8: bool = False) -> int:
    if int8:
        _require(cache.dtype == torch.int8, f"key/value cache must be int8, got {cache.dtype}")
        return _cabi.KV_INT8
    if not fp8:
        _require(cache.dtype == torch.float16, f"key/value cache must be float16, got {cache.dtype}")
        return _cabi.KV_F16
    if cache.dtype == torch.float8_e4m3fn:
        return _cabi.KV_FP8_E4M3
    # uint8 storage means e5m2, the format the reference binding hard-wires
    # (paged_attention_fp8_loop/paged_attention_fp8_loop.cpp:43)
    _require(cache.dtype in (torch.float8_e5m2, torch.uint8),
             f"FP8 cache must be float8_e5m2, float8_e4m3fn or uint8, got {cache.dtype}")
    return _cabi.KV_FP8_E5M2


def _block_scale(t: torch.Tensor, name: str, shape, index: int, fp8: bool) -> int:
    if not fp8:
        raise RuntimeError("per-block scales belong to the FP8 and int8 operators")
    if t.dtype is not _F32 or t.shape != shape or t.get_device() != index or not t.is_contiguous():
        raise RuntimeError(f"{name} must be float32 [num_blocks, num_kv_heads] on the device")
    return t.data_ptr()


def build_params(max_logits, exp_sums, tem_output, output, debug_output, query, key_cache,
                 value_cache, block_tables, context_lens, num_queries_per_tokens, sm_scale,
                 fp8_scale, block_size, max_context_len, alibi_slopes, sinks, softcap,
                 fp8: bool, k_scale_per_head=None, v_scale_per_head=None,
                 use_alibi: bool = False, use_softcap: bool = False,
                 k_scale_per_block=None, v_scale_per_block=None, int8: bool = False) -> _cabi.PaParams:
    """Validates what the reference's ``data_ptr<float>()`` calls would and fills pa_params.

    ``debug_output``, ``alibi_slopes``, ``softcap`` are accepted and ignored like in the
    reference (paged_attention_kernel_loop.hpp:175-178,329-342).  ``int8`` (with ``fp8``, whose
    scale arguments it shares) selects the integer cache.
    """
    if not query.is_cuda:
        raise RuntimeError("paged attention needs CUDA tensors (no CPU fallback exists)")
    # the reference's data_ptr<float>() calls reject other dtypes (paged_attention_loop.cpp:47-52)
    if (max_logits.dtype is not _F32 or exp_sums.dtype is not _F32 or alibi_slopes.dtype is not _F32
            or (debug_output is not None and debug_output.dtype is not _F32)):
        # callers of this package that have no debug tensor pass None
        for name, t in (("max_logits", max_logits), ("exp_sums", exp_sums), ("alibi_slopes", alibi_slopes),
                        ("debug_output", debug_output)):
            if t is not None:
                _require(t.dtype == torch.float32, f"expected scalar type Float but found {t.dtype} ({name})")
    if query.dtype is not _F16 or output.dtype is not _F16:
        raise RuntimeError("query and output must be float16")
    if block_tables.dtype is not _I32 or context_lens.dtype is not _I32:
        raise RuntimeError("block_tables and context_lens must be int32")
    if query.dim() != 3 or key_cache.dim() != 4 or block_tables.dim() != 2 or max_logits.dim() != 3:
        raise RuntimeError("unexpected tensor rank")
    num_blocks, rows, kv_heads, cache_head_size = cache_shape = key_cache.shape
    if cache_shape != value_cache.shape or key_cache.dtype is not value_cache.dtype:
        raise RuntimeError("key_cache and value_cache must have the same shape and dtype")
    if sinks is not None and sinks.dtype is not _F16:
        raise RuntimeError("sinks must be float16")
    index = query.get_device()
    for t in (max_logits, exp_sums, tem_output, output, query, key_cache, value_cache, block_tables, context_lens, sinks):
        if t is None:
            continue
        if not t.is_contiguous():
            raise RuntimeError("all tensors must be contiguous")
        if t.get_device() != index:
            raise RuntimeError("all tensors must be on the same device")
    num_seqs, num_heads, head_size = query.shape
    table_rows, table_columns = block_tables.shape
    if rows != block_size:
        raise RuntimeError("block_size does not match key_cache.size(1)")
    if cache_head_size != head_size:
        raise RuntimeError("head_size of cache and query differ")
    if context_lens.numel() != num_seqs or table_rows != num_seqs:
        raise RuntimeError("context_lens / block_tables do not match the number of sequences")

    p = _cabi.PaParams()
    p.out = output.data_ptr()
    p.max_logits = max_logits.data_ptr()
    p.exp_sums = exp_sums.data_ptr()
    p.tmp_out = tem_output.data_ptr()
    p.query = query.data_ptr()
    p.key_cache = key_cache.data_ptr()
    p.value_cache = value_cache.data_ptr()
    p.sinks = sinks.data_ptr() if sinks is not None else None
    p.block_tables = block_tables.data_ptr()
    p.context_lens = context_lens.data_ptr()
    p.num_seqs = num_seqs
    p.num_heads = num_heads
    p.head_size = head_size
    p.num_kv_heads = kv_heads
    p.max_num_partitions = max_logits.shape[2]
    p.max_blocks_per_seq = table_columns
    p.block_size = int(block_size)
    p.num_queries_per_tokens = int(num_queries_per_tokens)
    p.max_context_len = max(0, min(int(max_context_len), 0xFFFFFFFF))
    p.num_blocks = num_blocks
    p.sm_scale = float(sm_scale)
    p.fp8_scale = float(fp8_scale)
    p.kv_dtype = _kv_dtype_of(key_cache, fp8, int8)
    if k_scale_per_head is not None or v_scale_per_head is not None:
        for name, t in (("k_scale_per_head", k_scale_per_head), ("v_scale_per_head", v_scale_per_head)):
            if t is not None:
                _require(fp8, "per-head scales belong to the FP8 and int8 operators")
                _require(t.dtype == torch.float32 and t.is_contiguous() and t.device == query.device
                         and t.numel() == kv_heads, f"{name} must be float32 [num_kv_heads] on the device")
                setattr(p, name, t.data_ptr())
    if k_scale_per_block is not None:
        p.k_scale_per_block = _block_scale(k_scale_per_block, "k_scale_per_block", (num_blocks, kv_heads), index, fp8)
    if v_scale_per_block is not None:
        p.v_scale_per_block = _block_scale(v_scale_per_block, "v_scale_per_block", (num_blocks, kv_heads), index, fp8)
    # opt-in only: by default alibi_slopes and softcap are ignored, as in the reference
    if use_alibi:
        _require(alibi_slopes.is_cuda and alibi_slopes.is_contiguous()
                 and alibi_slopes.numel() == query.size(1), "alibi_slopes must be float32 [num_heads] on the device")
        p.alibi_slopes = alibi_slopes.data_ptr()
    if use_softcap and softcap > 0:
        p.softcap = float(softcap)
    return p


def check_scratch(p: _cabi.PaParams, max_logits, exp_sums, tem_output) -> None:
    """The split variant writes [S, H, NP] and [S, H, NP, D] scratch: check the extents."""
    s, h, npart, d = p.num_seqs, p.num_heads, p.max_num_partitions, p.head_size
    _require(tuple(max_logits.shape) == (s, h, npart) and tuple(exp_sums.shape) == (s, h, npart),
             "max_logits / exp_sums must be [num_seqs, num_heads, max_num_partitions]")
    if p.kv_dtype == _cabi.KV_INT8 and tem_output.dtype == torch.float32:
        p.tmp_out_f32 = 1  # the split int8 operator keeps its partial rows in the scratch's type
    else:
        _require(tem_output.dtype == torch.float16, "tem_output must be float16 (int8 caches: or float32)")
    _require(tem_output.numel() >= s * h * npart * d,
             "tem_output must be [num_seqs, num_heads, max_num_partitions, head_size]")


def run_entry(entry: str, p: _cabi.PaParams, device: torch.device) -> list[float]:
    """Blocking launch on torch's current stream; returns device microseconds per kernel."""
    with torch.cuda.device(device):
        stream = torch.cuda.current_stream(device).cuda_stream
        return _cabi.launch(entry, p, stream, timed=True)


def enqueue_entry(entry: str, p: _cabi.PaParams, device: torch.device) -> None:
    """Asynchronous launch on torch's current stream (no timing, no host sync)."""
    index = device.index if device.index is not None else torch.cuda.current_device()
    _launch.call(getattr(_cabi.load_library(), entry), p, index, None)
