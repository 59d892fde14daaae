"""``paged_attention_diff``: differential attention over the paged KV cache, one decode token per sequence.

No reference counterpart.  Head h of the result has two query maps, rows 2 h and 2 h + 1 of ``query``
[num_seqs, 2 H, head_size]; KV pair k = h / (H / HK) holds its two K heads at 2 k and 2 k + 1 of the cache
and its value vector of 2 * head_size elements as V heads 2 k and 2 k + 1 side by side, so both caches are
[num_blocks, block_size, 2 HK, head_size] and ``cache_ops`` fills them like any other:

    o[h] = (softmax(s q[2h] K[2k]^T) - lambdas[h] softmax(s q[2h+1] K[2k+1]^T)) [V[2k] V[2k+1]]

and, with ``norm_weight`` w, o[h] / sqrt(mean(o[h]^2) + norm_eps) * w * norm_scale (the head-wise norm of a
differential transformer, norm_scale = 1 - lambda_init).  An empty context gives zeros.  Cache types: fp16,
FP8 and int8, with one scale (``kv_scale``), or one per cache head, or one per block and cache head.
"""
from __future__ import annotations

import ctypes

import torch

from .. import _cabi, _launch
from . import _shim

_F32 = torch.float32

ENTRY = "launch_kernels_diff"


def _kv_dtype(cache: torch.Tensor) -> int:
    return _shim._kv_dtype_of(cache, cache.dtype != torch.float16, cache.dtype == torch.int8)


def scratch(query: torch.Tensor, key_cache: torch.Tensor, max_context_len: int):
    """(max_logits, exp_sums, tem_output) for calls of this shape: float32 [S, 2 H, NP], the same, and
    [S, 2 H, NP, 2 D].  NP sets how finely a context is split; any NP >= 1 gives a correct result.  For large batches
    of long contexts that is memory: 256 sequences of 32768 tokens with 32 heads of 128 over an fp16 cache get 2.1 GB."""
    s, h2, d = query.shape
    kv_dtype = _kv_dtype(key_cache)
    hint = max(0, min(int(max_context_len), 0xFFFFFFFF))
    npart = int(_cabi.load_library().pa_diff_num_partitions(s, key_cache.size(2), d, hint, kv_dtype))
    _shim._require(npart > 0, "Unsupported head size or number of KV heads")
    stats = torch.empty(2, s, h2, npart, dtype=torch.float32, device=query.device)
    return stats[0], stats[1], torch.empty(s, h2, npart, 2 * d, dtype=torch.float32, device=query.device)


def params(max_logits, exp_sums, tem_output, output, query, key_cache, value_cache, block_tables, context_lens,
           lambdas, sm_scale, kv_scale, block_size, max_context_len, *, norm_weight=None, norm_eps=1e-5,
           norm_scale=1.0, k_scale_per_head=None, v_scale_per_head=None, k_scale_per_block=None,
           v_scale_per_block=None) -> _cabi.PaDiffParams:
    """The checked argument block (`pa_diff_params`) of an ``enqueue`` call with these arguments."""
    index = query.get_device()
    if index < 0:
        raise RuntimeError("paged attention needs CUDA tensors (no CPU fallback exists)")
    if query.dim() != 3 or key_cache.dim() != 4 or block_tables.dim() != 2 or max_logits.dim() != 3:
        raise RuntimeError("unexpected tensor rank")
    s, h2, d = query.shape
    num_blocks, rows, kv_heads, cache_head_size = cache_shape = key_cache.shape
    table_rows, table_columns = block_tables.shape
    npart = max_logits.shape[2]
    if h2 % 2 or kv_heads % 2 or kv_heads == 0:
        raise RuntimeError("differential attention needs query heads and KV heads in pairs")
    if h2 % kv_heads:
        raise RuntimeError("the number of query heads must be a multiple of the number of KV heads")
    if query.dtype is not torch.float16 or output.dtype is not torch.float16:
        raise RuntimeError("query and output must be float16")
    if output.shape != (s, h2 // 2, 2 * d):
        raise RuntimeError("output must be [num_seqs, H, 2 * head_size]")
    if max_logits.dtype is not _F32 or exp_sums.dtype is not _F32 or tem_output.dtype is not _F32:
        raise RuntimeError("the scratch must be float32")
    if (max_logits.shape != (s, h2, npart) or exp_sums.shape != (s, h2, npart)
            or tem_output.numel() < s * h2 * npart * 2 * d):
        raise RuntimeError("the scratch must be [num_seqs, 2 H, NP] twice and [num_seqs, 2 H, NP, 2 * head_size]")
    if block_tables.dtype is not torch.int32 or context_lens.dtype is not torch.int32:
        raise RuntimeError("block_tables and context_lens must be int32")
    if context_lens.numel() != s or table_rows != s:
        raise RuntimeError("context_lens / block_tables do not match the number of sequences")
    if cache_shape != value_cache.shape or key_cache.dtype is not value_cache.dtype:
        raise RuntimeError("key_cache and value_cache must have the same shape and dtype")
    if rows != block_size:
        raise RuntimeError("block_size does not match key_cache.size(1)")
    if cache_head_size != d:
        raise RuntimeError("head_size of cache and query differ")
    if lambdas.dtype is not _F32 or lambdas.numel() != h2 // 2:
        raise RuntimeError("lambdas must be float32 [H]")
    if norm_weight is not None and (norm_weight.dtype is not _F32 or norm_weight.numel() != 2 * d):
        raise RuntimeError("norm_weight must be float32 [2 * head_size]")
    for t in (max_logits, exp_sums, tem_output, output, query, key_cache, value_cache, block_tables, context_lens,
              lambdas, norm_weight):
        if t is not None and (not t.is_contiguous() or t.get_device() != index):
            raise RuntimeError("all tensors must be contiguous and on the same device")
    q = _cabi.PaDiffParams()
    p = q.attn
    p.out, p.max_logits, p.exp_sums = output.data_ptr(), max_logits.data_ptr(), exp_sums.data_ptr()
    p.tmp_out, p.query = tem_output.data_ptr(), query.data_ptr()
    p.key_cache, p.value_cache = key_cache.data_ptr(), value_cache.data_ptr()
    p.block_tables, p.context_lens = block_tables.data_ptr(), context_lens.data_ptr()
    p.num_seqs, p.num_heads, p.head_size, p.num_kv_heads = s, h2, d, kv_heads
    p.max_num_partitions, p.max_blocks_per_seq = npart, table_columns
    p.block_size, p.num_queries_per_tokens = int(block_size), h2 // kv_heads
    p.max_context_len = max(0, min(int(max_context_len), 0xFFFFFFFF))
    p.num_blocks, p.sm_scale, p.fp8_scale = num_blocks, float(sm_scale), float(kv_scale)
    p.kv_dtype = _kv_dtype(key_cache)
    if not (k_scale_per_head is v_scale_per_head is k_scale_per_block is v_scale_per_block is None):
        if key_cache.dtype == torch.float16:
            raise RuntimeError("scale arrays belong to FP8 and int8 caches")
        for name, t, shape in (("k_scale_per_head", k_scale_per_head, (kv_heads,)),
                               ("v_scale_per_head", v_scale_per_head, (kv_heads,)),
                               ("k_scale_per_block", k_scale_per_block, (num_blocks, kv_heads)),
                               ("v_scale_per_block", v_scale_per_block, (num_blocks, kv_heads))):
            if t is not None:
                if t.dtype is not _F32 or not t.is_contiguous() or t.get_device() != index or t.shape != shape:
                    raise RuntimeError(f"{name} must be a contiguous float32 tensor of shape {shape} on the device")
                setattr(p, name, t.data_ptr())
    q.lambdas = lambdas.data_ptr()
    if norm_weight is not None:
        q.norm_weight, q.norm_eps = norm_weight.data_ptr(), float(norm_eps)
    q.norm_scale = float(norm_scale)
    return q


def enqueue(max_logits, exp_sums, tem_output, output, query, key_cache, value_cache, block_tables, context_lens,
            lambdas, sm_scale, kv_scale, block_size, max_context_len, *, norm_weight=None, norm_eps=1e-5,
            norm_scale=1.0, k_scale_per_head=None, v_scale_per_head=None, k_scale_per_block=None,
            v_scale_per_block=None) -> None:
    """One decode step, asynchronous on torch's current stream; writes ``output`` [S, H, 2 * head_size].

    The first three arguments are scratch (``scratch`` makes it).  ``max_context_len`` is a hint: results
    never depend on it."""
    q = params(max_logits, exp_sums, tem_output, output, query, key_cache, value_cache, block_tables, context_lens,
               lambdas, sm_scale, kv_scale, block_size, max_context_len, norm_weight=norm_weight, norm_eps=norm_eps,
               norm_scale=norm_scale, k_scale_per_head=k_scale_per_head, v_scale_per_head=v_scale_per_head,
               k_scale_per_block=k_scale_per_block, v_scale_per_block=v_scale_per_block)
    _launch.call(_cabi.load_library().launch_kernels_diff, q, query.get_device(), None)


def run(max_logits, exp_sums, tem_output, output, query, key_cache, value_cache, block_tables, context_lens,
        lambdas, sm_scale, kv_scale, block_size, max_context_len, *, norm_weight=None, norm_eps=1e-5,
        norm_scale=1.0, k_scale_per_head=None, v_scale_per_head=None, k_scale_per_block=None,
        v_scale_per_block=None) -> list[float]:
    """``enqueue``, blocking; returns device microseconds [attention, merge]."""
    q = params(max_logits, exp_sums, tem_output, output, query, key_cache, value_cache, block_tables, context_lens,
               lambdas, sm_scale, kv_scale, block_size, max_context_len, norm_weight=norm_weight, norm_eps=norm_eps,
               norm_scale=norm_scale, k_scale_per_head=k_scale_per_head, v_scale_per_head=v_scale_per_head,
               k_scale_per_block=k_scale_per_block, v_scale_per_block=v_scale_per_block)
    us = (ctypes.c_float * 2)()
    _launch.call(_cabi.load_library().launch_kernels_diff, q, query.get_device(), us)
    return [float(us[0]), float(us[1])]
