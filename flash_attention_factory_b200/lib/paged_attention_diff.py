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

from .. import _cabi
from . import _shim

ENTRY = "launch_kernels_diff"


def _kv_dtype(cache: torch.Tensor) -> int:
    return _shim._kv_dtype_of(cache, cache.dtype != torch.float16, cache.dtype == torch.int8)


def scratch(query: torch.Tensor, key_cache: torch.Tensor, max_context_len: int):
    """(max_logits, exp_sums, tem_output) for calls of this shape: float32 [S, 2 H, NP], the same, and
    [S, 2 H, NP, 2 D].  NP sets how finely a context is split; any NP >= 1 gives a correct result."""
    s, h2, d = query.shape
    kv_dtype = _kv_dtype(key_cache)
    npart = int(_cabi.load_library().pa_diff_num_partitions(s, key_cache.size(2), d, max(0, int(max_context_len)), kv_dtype))
    _shim._require(npart > 0, "Unsupported head size or number of KV heads")
    stats = torch.empty(2, s, h2, npart, dtype=torch.float32, device=query.device)
    return stats[0], stats[1], torch.empty(s, h2, npart, 2 * d, dtype=torch.float32, device=query.device)


def params(max_logits, exp_sums, tem_output, output, query, key_cache, value_cache, block_tables, context_lens,
           lambdas, sm_scale, kv_scale, block_size, max_context_len, *, norm_weight=None, norm_eps=1e-5,
           norm_scale=1.0, k_scale_per_head=None, v_scale_per_head=None, k_scale_per_block=None,
           v_scale_per_block=None) -> _cabi.PaDiffParams:
    """The checked argument block (`pa_diff_params`) of an ``enqueue`` call with these arguments."""
    require = _shim._require
    require(query.is_cuda, "paged attention needs CUDA tensors (no CPU fallback exists)")
    require(query.dim() == 3 and key_cache.dim() == 4 and block_tables.dim() == 2 and max_logits.dim() == 3,
            "unexpected tensor rank")
    s, h2, d = query.shape
    npart, device = max_logits.size(2), query.device
    require(h2 % 2 == 0 and key_cache.size(2) % 2 == 0 and key_cache.size(2) > 0,
            "differential attention needs query heads and KV heads in pairs")
    require(h2 % key_cache.size(2) == 0, "the number of query heads must be a multiple of the number of KV heads")
    require(query.dtype == torch.float16 and output.dtype == torch.float16, "query and output must be float16")
    require(tuple(output.shape) == (s, h2 // 2, 2 * d), "output must be [num_seqs, H, 2 * head_size]")
    require(max_logits.dtype == exp_sums.dtype == tem_output.dtype == torch.float32, "the scratch must be float32")
    require(tuple(max_logits.shape) == (s, h2, npart) and tuple(exp_sums.shape) == (s, h2, npart)
            and tem_output.numel() >= s * h2 * npart * 2 * d,
            "the scratch must be [num_seqs, 2 H, NP] twice and [num_seqs, 2 H, NP, 2 * head_size]")
    require(block_tables.dtype == torch.int32 and context_lens.dtype == torch.int32,
            "block_tables and context_lens must be int32")
    require(context_lens.numel() == s and block_tables.size(0) == s,
            "context_lens / block_tables do not match the number of sequences")
    require(key_cache.shape == value_cache.shape and key_cache.dtype == value_cache.dtype,
            "key_cache and value_cache must have the same shape and dtype")
    require(key_cache.size(1) == block_size, "block_size does not match key_cache.size(1)")
    require(key_cache.size(3) == d, "head_size of cache and query differ")
    require(lambdas.dtype == torch.float32 and lambdas.numel() == h2 // 2, "lambdas must be float32 [H]")
    require(norm_weight is None or (norm_weight.dtype == torch.float32 and norm_weight.numel() == 2 * d),
            "norm_weight must be float32 [2 * head_size]")
    for t in (max_logits, exp_sums, tem_output, output, query, key_cache, value_cache, block_tables, context_lens,
              lambdas, norm_weight):
        require(t is None or (t.is_contiguous() and t.device == device), "all tensors must be contiguous and on the same device")
    q = _cabi.PaDiffParams()
    p = q.attn
    p.out, p.max_logits, p.exp_sums = output.data_ptr(), max_logits.data_ptr(), exp_sums.data_ptr()
    p.tmp_out, p.query = tem_output.data_ptr(), query.data_ptr()
    p.key_cache, p.value_cache = key_cache.data_ptr(), value_cache.data_ptr()
    p.block_tables, p.context_lens = block_tables.data_ptr(), context_lens.data_ptr()
    p.num_seqs, p.num_heads, p.head_size, p.num_kv_heads = s, h2, d, key_cache.size(2)
    p.max_num_partitions, p.max_blocks_per_seq = npart, block_tables.size(1)
    p.block_size, p.num_queries_per_tokens = int(block_size), h2 // key_cache.size(2)
    p.max_context_len = max(0, min(int(max_context_len), 0xFFFFFFFF))
    p.num_blocks, p.sm_scale, p.fp8_scale = key_cache.size(0), float(sm_scale), float(kv_scale)
    fp16 = key_cache.dtype == torch.float16
    p.kv_dtype = _kv_dtype(key_cache)
    per_head, per_block = (key_cache.size(2),), (key_cache.size(0), key_cache.size(2))
    for name, t, shape in (("k_scale_per_head", k_scale_per_head, per_head), ("v_scale_per_head", v_scale_per_head, per_head),
                           ("k_scale_per_block", k_scale_per_block, per_block),
                           ("v_scale_per_block", v_scale_per_block, per_block)):
        if t is not None:
            require(not fp16, "scale arrays belong to FP8 and int8 caches")
            require(t.dtype == torch.float32 and t.is_contiguous() and t.device == device and tuple(t.shape) == shape,
                    f"{name} must be a contiguous float32 tensor of shape {shape} on the device")
            setattr(p, name, t.data_ptr())
    q.lambdas = lambdas.data_ptr()
    if norm_weight is not None:
        q.norm_weight, q.norm_eps = norm_weight.data_ptr(), float(norm_eps)
    q.norm_scale = float(norm_scale)
    return q


def _launch(q: _cabi.PaDiffParams, device, timed: bool):
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            return _launch(q, torch.device("cuda", torch.cuda.current_device()), timed)
    us = (ctypes.c_float * 2)() if timed else None
    stream = ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)
    _cabi.check(_cabi.load_library().launch_kernels_diff(ctypes.byref(q), stream, us))
    return [float(us[0]), float(us[1])] if timed else None


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
    _launch(q, query.device, timed=False)


def run(*args, **kwargs) -> list[float]:
    """``enqueue``, blocking; returns device microseconds [attention, merge]."""
    return _launch(params(*args, **kwargs), args[4].device, timed=True)
