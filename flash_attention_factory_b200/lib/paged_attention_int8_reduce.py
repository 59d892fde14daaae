"""``paged_attention_int8_reduce.run``: 8-bit integer KV cache, split-context (attention + merge kernel).

No reference counterpart: the surface is that of ``paged_attention_fp8_reduce`` (18 positional
arguments, ``int8_scale`` in the place of ``fp8_scale``) over ``torch.int8`` caches, whose codes
stand for code * scale.  The scale is ``int8_scale``, or one per KV head, or one for each block
of tokens and KV head; ``cache_ops.append_block_scaled`` fills and keeps the latter.
``tem_output`` may be float32 instead of float16: partial rows are then not rounded on their way
to the merge (an error of 2.1e-4 of a result on average, its own rounding, instead of 2.9e-4).
"""
from __future__ import annotations

from . import _shim

ENTRY = _ENTRY = "launch_kernels_int8_reduce"


def run(max_logits, exp_sums, tem_output, output, debug_output, query, key_cache, value_cache,
        block_tables, context_lens, num_queries_per_tokens, sm_scale, int8_scale, block_size,
        max_context_len, alibi_slopes, sinks, softcap):
    p = _shim.build_params(max_logits, exp_sums, tem_output, output, debug_output, query, key_cache,
                           value_cache, block_tables, context_lens, num_queries_per_tokens, sm_scale,
                           int8_scale, block_size, max_context_len, alibi_slopes, sinks, softcap,
                           fp8=True, int8=True)
    _shim.check_scratch(p, max_logits, exp_sums, tem_output)
    return _shim.run_entry(_ENTRY, p, query.device)


def params(max_logits, exp_sums, tem_output, output, debug_output, query, key_cache, value_cache,
           block_tables, context_lens, num_queries_per_tokens, sm_scale, int8_scale, block_size,
           max_context_len, alibi_slopes, sinks, softcap, *, k_scale_per_head=None, v_scale_per_head=None,
           use_alibi=False, use_softcap=False, k_scale_per_block=None, v_scale_per_block=None):
    """The checked argument block (`pa_params`) of an ``enqueue`` call with these arguments,
    for callers that launch many steps on the same tensors (`host_io.DecodeStepIO.bind`)."""
    p = _shim.build_params(max_logits, exp_sums, tem_output, output, debug_output, query, key_cache,
                           value_cache, block_tables, context_lens, num_queries_per_tokens, sm_scale,
                           int8_scale, block_size, max_context_len, alibi_slopes, sinks, softcap,
                           fp8=True, int8=True, k_scale_per_head=k_scale_per_head, v_scale_per_head=v_scale_per_head,
                           use_alibi=use_alibi, use_softcap=use_softcap, k_scale_per_block=k_scale_per_block,
                           v_scale_per_block=v_scale_per_block)
    _shim.check_scratch(p, max_logits, exp_sums, tem_output)
    return p


def enqueue(max_logits, exp_sums, tem_output, output, debug_output, query, key_cache, value_cache,
            block_tables, context_lens, num_queries_per_tokens, sm_scale, int8_scale, block_size,
            max_context_len, alibi_slopes, sinks, softcap, *, k_scale_per_head=None, v_scale_per_head=None,
            use_alibi=False, use_softcap=False, k_scale_per_block=None, v_scale_per_block=None):
    """Same arguments as ``run`` but asynchronous on the current stream (returns nothing).

    ``k_scale_per_head`` / ``v_scale_per_head`` (float32 [num_kv_heads], optional, no reference
    counterpart) replace the scalar ``int8_scale`` for K / V with one scale per KV head;
    ``k_scale_per_block`` / ``v_scale_per_block`` (float32 [num_blocks, num_kv_heads]) with one per
    block and head."""
    p = params(max_logits, exp_sums, tem_output, output, debug_output, query, key_cache, value_cache,
               block_tables, context_lens, num_queries_per_tokens, sm_scale, int8_scale, block_size,
               max_context_len, alibi_slopes, sinks, softcap, k_scale_per_head=k_scale_per_head,
               v_scale_per_head=v_scale_per_head, use_alibi=use_alibi, use_softcap=use_softcap,
               k_scale_per_block=k_scale_per_block, v_scale_per_block=v_scale_per_block)
    _shim.enqueue_entry(_ENTRY, p, query.device)
