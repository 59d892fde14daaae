"""torch custom-op registration of the operators (asynchronous form).

`import flash_attention_factory_b200.torch_ops` registers
`torch.ops.paged_attention_b200.{loop, reduce, fp8_loop, fp8_reduce, int8_loop, int8_reduce, diff,
rope_and_cache, append_block_scaled}`: in-place operators on
torch's current stream that a serving stack can call from traced / graph-captured code
without the blocking, time-returning `run(...)` of the reference surface.  The argument order
is the reference's (paged_attention_loop/paged_attention_loop.cpp:21-38); `debug_output` is
dropped because nothing ever reads it.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import cache_ops
from .lib import (paged_attention_diff, paged_attention_fp8_loop, paged_attention_fp8_reduce, paged_attention_int8_loop,
                  paged_attention_int8_reduce, paged_attention_loop, paged_attention_reduce)

_MUTATED = ("max_logits", "exp_sums", "tem_output", "output")


@torch.library.custom_op("paged_attention_b200::loop", mutates_args=_MUTATED)
def loop(max_logits: torch.Tensor, exp_sums: torch.Tensor, tem_output: torch.Tensor, output: torch.Tensor,
         query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, block_tables: torch.Tensor,
         context_lens: torch.Tensor, num_queries_per_tokens: int, sm_scale: float, block_size: int,
         max_context_len: int, alibi_slopes: torch.Tensor, sinks: Optional[torch.Tensor], softcap: float) -> None:
    paged_attention_loop.enqueue(max_logits, exp_sums, tem_output, output, None, query, key_cache, value_cache,
                                 block_tables, context_lens, num_queries_per_tokens, sm_scale, block_size,
                                 max_context_len, alibi_slopes, sinks, softcap)


@torch.library.custom_op("paged_attention_b200::reduce", mutates_args=_MUTATED)
def reduce(max_logits: torch.Tensor, exp_sums: torch.Tensor, tem_output: torch.Tensor, output: torch.Tensor,
           query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, block_tables: torch.Tensor,
           context_lens: torch.Tensor, num_queries_per_tokens: int, sm_scale: float, block_size: int,
           max_context_len: int, alibi_slopes: torch.Tensor, sinks: Optional[torch.Tensor], softcap: float) -> None:
    paged_attention_reduce.enqueue(max_logits, exp_sums, tem_output, output, None, query, key_cache, value_cache,
                                   block_tables, context_lens, num_queries_per_tokens, sm_scale, block_size,
                                   max_context_len, alibi_slopes, sinks, softcap)


@torch.library.custom_op("paged_attention_b200::fp8_loop", mutates_args=_MUTATED)
def fp8_loop(max_logits: torch.Tensor, exp_sums: torch.Tensor, tem_output: torch.Tensor, output: torch.Tensor,
             query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, block_tables: torch.Tensor,
             context_lens: torch.Tensor, num_queries_per_tokens: int, sm_scale: float, fp8_scale: float,
             block_size: int, max_context_len: int, alibi_slopes: torch.Tensor, sinks: Optional[torch.Tensor],
             softcap: float, k_scale_per_block: Optional[torch.Tensor] = None,
             v_scale_per_block: Optional[torch.Tensor] = None, k_scale_per_head: Optional[torch.Tensor] = None,
             v_scale_per_head: Optional[torch.Tensor] = None) -> None:
    paged_attention_fp8_loop.enqueue(max_logits, exp_sums, tem_output, output, None, query, key_cache,
                                     value_cache, block_tables, context_lens, num_queries_per_tokens, sm_scale,
                                     fp8_scale, block_size, max_context_len, alibi_slopes, sinks, softcap,
                                     k_scale_per_block=k_scale_per_block, v_scale_per_block=v_scale_per_block,
                                     k_scale_per_head=k_scale_per_head, v_scale_per_head=v_scale_per_head)


@torch.library.custom_op("paged_attention_b200::fp8_reduce", mutates_args=_MUTATED)
def fp8_reduce(max_logits: torch.Tensor, exp_sums: torch.Tensor, tem_output: torch.Tensor, output: torch.Tensor,
               query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, block_tables: torch.Tensor,
               context_lens: torch.Tensor, num_queries_per_tokens: int, sm_scale: float, fp8_scale: float,
               block_size: int, max_context_len: int, alibi_slopes: torch.Tensor, sinks: Optional[torch.Tensor],
               softcap: float, k_scale_per_block: Optional[torch.Tensor] = None,
               v_scale_per_block: Optional[torch.Tensor] = None, k_scale_per_head: Optional[torch.Tensor] = None,
               v_scale_per_head: Optional[torch.Tensor] = None) -> None:
    paged_attention_fp8_reduce.enqueue(max_logits, exp_sums, tem_output, output, None, query, key_cache,
                                       value_cache, block_tables, context_lens, num_queries_per_tokens, sm_scale,
                                       fp8_scale, block_size, max_context_len, alibi_slopes, sinks, softcap,
                                       k_scale_per_block=k_scale_per_block, v_scale_per_block=v_scale_per_block,
                                       k_scale_per_head=k_scale_per_head, v_scale_per_head=v_scale_per_head)


@torch.library.custom_op("paged_attention_b200::int8_loop", mutates_args=_MUTATED)
def int8_loop(max_logits: torch.Tensor, exp_sums: torch.Tensor, tem_output: torch.Tensor, output: torch.Tensor,
              query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, block_tables: torch.Tensor,
              context_lens: torch.Tensor, num_queries_per_tokens: int, sm_scale: float, int8_scale: float,
              block_size: int, max_context_len: int, alibi_slopes: torch.Tensor, sinks: Optional[torch.Tensor],
              softcap: float, k_scale_per_block: Optional[torch.Tensor] = None,
              v_scale_per_block: Optional[torch.Tensor] = None, k_scale_per_head: Optional[torch.Tensor] = None,
              v_scale_per_head: Optional[torch.Tensor] = None) -> None:
    paged_attention_int8_loop.enqueue(max_logits, exp_sums, tem_output, output, None, query, key_cache,
                                      value_cache, block_tables, context_lens, num_queries_per_tokens, sm_scale,
                                      int8_scale, block_size, max_context_len, alibi_slopes, sinks, softcap,
                                      k_scale_per_block=k_scale_per_block, v_scale_per_block=v_scale_per_block,
                                      k_scale_per_head=k_scale_per_head, v_scale_per_head=v_scale_per_head)


@torch.library.custom_op("paged_attention_b200::int8_reduce", mutates_args=_MUTATED)
def int8_reduce(max_logits: torch.Tensor, exp_sums: torch.Tensor, tem_output: torch.Tensor, output: torch.Tensor,
              query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, block_tables: torch.Tensor,
              context_lens: torch.Tensor, num_queries_per_tokens: int, sm_scale: float, int8_scale: float,
              block_size: int, max_context_len: int, alibi_slopes: torch.Tensor, sinks: Optional[torch.Tensor],
              softcap: float, k_scale_per_block: Optional[torch.Tensor] = None,
              v_scale_per_block: Optional[torch.Tensor] = None, k_scale_per_head: Optional[torch.Tensor] = None,
              v_scale_per_head: Optional[torch.Tensor] = None) -> None:
    paged_attention_int8_reduce.enqueue(max_logits, exp_sums, tem_output, output, None, query, key_cache,
                                      value_cache, block_tables, context_lens, num_queries_per_tokens, sm_scale,
                                      int8_scale, block_size, max_context_len, alibi_slopes, sinks, softcap,
                                      k_scale_per_block=k_scale_per_block, v_scale_per_block=v_scale_per_block,
                                      k_scale_per_head=k_scale_per_head, v_scale_per_head=v_scale_per_head)


@torch.library.custom_op("paged_attention_b200::diff", mutates_args=_MUTATED)
def diff(max_logits: torch.Tensor, exp_sums: torch.Tensor, tem_output: torch.Tensor, output: torch.Tensor,
         query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, block_tables: torch.Tensor,
         context_lens: torch.Tensor, lambdas: torch.Tensor, sm_scale: float, kv_scale: float, block_size: int,
         max_context_len: int, norm_weight: Optional[torch.Tensor] = None, norm_eps: float = 1e-5,
         norm_scale: float = 1.0, k_scale_per_head: Optional[torch.Tensor] = None,
         v_scale_per_head: Optional[torch.Tensor] = None, k_scale_per_block: Optional[torch.Tensor] = None,
         v_scale_per_block: Optional[torch.Tensor] = None) -> None:
    paged_attention_diff.enqueue(max_logits, exp_sums, tem_output, output, query, key_cache, value_cache, block_tables,
                                 context_lens, lambdas, sm_scale, kv_scale, block_size, max_context_len,
                                 norm_weight=norm_weight, norm_eps=norm_eps, norm_scale=norm_scale,
                                 k_scale_per_head=k_scale_per_head, v_scale_per_head=v_scale_per_head,
                                 k_scale_per_block=k_scale_per_block, v_scale_per_block=v_scale_per_block)


@torch.library.custom_op("paged_attention_b200::rope_and_cache", mutates_args=("query_out", "key_cache", "value_cache"))
def rope_and_cache(query: Optional[torch.Tensor], key: torch.Tensor, value: torch.Tensor, positions: torch.Tensor,
                   cos_sin: torch.Tensor, query_out: Optional[torch.Tensor], key_cache: torch.Tensor, value_cache: torch.Tensor,
                   slot_mapping: torch.Tensor, fp8_scale: float = 1.0, interleaved: bool = False,
                   k_scale_per_head: Optional[torch.Tensor] = None, v_scale_per_head: Optional[torch.Tensor] = None,
                   k_scale_per_block: Optional[torch.Tensor] = None,
                   v_scale_per_block: Optional[torch.Tensor] = None) -> None:
    cache_ops.rope_and_cache(query, key, value, positions, cos_sin, query_out, key_cache, value_cache, slot_mapping,
                             fp8_scale, interleaved=interleaved, k_scale_per_head=k_scale_per_head,
                             v_scale_per_head=v_scale_per_head, k_scale_per_block=k_scale_per_block,
                             v_scale_per_block=v_scale_per_block)


@torch.library.custom_op("paged_attention_b200::append_block_scaled",
                         mutates_args=("key_cache", "value_cache", "k_scale_per_block", "v_scale_per_block", "query_out"))
def append_block_scaled(key: torch.Tensor, value: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                        k_scale_per_block: torch.Tensor, v_scale_per_block: torch.Tensor, block_tables: torch.Tensor,
                        context_lens: torch.Tensor, cu_tokens: Optional[torch.Tensor] = None,
                        query: Optional[torch.Tensor] = None, query_out: Optional[torch.Tensor] = None,
                        cos_sin: Optional[torch.Tensor] = None, interleaved: bool = False) -> None:
    cache_ops.append_block_scaled(key, value, key_cache, value_cache, k_scale_per_block, v_scale_per_block, block_tables,
                                  context_lens, cu_tokens=cu_tokens, query=query, query_out=query_out, cos_sin=cos_sin,
                                  interleaved=interleaved)
