"""The operators beside the reference's four: signatures and host-side arithmetic."""
import inspect

import pytest


def test_the_forms_of_differential_attention_take_the_same_arguments():
    from flash_attention_factory_b200.lib import paged_attention_diff as diff

    want = inspect.signature(diff.enqueue).parameters
    for fn in (diff.run, diff.params):
        assert list(inspect.signature(fn).parameters.values()) == list(want.values())


@pytest.mark.gpu
def test_blocking_differential_attention_with_keywords(cuda_device):
    import torch

    from _fp64 import paged_case, to
    from flash_attention_factory_b200.lib import paged_attention_diff as diff

    c = to(paged_case(3, [70, 9], 8, 4, 64, 16, cache="int8"), cuda_device)
    outs = [torch.empty(2, 4, 128, dtype=torch.float16, device=cuda_device) for _ in range(2)]
    ml, es, tmp = diff.scratch(c["query"], c["key_cache"], 70)
    lam = torch.full((4,), 0.5, device=cuda_device)
    for fn, out in zip((diff.run, diff.enqueue), outs):
        us = fn(max_logits=ml, exp_sums=es, tem_output=tmp, output=out, query=c["query"], key_cache=c["key_cache"],
                value_cache=c["value_cache"], block_tables=c["block_tables"], context_lens=c["context_lens"], lambdas=lam,
                sm_scale=0.125, kv_scale=1.0, block_size=16, max_context_len=70, k_scale_per_block=c["k_scale"],
                v_scale_per_block=c["v_scale"])
        assert fn is diff.enqueue or len(us) == 2
    assert torch.equal(*outs)


def test_partition_counts_of_the_largest_hints():
    """A hint near 2^32 is a long context, not an overflow; one beyond it is the largest."""
    import torch

    from flash_attention_factory_b200 import _cabi, build
    from flash_attention_factory_b200.lib import paged_attention_diff as diff

    build.build()
    n = _cabi.load_library().pa_diff_num_partitions
    for kv in range(4):
        for heads in (2, 8):
            for seqs in (1, 3, 3000):
                counts = [n(seqs, heads, 64, hint, kv) for hint in (2 ** 31, 2 ** 32 - 2000, 2 ** 32 - 64, 2 ** 32 - 1)]
                assert counts == [counts[0]] * 4 and counts[0] >= 1, (kv, heads, seqs, counts)
    cache = torch.empty(1, 16, 2, 64, dtype=torch.float16)
    scratch = diff.scratch(torch.empty(1, 2, 64, dtype=torch.float16, device="meta"), cache, 2 ** 40)
    assert scratch[0].shape[2] == n(1, 2, 64, 2 ** 32 - 1, 0)
