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


def test_registered_operators_take_what_the_python_forms_take():
    import torch

    import flash_attention_factory_b200.torch_ops  # noqa: F401
    from flash_attention_factory_b200.serving import paged_attention_auto

    ops = torch.ops.paged_attention_b200
    scales = [f"{n}_scale_per_{kind}" for kind in ("block", "head") for n in "kv"]
    for name in ("int8_loop", "int8_reduce", "fp8_loop", "fp8_reduce", "diff", "rope_and_cache"):
        args = {a.name: a for a in getattr(ops, name).default._schema.arguments}
        assert all(str(args[s].type) == "Optional[Tensor]" and args[s].default_value is None for s in scales), name
    args = {a.name: str(a.type) for a in ops.rope_and_cache.default._schema.arguments}
    assert args["query"] == args["query_out"] == "Optional[Tensor]"
    assert set(scales) <= set(inspect.signature(paged_attention_auto).parameters)


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["int8", "e4m3"])
@pytest.mark.parametrize("kind", ["head", "block"])
def test_scale_arrays_through_the_other_surfaces(cuda_device, cache, kind):
    """torch.ops and serving against the direct call, bit for bit."""
    import torch

    import flash_attention_factory_b200.torch_ops  # noqa: F401
    from _fp64 import paged_case, to
    from flash_attention_factory_b200.serving import AutoDecodePlan, paged_attention_auto
    from test_zero_head_scales_gpu import attend

    family, dev, lens = "int8" if cache == "int8" else "fp8", cuda_device, [700, 40, 1500, 9]
    case = paged_case(13, lens, 8, 4, 128, 16, cache=cache, scale=kind)
    c = to(case, dev)
    names = {f"{n}_scale_per_{kind}": f"{n}_scale" for n in "kv"}
    direct = {v: attend(family, v, case, dev, **{a: case[b] for a, b in names.items()}) for v in ("loop", "reduce")}
    kw = {a: c[b] for a, b in names.items()}
    ml, tmp = torch.empty(4, 8, 3, device=dev), torch.empty(4, 8, 3, 128, dtype=torch.float16, device=dev)
    out = torch.empty(4, 8, 128, dtype=torch.float16, device=dev)
    for variant, want in direct.items():
        out.zero_()
        getattr(torch.ops.paged_attention_b200, f"{family}_{variant}")(
            ml, ml.clone(), tmp, out, c["query"], c["key_cache"], c["value_cache"], c["block_tables"], c["context_lens"], 2,
            case["sm_scale"], 1.0, 16, 1500, torch.ones(8, device=dev), None, -1.0, **kw)
        assert torch.equal(out.cpu(), want), variant
    out.zero_()
    plan = AutoDecodePlan(lens, 8, 128, 16, c["block_tables"].size(1), dev)  # one long sequence carries the batch: reduce
    paged_attention_auto(plan, out, c["query"], c["key_cache"], c["value_cache"], c["block_tables"], c["context_lens"], 2,
                         case["sm_scale"], **kw)
    assert plan.loop is None and torch.equal(out.cpu(), direct["reduce"])


@pytest.mark.gpu
def test_registered_rope_and_cache_without_queries(cuda_device):
    import torch

    import flash_attention_factory_b200.torch_ops  # noqa: F401
    from flash_attention_factory_b200 import cache_ops
    from test_rope_cache_gpu import table

    dev, g = cuda_device, torch.Generator().manual_seed(1)
    k, v = (torch.randn(3, 2, 64, generator=g).half().to(dev) for _ in range(2))
    pos, slots, angles = torch.tensor([4, 0, 90], device=dev), torch.tensor([17, 3, 40], device=dev), table(100, 64).to(dev)
    sides = []
    for fn in (torch.ops.paged_attention_b200.rope_and_cache, cache_ops.rope_and_cache):
        pools = [torch.zeros(4, 16, 2, 64, dtype=torch.float16, device=dev) for _ in range(2)]
        fn(None, k, v, pos, angles, None, *pools, slots)
        sides.append(pools)
    assert all(torch.equal(a, b) for a, b in zip(*sides)) and int(sides[0][0].count_nonzero()) > 0
