"""The split int8 operator with float32 scratch: partial rows that are not rounded to fp16."""
import ctypes
from types import SimpleNamespace

import pytest
import torch

from _fp64 import HALF, attention64, check, paged_case, to
from test_zero_head_scales_gpu import attend


def scales(case):
    return {f"{n}_scale_per_block": case[f"{n}_scale"] for n in "kv"}


def rms(x):
    return float(x.double().square().mean().sqrt())


@pytest.mark.gpu
@pytest.mark.parametrize("hk,group,d,bs", [(8, 4, 128, 16), (8, 5, 64, 64), (2, 8, 128, 32), (1, 3, 64, 128), (3, 2, 128, 16),
                                           (16, 2, 64, 32)])
def test_against_fp64(cuda_device, hk, group, d, bs):
    """Every number of heads per CTA, contexts of one partition and of many.

    With two-part weights and fp32 rows the rounding of the result is the only one of its size: the largest error is
    half a step plus HALF / 4 of a = sum p |v| for the fp32 chains (128-term dot products at 2^-23 of logits of at most
    about 20, exponentials at 2^-21: 2^-14 of a together), and the RMS error is that of rounding the exact result."""
    case = paged_case(200 + hk, [0, 1, 17, 513, 2900, 1100, 512, 4096], hk * group, hk, d, bs, spread=2.0)
    want, tol = attention64(case, case["k_scale"], case["v_scale"])
    got = attend("int8", "reduce", case, cuda_device, torch.float32, **scales(case))
    check(got, want, tol, f"hk{hk} d{d}")
    absolute = (tol - 2.0 ** -24 - torch.tensor([float(n) for n in case["context_lens"]]).view(-1, 1, 1) * 2.0 ** -25
                * _largest(case).view(-1, 1, 1)) / (4 * HALF)  # a itself, out of the wider bound
    # a weight's rest that is subnormal is off by 2^-25 of the reference: the n 2^-25 max|v| of the wider bound
    tight = HALF * want.abs() + HALF / 4 * absolute + (tol - 4 * HALF * absolute)
    check(got, want, tight, f"hk{hk} d{d}, tight")
    assert rms(got.double() - want) <= 1.1 * rms(want.half().double() - want)


def _largest(case):
    from _fp64 import cache_values, sequence

    v = cache_values(case["value_cache"], case["v_scale"])
    return torch.stack([sequence(v, row, n).abs().max() if n else torch.zeros(()).double()
                        for row, n in zip(case["block_tables"], case["context_lens"].tolist())])


@pytest.mark.gpu
def test_many_pairs_and_wide_launches(cuda_device):
    """The merge with a warp per pair (2048 pairs and more) and the 8-warp CTA: the bits of a sequence alone."""
    case = paged_case(210, [1024] * 160, 16, 8, 64, 64, spread=3.0)
    batch = attend("int8", "reduce", case, cuda_device, torch.float32, **scales(case))
    one = {**case, "query": case["query"][7:8], "block_tables": case["block_tables"][7:8], "context_lens": case["context_lens"][7:8]}
    assert torch.equal(attend("int8", "reduce", one, cuda_device, torch.float32, **scales(one))[0], batch[7])
    case = paged_case(211, [1100] * 130, 32, 8, 128, 16, spread=3.0)
    batch = attend("int8", "reduce", case, cuda_device, torch.float32, **scales(case))
    one = {**case, "query": case["query"][9:10], "block_tables": case["block_tables"][9:10], "context_lens": case["context_lens"][9:10]}
    assert torch.equal(attend("int8", "reduce", one, cuda_device, torch.float32, **scales(one))[0], batch[9])


@pytest.mark.gpu
def test_through_serving_torch_ops_and_host_batches(cuda_device):
    import flash_attention_factory_b200.torch_ops  # noqa: F401
    from flash_attention_factory_b200 import _cabi
    from flash_attention_factory_b200.lib import paged_attention_int8_reduce as mod
    from flash_attention_factory_b200.serving import AutoDecodePlan, paged_attention_auto

    dev, lens = cuda_device, [700, 40, 1500, 9, 300, 0, 513, 77]
    case = paged_case(212, lens, 8, 4, 128, 16)
    c = to(case, dev)
    direct = attend("int8", "reduce", case, dev, torch.float32, **scales(case))
    plan = AutoDecodePlan(lens, 8, 128, 16, c["block_tables"].size(1), dev, fold_short_fraction=1.0, partial_dtype=torch.float32)
    out = torch.zeros(8, 8, 128, dtype=torch.float16, device=dev)
    paged_attention_auto(plan, out, c["query"], c["key_cache"], c["value_cache"], c["block_tables"], c["context_lens"], 2,
                         case["sm_scale"], k_scale_per_block=c["k_scale"], v_scale_per_block=c["v_scale"])
    assert plan.loop is None and torch.equal(out.cpu(), direct)
    ml, es = (torch.empty(8, 8, 3, device=dev) for _ in range(2))
    tmp = torch.empty(8, 8, 3, 128, device=dev)
    alibi = torch.ones(8, device=dev)
    out.zero_()
    torch.ops.paged_attention_b200.int8_reduce(ml, es, tmp, out, c["query"], c["key_cache"], c["value_cache"], c["block_tables"],
                                               c["context_lens"], 2, case["sm_scale"], 1.0, 16, 1500, alibi, None, -1.0,
                                               c["k_scale"], c["v_scale"])
    assert torch.equal(out.cpu(), direct)
    q, bt, cl = (torch.empty_like(c[n]) for n in ("query", "block_tables", "context_lens"))
    guard = torch.full((8 * 8 * 3 * 128 + 64,), 7.0, device=dev)  # the scratch and what lies behind it
    p = mod.params(ml, es, guard[:-64].view(8, 8, 3, 128), out, None, q, c["key_cache"], c["value_cache"], bt, cl, 2,
                   case["sm_scale"], 1.0, 16, 1500, alibi, None, -1.0, k_scale_per_block=c["k_scale"], v_scale_per_block=c["v_scale"])
    host = [case[n].pin_memory() for n in ("query", "block_tables", "context_lens")]
    for n in (1, 3):
        host_out = torch.zeros(8, 8, 128, dtype=torch.float16).pin_memory()
        io = _cabi.PaHostBatch()
        io.host_query, io.host_block_tables, io.host_context_lens = (t.data_ptr() for t in host)
        io.host_out, io.sub_batches = host_out.data_ptr(), n
        _cabi.check(_cabi.load_library().pa_decode_step_host_batch(
            _cabi.ENTRY_IDS[mod.ENTRY], ctypes.byref(p), ctypes.byref(io),
            ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream), 1))
        assert torch.equal(host_out, direct), n
    assert (guard[-64:] == 7.0).all()


def test_only_the_int8_operator_takes_float32_scratch():
    from flash_attention_factory_b200 import _cabi
    from flash_attention_factory_b200.lib import _shim

    stats, rows = torch.empty(2, 4, 3), torch.empty(2, 4, 3, 64)
    base = dict(num_seqs=2, num_heads=4, max_num_partitions=3, head_size=64)
    for kv in (_cabi.KV_F16, _cabi.KV_FP8_E5M2, _cabi.KV_FP8_E4M3):
        p = SimpleNamespace(kv_dtype=kv, tmp_out_f32=0, **base)
        _shim.check_scratch(p, stats, stats, rows.half())
        with pytest.raises(RuntimeError, match="float16"):
            _shim.check_scratch(p, stats, stats, rows)
        assert p.tmp_out_f32 == 0
    for t, flag in ((rows, 1), (rows.half(), 0)):
        p = SimpleNamespace(kv_dtype=_cabi.KV_INT8, tmp_out_f32=0, **base)
        _shim.check_scratch(p, stats, stats, t)
        assert p.tmp_out_f32 == flag
    for t in (rows.bfloat16(), rows.double(), rows[:1]):
        with pytest.raises(RuntimeError):
            _shim.check_scratch(SimpleNamespace(kv_dtype=_cabi.KV_INT8, tmp_out_f32=0, **base), stats, stats, t)
