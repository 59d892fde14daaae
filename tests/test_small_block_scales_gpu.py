"""FP8 attention under the block scales that append_block_scaled writes: max|row| / 448 or / 57344, far below
the normal halves for e5m2.  The weights of spread-out contexts have to keep their bits under them."""
import pytest
import torch

from _fp64 import attention64, check, paged_case
from test_zero_head_scales_gpu import attend

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("variant", ["loop", "reduce"])
@pytest.mark.parametrize("cache", ["e4m3", "e5m2"])
@pytest.mark.parametrize("hk,group,d,bs", [(4, 2, 128, 16), (2, 4, 64, 64), (1, 3, 128, 32), (8, 2, 64, 16), (4, 1, 64, 64)])
def test_spread_out_contexts(cuda_device, variant, cache, hk, group, d, bs):
    """V values of about 1, 0.1 and 0.001; the bound has no term for the codes' size (max|v| carries it)."""
    for size in (1.0, 0.1, 1e-3):
        case = paged_case(70 + hk, [1, 700, 2049, 33, 0], hk * group, hk, d, bs, cache=cache, spread=4.0)
        case["v_scale"] *= size
        got = attend("fp8", variant, case, cuda_device, k_scale_per_block=case["k_scale"], v_scale_per_block=case["v_scale"])
        check(got, *attention64(case, case["k_scale"], case["v_scale"]), f"{cache} {variant} values of {size}")


def test_wide_launch_gives_the_bits_of_the_narrow_one(cuda_device):
    case = paged_case(80, [1024] * 160, 8, 8, 64, 64, cache="e5m2", spread=3.0)
    kw = lambda c: dict(k_scale_per_block=c["k_scale"], v_scale_per_block=c["v_scale"])
    batch = attend("fp8", "reduce", case, cuda_device, **kw(case))
    one = {**case, "query": case["query"][7:8], "block_tables": case["block_tables"][7:8], "context_lens": case["context_lens"][7:8]}
    assert torch.equal(attend("fp8", "reduce", one, cuda_device, **kw(one))[0], batch[7])
    some = {**case, "query": case["query"][:6], "block_tables": case["block_tables"][:6], "context_lens": case["context_lens"][:6]}
    want, tol = attention64(some, case["k_scale"], case["v_scale"])
    check(batch[:6], want, tol, "wide launch")


@pytest.mark.parametrize("variant", ["loop", "reduce"])
@pytest.mark.parametrize("cache", ["e4m3", "e5m2"])
@pytest.mark.parametrize("hk,d,bs", [(4, 128, 16), (2, 64, 64), (8, 64, 16)])
def test_negative_scales(cuda_device, variant, cache, hk, d, bs):
    """A block's FP8 scales are factors of any sign: V negative throughout, or in some blocks; K in some."""
    case = paged_case(90 + hk, [1, 700, 2049, 33], 2 * hk, hk, d, bs, cache=cache, spread=4.0)
    sizes = {n: case[f"{n}_scale"] for n in "kv"}
    sign = 1.0 - 2.0 * (torch.rand(sizes["v"].shape, generator=torch.Generator().manual_seed(4)) < 0.5)
    for k_sign, v_sign in ((1.0, -1.0), (1.0, sign), (sign.flip(0), sign)):
        case["k_scale"], case["v_scale"] = sizes["k"] * k_sign, sizes["v"] * v_sign
        got = attend("fp8", variant, case, cuda_device, k_scale_per_block=case["k_scale"], v_scale_per_block=case["v_scale"])
        check(got, *attention64(case, case["k_scale"], case["v_scale"]), f"{cache} {variant}")


@pytest.mark.parametrize("hk,group", [(4, 2), (1, 3)])
def test_many_short_sequences(cuda_device, hk, group):
    """Whole-context items of the persistent form, with a warp per head and with warps that share one."""
    lens = torch.randint(0, 90, (700,), generator=torch.Generator().manual_seed(1)).tolist()
    case = paged_case(95, lens, hk * group, hk, 64, 16, cache="e5m2", spread=6.0)
    got = attend("fp8", "loop", case, cuda_device, k_scale_per_block=case["k_scale"], v_scale_per_block=case["v_scale"])
    check(got, *attention64(case, case["k_scale"], case["v_scale"]), f"hk{hk}")


@pytest.mark.parametrize("variant", ["loop", "reduce"])
@pytest.mark.parametrize("cache", ["e4m3", "e5m2"])
def test_what_the_append_stored_is_read_back(cuda_device, variant, cache):
    """append_block_scaled over prompts with values of about 0.1, then attention over the caches and scales it left."""
    from flash_attention_factory_b200.cache_ops import append_block_scaled

    dev, hk, d, bs, lens = cuda_device, 2, 64, 16, [700, 90, 33]
    case = paged_case(81, lens, 8, hk, d, bs, cache=cache)
    g = torch.Generator().manual_seed(9)
    k, v = (torch.randn(sum(lens), hk, d, generator=g).half() for _ in range(2))
    v = (v * 0.1).half()
    x = {n: case[n].to(dev) for n in ("key_cache", "value_cache", "k_scale", "v_scale", "block_tables", "context_lens")}
    append_block_scaled(k.to(dev), v.to(dev), x["key_cache"], x["value_cache"], x["k_scale"], x["v_scale"], x["block_tables"],
                        x["context_lens"], cu_tokens=torch.tensor([0] + lens).cumsum(0).int().to(dev))
    torch.cuda.synchronize(dev)
    case.update({n: t.cpu() for n, t in x.items()})
    got = attend("fp8", variant, case, dev, k_scale_per_block=case["k_scale"], v_scale_per_block=case["v_scale"])
    check(got, *attention64(case, case["k_scale"], case["v_scale"]), f"{cache} {variant}")
