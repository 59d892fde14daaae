"""The second part of the weights: int8 and differential attention err by the rounding of their result alone.

The RMS error against fp64 is compared with e0, that of rounding the exact result to fp16.  Weights rounded once to fp16
add errors of p_t v_t whose RMS is that rounding relative to |o| for values of random sign (sum p_t^2 v_t^2 is then
o^2 on average), in every one of the two maps of differential attention: sqrt(2) e0 together, sqrt(3) e0 there.  With the
second part what is left is fp32 arithmetic, 2^-20 of the weights at most.  1.2 e0 separates the two."""
import pytest
import torch

import test_differential_attention_gpu as diff
from _fp64 import attention64, paged_case
from test_zero_head_scales_gpu import attend

pytestmark = pytest.mark.gpu
LENS = [1500, 700, 2049, 330, 1024, 999]


def rms(x):
    return float(x.double().square().mean().sqrt())


def assert_only_the_result_is_rounded(got, want):
    e0 = rms(want.half().double() - want)
    assert rms(got.double() - want) <= 1.2 * e0, (rms(got.double() - want) / e0)


@pytest.mark.parametrize("variant,partials", [("loop", torch.float16), ("reduce", torch.float32)])
@pytest.mark.parametrize("kind", ["block", "head"])
@pytest.mark.parametrize("hk,group,d,bs", [(8, 4, 128, 16), (4, 5, 64, 64), (2, 4, 128, 32), (1, 8, 64, 128)])
def test_int8(cuda_device, variant, partials, kind, hk, group, d, bs):
    case = paged_case(220 + hk, LENS, hk * group, hk, d, bs, scale=kind, spread=2.0)
    kw = {f"{n}_scale_per_{kind}": case[f"{n}_scale"] for n in "kv"}
    want, _ = attention64(case, case["k_scale"], case["v_scale"])
    assert_only_the_result_is_rounded(attend("int8", variant, case, cuda_device, partials, **kw), want)


@pytest.mark.parametrize("cache,scale", [("fp16", "none"), ("e4m3", "block"), ("e4m3", "head"), ("e5m2", "block"), ("int8", "block")])
@pytest.mark.parametrize("pairs,group,d,bs", [(4, 4, 128, 16), (1, 8, 64, 128), (3, 2, 64, 32)])
def test_differential(cuda_device, cache, scale, pairs, group, d, bs):
    case = paged_case(230 + pairs, LENS, 2 * pairs * group, 2 * pairs, d, bs, cache=cache, scale=scale, spread=2.0)
    lam = torch.full((pairs * group,), 0.8)
    want, _ = diff.reference(case, lam)
    assert_only_the_result_is_rounded(diff.run(case, cuda_device, lam), want)
