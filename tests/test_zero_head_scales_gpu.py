"""A per-head scale of 0 is a head of zeros: K of zeros weighs every token alike, V of zeros gives zeros."""
import pytest
import torch

import test_differential_attention_gpu as diff
from _fp64 import attention64, check, paged_case, to

pytestmark = pytest.mark.gpu


def attend(family, variant, case, device, tmp_dtype=torch.float16, **kw):
    """out of paged_attention_{family}_{variant}; kw: scale arrays."""
    from flash_attention_factory_b200 import lib

    c = to(case, device)
    s, h, d = c["query"].shape
    longest = int(case["context_lens"].max())
    npart = max(1, -(-longest // (512 if d == 128 else 256)))
    ml = torch.full((s, h, npart), float("nan"), device=device)
    tmp = torch.full((s, h, npart, d), float("nan"), dtype=tmp_dtype, device=device)
    out = torch.full((s, h, d), float("nan"), dtype=torch.float16, device=device)
    getattr(lib, f"paged_attention_{family}_{variant}").enqueue(
        ml, ml.clone(), tmp, out, None, c["query"], c["key_cache"], c["value_cache"], c["block_tables"], c["context_lens"],
        h // c["key_cache"].size(2), case["sm_scale"], 1.0, case["block_size"], longest, torch.ones(h, device=device), None, -1.0,
        **{k: v.to(device) for k, v in kw.items()})
    torch.cuda.synchronize(device)
    return out.cpu()


LENS = [1, 17, 700, 0, 64, 1025]


def zeroed(case):
    """The first K scale and the last V scale are 0 (the codes stay: their values are 0 all the same)."""
    case["k_scale"][0] = 0.0
    case["v_scale"][-1] = 0.0
    return case


@pytest.mark.parametrize("variant", ["loop", "reduce"])
@pytest.mark.parametrize("family,cache", [("int8", "int8"), ("fp8", "e4m3"), ("fp8", "e5m2")])
@pytest.mark.parametrize("hk,group,d,bs", [(4, 2, 128, 16), (2, 3, 64, 64), (1, 4, 128, 32), (8, 1, 64, 16)])
def test_ordinary_attention(cuda_device, variant, family, cache, hk, group, d, bs):
    case = zeroed(paged_case(50 + hk, LENS, hk * group, hk, d, bs, cache=cache, scale="head"))
    got = attend(family, variant, case, cuda_device, k_scale_per_head=case["k_scale"], v_scale_per_head=case["v_scale"])
    check(got, *attention64(case, case["k_scale"], case["v_scale"]), f"{cache} {variant}")


@pytest.mark.parametrize("cache", ["int8", "e4m3", "e5m2"])
def test_differential_attention(cuda_device, cache):
    case = zeroed(paged_case(60, LENS, 8, 4, 64, 16, cache=cache, scale="head"))
    lam, w = diff.learned(4, 64)
    check(diff.run(case, cuda_device, lam, norm_weight=w), *diff.reference(case, lam, w), cache)
