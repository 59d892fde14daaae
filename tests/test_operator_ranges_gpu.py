"""Allowed calls at the ends of the operators' ranges: prompt-sized calls into 8-bit caches, many decode tokens with a
prompt chunk among them, blocks that lie behind 2^31 elements, other streams, queries rotated in place."""
import pytest
import torch

import test_rope_cache_gpu as rope
from _fp64 import attention64, cache_values, check, paged_case
from test_block_scaled_append_gpu import bits, compare, make, reference, run
from test_zero_head_scales_gpu import attend

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache,scales", [("int8", "block"), ("int8", "head"), ("e4m3", "scalar"), ("e4m3", "block"), ("e5m2", "head")])
@pytest.mark.parametrize("interleaved", [False, True])
def test_prompts_into_8_bit_caches(cuda_device, cache, scales, interleaved):
    """More than 4096 tokens: the launch that is not chained to its neighbours.

    What is rounded to a code is the fp32 quotient x / s, off by 2^-23 of itself at most (one unit in the last place), so a
    value next to the middle of two codes may go either way: a stored value is off by half a step plus 2^-23 |x|, V's too.
    Of 576 000 values of V one lay 9e-9 beyond half a code, where 2^-23 |x| is up to 5e-7."""
    c = rope.case(5, 4500, 3, 2, 64, 32, 16, cache, scales)
    c["slots"][[0, 17, 4499]] = -1
    q, kc, vc = rope.call(c, cuda_device, interleaved)
    live = c["slots"] >= 0
    pos, slot = c["positions"][live], c["slots"][live]
    want, size = rope.rotated64(c["q"][live], c["table"], pos, interleaved)
    assert ((q.cpu()[live].double() - want).abs() <= rope.half_step(want, size, "fp16", 1.0)).all()
    assert (q.cpu()[~live] == 7.0).all()
    for got, before, x, s, turn in ((kc, c["kc"], c["k"], c["ks"], True), (vc, c["vc"], c["v"], c["vs"], False)):
        got = got.cpu()
        want, size = rope.rotated64(x[live], c["table"], pos, interleaved) if turn else (x[live].double(), x[live].double().abs())
        per = (s[slot // c["bs"]][:, :, None] if s.dim() == 2 else s[:, None] if s.dim() == 1 else s).double()
        rows = cache_values(got.view(1, -1, *got.shape[2:]))[0][slot] * per
        assert ((rows - want).abs() <= rope.half_step(want, size, cache, per)).all(), "K" if turn else "V"
        rest = torch.ones(got.size(0) * got.size(1), dtype=torch.bool)
        rest[slot] = False
        assert torch.equal(bits(got).flatten(0, 1)[rest], bits(before).flatten(0, 1)[rest])


@pytest.mark.parametrize("cache", ["int8", "e4m3", "e5m2"])
@pytest.mark.parametrize("hk,d,bs,rotary,h", [(2, 128, 16, 128, 4), (3, 64, 64, 32, 0), (1, 256, 128, 0, 0)])
def test_decode_tokens_with_prompt_chunks_among_them(cuda_device, cache, hk, d, bs, rotary, h):
    """The average of new tokens is about 2 or 3, a block's new rows up to its size."""
    g = torch.Generator().manual_seed(d)
    old = torch.randint(0, 300, (120,), generator=g).tolist()
    new = [1] * 120
    new[7], new[90], new[119] = 200, 3, 65
    c = make(hk + d, old, new, hk, d, bs, cache, rotary, h)
    compare(run(c, cuda_device), reference(c))


def test_append_into_blocks_behind_2_31_elements(cuda_device):
    from flash_attention_factory_b200.cache_ops import append_block_scaled

    dev, hk, d, bs = cuda_device, 8, 128, 16
    c = make(3, [10, 0], [9, 40], hk, d, bs, "int8")
    used = c["kc"].size(0)
    nb = 2 ** 31 // (bs * hk * d) + 2 * used
    first = nb - used
    pools = [torch.zeros(nb, bs, hk, d, dtype=torch.int8, device=dev) for _ in range(2)]
    scales = [torch.zeros(nb, hk, device=dev) for _ in range(2)]
    for t, n in zip(pools + scales, ("kc", "vc", "ks", "vs")):
        t[first:] = c[n].to(dev)
    append_block_scaled(c["k"].to(dev), c["v"].to(dev), *pools, *scales, (c["bt"] + first).to(dev), c["ctx"].to(dev),
                        cu_tokens=torch.tensor([0, 9, 49], dtype=torch.int32, device=dev))
    torch.cuda.synchronize(dev)
    compare([t[first:].cpu() for t in pools + scales] + [None], reference(c))
    assert all(int(t[:first].count_nonzero()) == 0 for t in pools + scales)
    # and attention over them
    case = paged_case(4, [700, 33], 16, hk, d, bs)
    n = case["key_cache"].size(0)
    for t, name in zip(pools + scales, ("key_cache", "value_cache", "k_scale", "v_scale")):
        t[nb - n:] = case[name].to(dev)
    far = dict(case, key_cache=pools[0], value_cache=pools[1], block_tables=case["block_tables"] + (nb - n))
    want, tol = attention64(case, case["k_scale"], case["v_scale"])
    for variant in ("loop", "reduce"):
        check(attend("int8", variant, far, dev, k_scale_per_block=scales[0], v_scale_per_block=scales[1]), want, tol, variant)


def test_append_on_a_side_stream_with_queries_in_place(cuda_device):
    from flash_attention_factory_b200.cache_ops import append_block_scaled

    dev = cuda_device
    c = make(9, [3, 40], [70, 5], 2, 64, 16, "e4m3", 64, 4)
    want = reference(c)
    x = {n: c[n].to(dev).contiguous() for n in ("q", "k", "v", "kc", "vc", "ks", "vs", "bt", "ctx", "table")}
    cu = torch.tensor([0, 70, 75], dtype=torch.int32, device=dev)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        append_block_scaled(x["k"], x["v"], x["kc"], x["vc"], x["ks"], x["vs"], x["bt"], x["ctx"], cu_tokens=cu, query=x["q"],
                            query_out=x["q"], cos_sin=x["table"])
    side.synchronize()
    compare([x[n].cpu() for n in ("kc", "vc", "ks", "vs", "q")], want)


def test_appends_of_two_streams_at_once(cuda_device):
    """Two batches with caches of their own, step after step; each gives the bits of its steps alone."""
    from flash_attention_factory_b200.cache_ops import append_block_scaled

    dev = cuda_device
    cases = [make(20 + i, [0] * 40, [17 + i] * 40, 4, 128, 16, "int8") for i in range(2)]
    xs = [{n: c[n].to(dev) for n in ("k", "v", "kc", "vc", "ks", "vs", "bt", "ctx")} for c in cases]
    cus = [(torch.arange(41, dtype=torch.int32) * (17 + i)).int().to(dev) for i in range(2)]
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    torch.cuda.synchronize(dev)
    for _ in range(5):
        for st, x, cu in zip(streams, xs, cus):
            with torch.cuda.stream(st):
                append_block_scaled(*(x[n] for n in ("k", "v", "kc", "vc", "ks", "vs", "bt", "ctx")), cu_tokens=cu)
    torch.cuda.synchronize(dev)
    for c, x in zip(cases, xs):
        want = reference(c)  # every block starts afresh, so five times gives what once gives
        for name, w in zip(("kc", "vc"), want[:2]):
            assert torch.equal(bits(x[name].cpu()), bits(w))
        assert torch.equal(x["ks"].cpu(), want[2]) and torch.equal(x["vs"].cpu(), want[3])
