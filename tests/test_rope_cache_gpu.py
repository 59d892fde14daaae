"""rope_and_cache: the rotation against fp64, within half a step of what each row is stored in."""
import pytest
import torch

from _fp64 import cache_values

pytestmark = pytest.mark.gpu

DTYPES = {"fp16": torch.float16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}


def table(max_position, rotary):
    i = torch.arange(rotary // 2, dtype=torch.float64)
    a = torch.arange(max_position, dtype=torch.float64)[:, None] * 10000.0 ** (-2 * i / rotary)
    return torch.cat([a.cos(), a.sin()], 1).float()


def rotated64(x, cos_sin, positions, interleaved):
    """(value, sum of the two products' sizes) in fp64 of rows x [T, heads, D]."""
    r = cos_sin.size(1)
    c, s = cos_sin[positions].double()[:, None].chunk(2, -1)
    y, size = x.double().clone(), x.double().abs()
    ia, ib = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = x.double()[..., ia], x.double()[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    size[..., ia] = size[..., ib] = a.abs() + b.abs()
    return y, size


def half_step(x, size, cache, scale):
    """Largest rounding error of x in the cache's type: half a step relative (fp16 2^-11, e4m3 2^-4, e5m2
    2^-3; int8 half a code) or half a subnormal step, plus three fp32 roundings of the rotation and one of
    the division, each 2^-24 of the sizes involved."""
    rel, low = {"fp16": (2.0 ** -11, 2.0 ** -25), "e4m3": (2.0 ** -4, scale * 2.0 ** -10),
                "e5m2": (2.0 ** -3, scale * 2.0 ** -17), "int8": (0.0, scale * 0.5)}[cache]
    return rel * x.abs() + low + 4 * 2.0 ** -24 * size


def case(seed, t, h, hk, d, rotary, bs, cache, scales, nb=None, strided=True, max_position=400):
    g = torch.Generator().manual_seed(seed)
    nb = nb or -(-t // bs) + 2
    qkv = torch.randn(t, h + 2 * hk, d, generator=g).half()
    q, k, v = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
    if not strided:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    kc = torch.randint(-100, 100, (nb, bs, hk, d), generator=g).to(DTYPES[cache])
    qmax = {"fp16": 1.0, "int8": 127.0, "e4m3": 448.0, "e5m2": 57344.0}[cache]
    base = 6.5 / qmax  # |rotated| <= sqrt(2) * 4.6
    shape = {"none": (), "scalar": (), "head": (hk,), "block": (nb, hk)}[scales]
    ks, vs = (base * (1 + torch.rand(shape, generator=g)) for _ in range(2))
    if scales == "scalar":
        vs = ks
    slots = torch.randperm(nb * bs, generator=g)[:t]
    positions = torch.randint(0, max_position, (t,), generator=g)
    return dict(q=q, k=k, v=v, kc=kc, vc=kc.flip(0).contiguous(), ks=ks, vs=vs, slots=slots, positions=positions,
                table=table(max_position, rotary), cache=cache, scales=scales, bs=bs, h=h)


def scale_kw(c, dev):
    if c["scales"] == "scalar":
        return dict(fp8_scale=float(c["ks"]))
    if c["scales"] == "none":
        return {}
    return {f"{n}_scale_per_{c['scales']}": c[f"{n}s"].to(dev) for n in "kv"}


def verify(c, got_q, got_k, got_v, interleaved, skipped=(), q_fill=7.0, queries=True):
    t = c["k"].size(0)
    live = torch.tensor([i for i in range(t) if i not in set(skipped)], dtype=torch.long)
    pos, slot = c["positions"][live], c["slots"][live]
    if queries:
        want, size = rotated64(c["q"][live], c["table"], pos, interleaved)
        off = (got_q.cpu()[live].double() - want).abs() - half_step(want, size, "fp16", 1.0)
        assert (off <= 0).all(), f"queries: {off.max()}"
        rest = torch.ones(t, dtype=torch.bool)
        rest[live] = False
        assert (got_q.cpu()[rest] == q_fill).all(), "a skipped token's query row was written"
    for got, before, x, s, turn in ((got_k, c["kc"], c["k"], c["ks"], True), (got_v, c["vc"], c["v"], c["vs"], False)):
        got = got.cpu()
        want, size = rotated64(x[live], c["table"], pos, interleaved) if turn else (x[live].double(), torch.zeros(1))
        per = s[slot // c["bs"]][:, :, None] if s.dim() == 2 else s[:, None] if s.dim() == 1 else s
        per = per.double() if c["cache"] != "fp16" else torch.ones(()).double()
        rows = cache_values(got.view(1, -1, *got.shape[2:]))[0][slot] * per
        off = (rows - want).abs() - half_step(want, size, c["cache"], per)
        assert (off <= 0).all(), f"{'K' if turn else 'V'}: {off.max()}"
        bits = torch.int16 if c["cache"] == "fp16" else torch.uint8
        untouched = torch.ones(got.size(0) * got.size(1), dtype=torch.bool)
        untouched[slot] = False
        assert torch.equal(got.view(bits).flatten(0, 1)[untouched], before.view(bits).flatten(0, 1)[untouched])


def call(c, dev, interleaved, q_out=None, queries=True):
    from flash_attention_factory_b200.cache_ops import rope_and_cache

    kc, vc = c["kc"].to(dev), c["vc"].to(dev)
    base = torch.cat([c["q"], c["k"], c["v"]], dim=1).to(dev) if not c["k"].is_contiguous() else None
    h, hk = c["h"], c["k"].size(1)
    q, k, v = ((base[:, :h], base[:, h:h + hk], base[:, h + hk:]) if base is not None
               else (c["q"].to(dev), c["k"].to(dev), c["v"].to(dev)))
    out = torch.full(c["q"].shape, 7.0, dtype=torch.float16, device=dev) if q_out is None else q_out
    kw = scale_kw(c, dev)
    rope_and_cache(q if queries else None, k, v, c["positions"].to(dev), c["table"].to(dev), out if queries else None,
                   kc, vc, c["slots"].to(dev), interleaved=interleaved, **kw)
    torch.cuda.synchronize(dev)
    return out, kc, vc


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("cache,scales", [("fp16", "none"), ("int8", "block"), ("int8", "scalar"), ("e4m3", "head"),
                                          ("e5m2", "block"), ("e4m3", "scalar")])
@pytest.mark.parametrize("t,h,hk,d,rotary,bs", [(1, 32, 8, 128, 128, 16), (37, 40, 8, 64, 32, 64), (131, 6, 3, 80, 16, 16),
                                                (5, 1, 1, 16, 16, 128), (70, 7, 7, 48, 48, 32), (3, 4, 2, 512, 256, 16)])
def test_rotated_append(cuda_device, interleaved, cache, scales, t, h, hk, d, rotary, bs):
    c = case(t * 7 + d, t, h, hk, d, rotary, bs, cache, scales, strided=t % 2 == 1)
    verify(c, *call(c, cuda_device, interleaved), interleaved)


def test_skipped_tokens_leave_their_rows(cuda_device):
    """Negative slots, slots behind the cache and positions outside the table: nothing of the token is written."""
    c = case(3, 50, 4, 2, 64, 64, 16, "int8", "head")
    nslots = c["kc"].size(0) * 16
    c["slots"][[4, 49]] = -1
    c["slots"][7], c["slots"][8] = nslots, 2 ** 62
    c["positions"][10], c["positions"][11], c["positions"][12] = -1, 400, 2 ** 40
    verify(c, *call(c, cuda_device, False), False, skipped=(4, 7, 8, 10, 11, 12, 49))


@pytest.mark.parametrize("cache,largest", [("int8", 127.0), ("e4m3", 448.0), ("e5m2", 57344.0)])
@pytest.mark.parametrize("scales", ["scalar", "head", "block"])
def test_infinities_saturate(cuda_device, cache, largest, scales):
    """An infinity over a finite scale is an infinity, and a cache stores that as its largest code, in V, in the
    unrotated and in the rotated dims of K (a' = inf cos, b' = inf sin); the values beside it are as ever."""
    c = case(11, 9, 2, 2, 64, 32, 16, cache, scales, strided=False)
    clean = call(c, cuda_device, False)
    inf = float("inf")
    c["positions"][:] = 1  # cos and sin of every angle are positive
    c["v"][3, 1, 7], c["v"][3, 1, 8], c["v"][4, 0, 63] = inf, -inf, inf
    c["k"][5, 0, 40], c["k"][6, 1, 33] = -inf, inf
    c["k"][7, 1, 2] = inf
    _, kc, vc = call(c, cuda_device, False)
    k, v = (cache_values(x.cpu().view(1, -1, 2, 64))[0][c["slots"]] for x in (kc, vc))
    before = cache_values(clean[2].cpu().view(1, -1, 2, 64))[0][c["slots"]]
    assert [v[3, 1, 7], v[3, 1, 8], v[4, 0, 63]] == [largest, -largest, largest]
    assert [k[5, 0, 40], k[6, 1, 33], k[7, 1, 2], k[7, 1, 18]] == [-largest, largest, largest, largest]
    same = c["v"].isfinite()
    assert torch.equal(v[same], before[same])


def test_without_queries_and_in_place(cuda_device):
    c = case(4, 33, 4, 2, 128, 128, 16, "fp16", "none", strided=False)
    out, kc, vc = call(c, cuda_device, False, queries=False)
    verify(c, None, kc, vc, False, queries=False)
    from flash_attention_factory_b200.cache_ops import rope_and_cache

    q, kc, vc = c["q"].to(cuda_device), c["kc"].to(cuda_device), c["vc"].to(cuda_device)
    rope_and_cache(q, c["k"].to(cuda_device), c["v"].to(cuda_device), c["positions"].to(cuda_device), c["table"].to(cuda_device),
                   q, kc, vc, c["slots"].to(cuda_device))
    verify(c, q, kc, vc, False)


def test_prefill_sized_call_and_far_slots(cuda_device):
    """More than 4096 tokens (the plain launch), into a cache whose last rows lie behind 2^31 elements."""
    t, hk, d, bs = 4500, 8, 128, 16
    c = case(5, t, 8, hk, d, 128, bs, "fp16", "none")
    verify(c, *call(c, cuda_device, False), False)
    nb = (2 ** 31 // (bs * hk * d)) + 4
    c = case(6, 9, 8, hk, d, 128, bs, "int8", "scalar")
    kc = torch.zeros(nb, bs, hk, d, dtype=torch.int8, device=cuda_device)
    vc = torch.zeros_like(kc)
    from flash_attention_factory_b200.cache_ops import rope_and_cache

    slots = torch.arange(nb * bs - 9, nb * bs, device=cuda_device)
    q_out = torch.zeros(9, 8, d, dtype=torch.float16, device=cuda_device)
    rope_and_cache(c["q"].to(cuda_device), c["k"].to(cuda_device), c["v"].to(cuda_device), c["positions"].to(cuda_device),
                   c["table"].to(cuda_device), q_out, kc, vc, slots, float(c["ks"]))
    tail = dict(c, slots=torch.arange(9), kc=torch.zeros(1, 16, hk, d, dtype=torch.int8), vc=torch.zeros(1, 16, hk, d, dtype=torch.int8))
    pad = torch.zeros(7, hk, d, dtype=torch.int8)
    verify(tail, q_out, torch.cat([kc.view(-1, hk, d)[-9:].cpu(), pad])[None], torch.cat([vc.view(-1, hk, d)[-9:].cpu(), pad])[None], False)
    assert int(kc[:-1].count_nonzero()) == 0


def test_graph_and_side_stream(cuda_device):
    from flash_attention_factory_b200.cache_ops import rope_and_cache

    c = case(8, 20, 8, 2, 64, 64, 16, "e4m3", "block")
    dev = cuda_device
    args = [c["q"].to(dev).contiguous(), c["k"].to(dev).contiguous(), c["v"].to(dev).contiguous(), c["positions"].to(dev),
            c["table"].to(dev), torch.full((20, 8, 64), 7.0, dtype=torch.float16, device=dev), c["kc"].to(dev), c["vc"].to(dev),
            c["slots"].to(dev)]
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    kw = scale_kw(c, dev)
    with torch.cuda.stream(side):
        rope_and_cache(*args, **kw)
    side.synchronize()
    verify(c, *args[5:8], False)
    args[6].view(torch.uint8).zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rope_and_cache(*args, **kw)
    args[0].copy_(args[0].flip(0))
    graph.replay()
    torch.cuda.synchronize(dev)
    verify(dict(c, q=c["q"].flip(0), kc=torch.zeros_like(c["kc"].view(torch.uint8)).view(c["kc"].dtype)), *args[5:8], False)
