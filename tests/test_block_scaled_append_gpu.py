"""append_block_scaled: scales and codes against the definition evaluated operation by operation in fp32
(the same bits), and the stored values against the rows in fp64."""
import pytest
import torch

from _fp64 import attention64, cache_values, check
from test_rope_cache_gpu import DTYPES, half_step, rotated64, table

pytestmark = pytest.mark.gpu
QMAX = {"int8": 127.0, "e4m3": 448.0, "e5m2": 57344.0}


def encode(x, cache):
    x = x.clamp(-QMAX[cache], QMAX[cache])
    return x.nan_to_num(0.0).round().to(torch.int8) if cache == "int8" else x.to(DTYPES[cache])


def rotate32(x, cos_sin, positions, interleaved):
    r = cos_sin.size(1)
    c, s = cos_sin[positions][:, None].chunk(2, -1)
    y = x.float().clone()
    ia, ib = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = x.float()[..., ia], x.float()[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    return y


def bits(t):
    return t.view(torch.uint8)


def reference(c):
    """Caches, scales and rotated queries after the append, by loops over sequences and blocks."""
    cache, bs = c["cache"], c["bs"]
    kc, vc, ks, vs = c["kc"].clone(), c["vc"].clone(), c["ks"].clone(), c["vs"].clone()
    qo = torch.full(c["q"].shape, 7.0).half() if c["q"] is not None else None
    limit = c["bt"].size(1) * bs
    if c["table"] is not None:
        limit = min(limit, c["table"].size(0))
    start = 0
    for i, (ctx, n) in enumerate(zip(c["ctx"].tolist(), c["new"])):
        pos = torch.arange(ctx - n, ctx)
        live = [j for j in range(n) if 0 <= ctx - n + j < limit and 0 <= int(c["bt"][i, (ctx - n + j) // bs]) < kc.size(0)]
        k, v = c["k"][start:start + n].float(), c["v"][start:start + n].float()
        k, v = (x.nan_to_num(float("nan"), 65504.0, -65504.0) for x in (k, v))
        if c["table"] is not None and live:
            k[live] = rotate32(k[live], c["table"], pos[live], c["interleaved"])
            if qo is not None:
                rows = [start + j for j in live]
                qo[rows] = rotate32(c["q"][rows], c["table"], pos[live], c["interleaved"]).half()
        j = 0
        while j < n:
            if j not in live:
                j += 1
                continue
            p = int(pos[j])
            block, r0 = int(c["bt"][i, p // bs]), p % bs
            m = 1
            while j + m < n and (j + m) in live and (p + m) // bs == p // bs:
                m += 1
            for x, pool, scale in ((k, kc, ks), (v, vc, vs)):
                rows = x[j:j + m]
                top = rows.abs().nan_to_num(0.0).amax((0, 2)) / torch.tensor(QMAX[cache])
                held = scale[block].clone() if r0 else torch.zeros_like(top)
                s = torch.maximum(held, top)
                by = torch.where(s > 0, s, torch.ones_like(s))[:, None]
                grown = (s > held)[:, None]
                if r0:
                    again = encode(pool[block, :r0].float() * held[:, None] / by, cache)
                    bits(pool)[block, :r0] = torch.where(grown, bits(again), bits(pool)[block, :r0])
                bits(pool)[block, r0:r0 + m] = bits(encode(rows / by, cache))
                scale[block] = s
            j += m
        start += n
    return kc, vc, ks, vs, qo


def make(seed, old, new, hk, d, bs, cache, rotary=0, h=0, interleaved=False, extra_rows=0, one_each=False):
    g = torch.Generator().manual_seed(seed)
    ctx = [o + n for o, n in zip(old, new)]
    counts = [-(-n // bs) for n in ctx]
    nb, mb = sum(counts) + 2, max(1, max(counts))
    perm = torch.randperm(nb, generator=g).int()
    bt = torch.zeros(len(old), mb, dtype=torch.int32)
    at = 0
    for i, n in enumerate(counts):
        bt[i, :n] = perm[at:at + n]
        at += n
    t = sum(new) + extra_rows
    size = 2.0 ** (torch.rand(t, 1, 1, generator=g) * 4 - 2)  # rows of different size, so that scales grow
    qkv = torch.randn(t, h + 2 * hk, d, generator=g) * size
    pools = [(torch.randint(-100, 101, (nb, bs, hk, d), generator=g)).float().to(DTYPES[cache]) for _ in range(2)]
    scales = [torch.rand(nb, hk, generator=g) * 4 / QMAX[cache] for _ in range(2)]
    return dict(q=qkv[:, :h].half() if h else None, k=qkv[:, h:h + hk].half(), v=qkv[:, h + hk:].half(), kc=pools[0],
                vc=pools[1], ks=scales[0], vs=scales[1], bt=bt, ctx=torch.tensor(ctx, dtype=torch.int32), new=list(new),
                table=table(4096, rotary) if rotary else None, cache=cache, bs=bs, interleaved=interleaved, one_each=one_each)


def run(c, dev, on_device=None):
    from flash_attention_factory_b200.cache_ops import append_block_scaled

    x = {n: c[n].to(dev) if torch.is_tensor(c[n]) else c[n] for n in c}
    cu = torch.tensor([0] + c["new"]).cumsum(0).int().to(dev)
    h = 0 if c["q"] is None else c["q"].size(1)
    both = torch.cat([x["q"], x["k"], x["v"]], 1) if h else torch.cat([x["k"], x["v"]], 1)  # slices of one tensor
    hk = c["k"].size(1)
    qo = torch.full(c["q"].shape, 7.0, dtype=torch.float16, device=dev) if h else None
    append_block_scaled(both[:, h:h + hk], both[:, h + hk:], x["kc"], x["vc"], x["ks"], x["vs"], x["bt"], x["ctx"],
                        cu_tokens=None if c["one_each"] else cu, query=both[:, :h] if h else None, query_out=qo,
                        cos_sin=x["table"], interleaved=c["interleaved"])
    torch.cuda.synchronize(dev)
    return x["kc"].cpu(), x["vc"].cpu(), x["ks"].cpu(), x["vs"].cpu(), qo.cpu() if h else None


def compare(got, want):
    for name, a, b in zip(("key scales", "value scales"), got[2:4], want[2:4]):
        assert torch.equal(a.view(torch.int32), b.view(torch.int32)), f"{name}: {int((a != b).sum())} differ"
    for name, a, b in zip(("key cache", "value cache"), got[:2], want[:2]):
        assert torch.equal(bits(a), bits(b)), f"{name}: {int((bits(a) != bits(b)).sum())} codes differ"
    if want[4] is not None:
        assert torch.equal(got[4].view(torch.int16), want[4].view(torch.int16)), "queries differ"


OLD = [0, 15, 16, 40, 1, 0, 255, 7, 64]
NEW = [1, 3, 0, 17, 64, 5, 300, 1, 1]


@pytest.mark.parametrize("cache", ["int8", "e4m3", "e5m2"])
@pytest.mark.parametrize("hk,d,bs,rotary,h,interleaved", [(8, 128, 16, 128, 8, False), (3, 64, 64, 32, 9, True), (1, 80, 32, 0, 0, False),
                                                          (2, 128, 128, 0, 0, False), (16, 16, 16, 16, 16, True), (1, 512, 16, 256, 2, False)])
def test_ragged_append_gives_the_defined_bits(cuda_device, cache, hk, d, bs, rotary, h, interleaved):
    c = make(hk + d + bs, OLD, NEW, hk, d, bs, cache, rotary, h, interleaved)
    compare(run(c, cuda_device), reference(c))


@pytest.mark.parametrize("cache", ["int8", "e4m3"])
def test_one_token_each(cuda_device, cache):
    old = list(range(0, 70))
    c = make(4, old, [1] * len(old), 8, 128, 16, cache, 128, 32, one_each=True)
    compare(run(c, cuda_device), reference(c))


@pytest.mark.parametrize("cache", ["int8", "e4m3", "e5m2"])
def test_stored_values_are_within_half_a_step(cuda_device, cache):
    """Fresh blocks: every stored value is its (rotated) row's within half a step of the block's scale."""
    new = [100, 33, 1]
    c = make(9, [0, 0, 0], new, 4, 64, 16, cache, 64)
    kc, vc, ks, vs, _ = run(c, cuda_device)
    start = 0
    for i, n in enumerate(new):
        pos = torch.arange(n)
        at = c["bt"][i, pos // 16].long()
        for x, pool, scale, turn in ((c["k"], kc, ks, True), (c["v"], vc, vs, False)):
            rows = x[start:start + n]
            want, size = rotated64(rows, c["table"], pos, False) if turn else (rows.double(), rows.double().abs())
            per = scale[at].double()[..., None]
            got = cache_values(pool)[at, pos % 16] * per
            # the block's largest value may lie a rounding beyond the last code: 2^-22 of it
            off = (got - want).abs() - half_step(want, size, cache, per) - per * QMAX[cache] * 2.0 ** -22
            assert (off <= 0).all()
        start += n


def test_special_values(cuda_device):
    """Rows of zeros (scale 0, codes 0, no NaN), infinities (the largest fp16 value), NaNs (not counted)."""
    c = make(5, [0, 3, 16, 5], [16, 2, 4, 1], 2, 64, 16, "int8")
    c["k"][:16] = 0
    c["v"][:16] = 0
    c["k"][16, 0, 3], c["v"][17, 1, 5] = float("inf"), -float("inf")
    c["k"][18, 0, 9] = float("nan")
    c["ks"][c["bt"][3, 0]] = 0.0  # a block of zeros that gets its first values
    c["kc"][c["bt"][3, 0]] = 0
    got, want = run(c, cuda_device), reference(c)
    compare(got, want)
    assert (got[2][int(c["bt"][0, 0])] == 0).all() and (got[0][int(c["bt"][0, 0])] == 0).all()
    assert float(got[2].max()) == pytest.approx(65504 / 127)


def test_padding_and_tokens_out_of_range_are_skipped(cuda_device):
    """Rows behind the last sequence; a context shorter than its new tokens, or longer than its table row or
    than the rotation table; block ids outside the cache."""
    c = make(6, [10, 20, 0, 30], [8, 9, 12, 4], 2, 64, 16, "e4m3", 64, 4, extra_rows=5)
    c["ctx"][2] = 7                                   # five of its 12 tokens have negative positions
    c["ctx"][0] += 16 * c["bt"].size(1)               # wholly behind its table row
    c["bt"][3, 30 // 16] = c["kc"].size(0) + 3        # two of its tokens land in a block that does not exist
    c["table"] = c["table"][:26]                      # sequence 1 reaches position 28
    compare(run(c, cuda_device), reference(c))


def test_repeated_appends_and_graph_replay(cuda_device):
    """Token by token over a block: the scale never falls, and a captured step replays on new inputs."""
    from flash_attention_factory_b200.cache_ops import append_block_scaled

    dev = cuda_device
    c = make(7, [0, 5], [1, 1], 2, 64, 16, "int8", one_each=True)
    x = {n: c[n].to(dev) for n in ("k", "v", "kc", "vc", "ks", "vs", "bt", "ctx")}
    x["k"], x["v"] = x["k"].contiguous(), x["v"].contiguous()
    args = [x[n] for n in ("k", "v", "kc", "vc", "ks", "vs", "bt", "ctx")]
    g = torch.Generator().manual_seed(1)
    graph = None
    for step in range(10):
        k, v = (torch.randn(2, 2, 64, generator=g).half() * (step + 1) ** 0.5 for _ in range(2))
        ctx = torch.tensor([1 + step, 6 + step], dtype=torch.int32)
        ref = dict(c, k=k, v=v, ctx=ctx, kc=x["kc"].cpu(), vc=x["vc"].cpu(), ks=x["ks"].cpu(), vs=x["vs"].cpu())
        x["k"].copy_(k)
        x["v"].copy_(v)
        x["ctx"].copy_(ctx)
        if graph is None and step == 3:
            torch.cuda.synchronize(dev)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                append_block_scaled(*args)
        if graph is not None:
            graph.replay()
        else:
            append_block_scaled(*args)
        torch.cuda.synchronize(dev)
        want = reference(ref)
        compare([x["kc"].cpu(), x["vc"].cpu(), x["ks"].cpu(), x["vs"].cpu(), None], want)


@pytest.mark.parametrize("cache", ["int8", "e4m3"])
def test_decode_steps_with_attention(cuda_device, cache):
    """Prompt, then decode steps: append with rotation and queries, then attention over what was stored."""
    from flash_attention_factory_b200 import lib
    from flash_attention_factory_b200.cache_ops import append_block_scaled

    dev, h, hk, d, bs = cuda_device, 8, 2, 64, 16
    old, steps = [40, 3, 0], 4
    c = make(11, [0] * 3, [o + steps for o in old], hk, d, bs, cache, d, h)
    x = {n: c[n].to(dev) for n in ("kc", "vc", "ks", "vs", "bt", "table")}
    prompt = [i for i, n in enumerate(c["new"]) for _ in range(n)]
    rows = torch.arange(len(prompt))
    starts = torch.tensor([0] + c["new"]).cumsum(0)
    pick = torch.cat([rows[starts[i]:starts[i] + o] for i, o in enumerate(old)])
    cu = torch.tensor([0] + old).cumsum(0).int().to(dev)
    append_block_scaled(c["k"][pick].to(dev), c["v"][pick].to(dev), x["kc"], x["vc"], x["ks"], x["vs"], x["bt"],
                        torch.tensor(old, dtype=torch.int32, device=dev), cu_tokens=cu, cos_sin=x["table"])
    module = lib.paged_attention_int8_reduce if cache == "int8" else lib.paged_attention_fp8_reduce
    for step in range(steps):
        ctx = torch.tensor([o + step + 1 for o in old], dtype=torch.int32)
        now = starts[:3] + torch.tensor(old) + step
        q, k, v = (c[n][now].to(dev) for n in "qkv")
        qo, out = torch.empty_like(q), torch.full((3, h, d), float("nan"), dtype=torch.float16, device=dev)
        append_block_scaled(k, v, x["kc"], x["vc"], x["ks"], x["vs"], x["bt"], ctx.to(dev), query=q, query_out=qo, cos_sin=x["table"])
        ml = torch.empty(3, h, 1, device=dev)
        module.enqueue(ml, ml.clone(), torch.empty(3, h, 1, d, dtype=torch.float16, device=dev), out, None, qo, x["kc"], x["vc"],
                       x["bt"], ctx.to(dev), h // hk, d ** -0.5, 1.0, bs, int(ctx.max()), torch.ones(h, device=dev), None, -1.0,
                       k_scale_per_block=x["ks"], v_scale_per_block=x["vs"])
        torch.cuda.synchronize(dev)
        held = dict(query=qo.cpu(), key_cache=x["kc"].cpu(), value_cache=x["vc"].cpu(), block_tables=c["bt"], context_lens=ctx,
                    sm_scale=d ** -0.5)
        # the e4m3 operator folds a block's scale into the weights before they are rounded: one output in
        # 1536 was 9.2e-6 off where two tokens, a weight of 1e-4 and a scale of 0.009 meet (bound 2 * 2^-25 * 448 = 2.7e-5)
        want, tol = attention64(held, x["ks"].cpu(), x["vs"].cpu(), weighted_code=0.0 if cache == "int8" else 448.0)
        check(out, want, tol, f"step {step}")
        turned, size = rotated64(c["q"][now], c["table"], ctx.long() - 1, False)
        assert ((qo.cpu().double() - turned).abs() <= half_step(turned, size, "fp16", 1.0)).all()


@pytest.mark.parametrize("seqs", [31, 32, 33, 500, 1000])
def test_many_sequences(cuda_device, seqs):
    """The search for a token's sequence: 31 is the last count that needs no memory, sequences without tokens among them."""
    g = torch.Generator().manual_seed(seqs)
    old = torch.randint(0, 40, (seqs,), generator=g).tolist()
    new = torch.randint(0, 4, (seqs,), generator=g).tolist()
    new[0], new[-1] = 0, 0
    c = make(seqs, old, new, 1, 16, 16, "int8", extra_rows=3)
    compare(run(c, cuda_device), reference(c))


def test_nothing_to_append(cuda_device):
    """No rows, and sequences of which none has a new token: caches and scales stay."""
    for rows in (0, 4):
        c = make(3, [5, 9], [0, 0], 2, 64, 16, "e4m3", extra_rows=rows)
        compare(run(c, cuda_device), reference(c))


def test_torch_ops_of_a_step(cuda_device):
    """The registered operators run a decode step: append with rotation, then attention; rope_and_cache and diff too."""
    import flash_attention_factory_b200.torch_ops  # noqa: F401
    from flash_attention_factory_b200.lib import paged_attention_diff

    dev = cuda_device
    c = make(21, [33, 7], [1, 1], 4, 64, 16, "int8", 64, 8, one_each=True)
    x = {n: c[n].to(dev).contiguous() for n in ("q", "k", "v", "kc", "vc", "ks", "vs", "bt", "ctx", "table")}
    qo = torch.empty_like(x["q"])
    ops = torch.ops.paged_attention_b200
    ops.append_block_scaled(x["k"], x["v"], x["kc"], x["vc"], x["ks"], x["vs"], x["bt"], x["ctx"], None, x["q"], qo, x["table"])
    torch.cuda.synchronize(dev)
    compare([x["kc"].cpu(), x["vc"].cpu(), x["ks"].cpu(), x["vs"].cpu(), qo.cpu()], reference(c))
    lam = torch.full((4,), 0.4, device=dev)
    out = [torch.empty(2, 4, 128, dtype=torch.float16, device=dev) for _ in range(2)]
    args = (qo, x["kc"], x["vc"], x["bt"], x["ctx"], lam, 0.125, 1.0, 16, 34)
    sc = paged_attention_diff.scratch(qo, x["kc"], 34)
    ops.diff(*sc, out[0], *args, k_scale_per_block=x["ks"], v_scale_per_block=x["vs"])
    paged_attention_diff.enqueue(*sc, out[1], *args, k_scale_per_block=x["ks"], v_scale_per_block=x["vs"])
    assert torch.equal(out[0], out[1])
    from flash_attention_factory_b200 import cache_ops

    slots = torch.tensor([3, 40], device=dev)
    pos = torch.tensor([9, 100], device=dev)
    sides = []
    for fn in (ops.rope_and_cache, cache_ops.rope_and_cache):
        kc, vc, q = torch.zeros(4, 16, 4, 64, dtype=torch.float16, device=dev), torch.zeros(4, 16, 4, 64, dtype=torch.float16, device=dev), torch.empty_like(qo)
        fn(x["q"], x["k"], x["v"], pos, x["table"], q, kc, vc, slots)
        sides.append((kc, vc, q))
    assert all(torch.equal(a, b) for a, b in zip(*sides)) and int(sides[0][0].count_nonzero()) > 0
