"""Differential attention over the paged cache against fp64."""
import ctypes

import pytest
import torch

from _fp64 import HALF, cache_values, check, paged_case, sequence, to

pytestmark = pytest.mark.gpu


def reference(case, lambdas, norm_weight=None, eps=1e-5, norm_scale=1.0):
    """(result, allowed error) [S, H, 2 D].  Per map, a = sum_t p_t |v_t|: weights rounded to fp16 (HALF a), fp32
    chains (below another HALF a), subnormal weights (n 2^-25 max|v|); partial rows are fp32.  The maps' errors add
    with lambda; the norm carries an error e of the row over as e / rms plus the row times |e|_2 / |o|_2; one
    rounding to fp16 at the end."""
    q, bt, lens = case["query"].double(), case["block_tables"], [int(c) for c in case["context_lens"]]
    kv, vv = cache_values(case["key_cache"], case["k_scale"]), cache_values(case["value_cache"], case["v_scale"])
    s, h2, d = q.shape
    h, pairs = h2 // 2, kv.shape[2] // 2
    lam = lambdas.double()[:, None]
    out, tol = torch.zeros(s, h, 2 * d).double(), torch.full((s, h, 2 * d), 2.0 ** -24).double()
    for i, n in enumerate(lens):
        if n == 0:
            continue
        k = sequence(kv, bt[i], n).view(n, pairs, 2, d)
        v = sequence(vv, bt[i], n).reshape(n, pairs, 2 * d)
        p = torch.softmax(torch.einsum("kgcd,tkcd->ckgt", q[i].view(pairs, h // pairs, 2, d), k) * case["sm_scale"], -1)
        o = torch.einsum("ckgt,tke->ckge", p, v).reshape(2, h, 2 * d)
        a = torch.einsum("ckgt,tke->ckge", p, v.abs()).reshape(2, h, 2 * d)
        x = o[0] - lam * o[1]
        e = 2 * HALF * (a[0] + lam.abs() * a[1]) + (1 + lam.abs()) * n * 2.0 ** -25 * v.abs().max()
        if norm_weight is not None:
            r = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
            w = norm_weight.double() * norm_scale
            y = x * r * w
            e = e * r * w.abs() + y.abs() * torch.sqrt(e.square().sum(-1, keepdim=True) / (x.square().sum(-1, keepdim=True) + 2 * d * eps))
            x = y
        out[i] = x
        tol[i] += e * 1.01 + HALF * x.abs()
    return out, tol


def run(case, device, lambdas, npart=None, hint=None, norm_weight=None, eps=1e-5, norm_scale=1.0, fill=float("nan")):
    from flash_attention_factory_b200.lib import paged_attention_diff as diff

    c = to(case, device)
    s, h2, d = c["query"].shape
    max_ctx = int(case["context_lens"].max()) if hint is None else hint
    ml, es, tmp = diff.scratch(c["query"], c["key_cache"], max_ctx)
    if npart is not None:
        ml, es = (torch.empty(s, h2, npart, device=device) for _ in range(2))
        tmp = torch.empty(s, h2, npart, 2 * d, device=device)
    for t in (ml, es, tmp):
        t.fill_(float("nan"))
    out = torch.full((s, h2 // 2, 2 * d), fill, dtype=torch.float16, device=device)
    kw, scale = {}, 1.0
    if torch.is_tensor(case["k_scale"]):
        kind = "block" if case["k_scale"].dim() == 2 else "head"
        kw = {f"{n}_scale_per_{kind}": c[f"{n}_scale"] for n in "kv"}
    elif case["k_scale"] is not None:
        scale = case["k_scale"]
    diff.enqueue(ml, es, tmp, out, c["query"], c["key_cache"], c["value_cache"], c["block_tables"], c["context_lens"],
                 lambdas.to(device), case["sm_scale"], scale, case["block_size"], max_ctx,
                 norm_weight=norm_weight.to(device) if norm_weight is not None else None, norm_eps=eps,
                 norm_scale=norm_scale, **kw)
    torch.cuda.synchronize(device)
    return out.cpu()


def learned(h, d, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.rand(h, generator=g) * 1.2 - 0.2, torch.rand(2 * d, generator=g) + 0.5


LENS = [0, 1, 15, 16, 17, 513, 255, 1100, 512, 64]


@pytest.mark.parametrize("cache,scale", [("fp16", "none"), ("e4m3", "block"), ("e5m2", "head"), ("int8", "block"), ("int8", "scalar")])
@pytest.mark.parametrize("pairs,group,d,bs", [(4, 4, 128, 16), (1, 8, 64, 64), (2, 1, 128, 128), (3, 3, 64, 16), (4, 5, 64, 32), (1, 2, 128, 32)])
def test_against_fp64(cuda_device, cache, scale, pairs, group, d, bs):
    case = paged_case(pairs * 10 + group, LENS, 2 * pairs * group, 2 * pairs, d, bs, cache=cache, scale=scale, spread=4.0)
    if scale == "scalar":
        case["k_scale"] = case["v_scale"] = max(case["k_scale"], case["v_scale"])
    lam, w = learned(pairs * group, d)
    check(run(case, cuda_device, lam), *reference(case, lam), f"{cache} {scale}")
    want = reference(case, lam, w, 1e-5, 0.2)
    check(run(case, cuda_device, lam, norm_weight=w, norm_scale=0.2), *want, f"{cache} {scale} with norm")


@pytest.mark.parametrize("npart,hint", [(1, None), (2, None), (5, None), (40, None), (3, 100), (2, 0), (7, 5000)])
def test_any_partition_count_and_hint(cuda_device, npart, hint):
    """The split follows the scratch; a hint that is too small, too large or missing changes no result."""
    case = paged_case(3, [1100, 0, 63, 64, 65, 700], 8, 4, 64, 16, cache="fp16")
    lam, _ = learned(4, 64)
    check(run(case, cuda_device, lam, npart=npart, hint=hint), *reference(case, lam), f"NP {npart} hint {hint}")


def test_many_partitions_long_context(cuda_device):
    case = paged_case(4, [40000, 30011], 8, 2, 128, 16, cache="e4m3", scale="head")
    lam, w = learned(4, 128)
    check(run(case, cuda_device, lam, norm_weight=w), *reference(case, lam, w), "long")


def test_garbage_behind_the_context(cuda_device):
    """NaN and infinity in the unused tail of the last blocks, and table entries beyond the context."""
    lens = [5, 33, 100]
    case = paged_case(5, lens, 8, 4, 128, 16, cache="fp16")
    lam, _ = learned(4, 128)
    want = reference(case, lam)
    for i, n in enumerate(lens):
        block = int(case["block_tables"][i, (n - 1) // 16])
        case["key_cache"][block, n % 16 or 16:] = float("nan")
        case["value_cache"][block, n % 16 or 16:] = float("inf")
        case["block_tables"][i, -(-n // 16):] = 10 ** 6
    check(run(case, cuda_device, lam), *want, "garbage")


def test_subnormal_value_scales(cuda_device):
    """Block scales whose reciprocal is infinite: the result is below every fp16 number."""
    case = paged_case(7, [300, 20], 8, 4, 64, 16, cache="e4m3", scale="block")
    case["v_scale"][:] = 1e-40
    assert (run(case, cuda_device, torch.full((4,), 0.5)) == 0).all()


def test_equal_maps_and_weight_one_cancel(cuda_device):
    """Both maps equal and lambda 1: the difference is a rounding of the partial sums, the norm keeps it finite."""
    case = paged_case(6, [300, 17], 4, 2, 64, 16, cache="fp16")
    case["key_cache"][:, :, 1] = case["key_cache"][:, :, 0]
    case["query"][:, 1::2] = case["query"][:, 0::2]
    lam = torch.ones(2)
    assert (run(case, cuda_device, lam) == 0).all()
    assert (run(case, cuda_device, lam, norm_weight=torch.ones(128)) == 0).all()


def test_subset_and_packed_tables(cuda_device):
    """seq_indices covers only its sequences (the others' rows stay), packed tables give the dense bits."""
    from flash_attention_factory_b200 import _cabi
    from flash_attention_factory_b200.host_io import pack_block_tables
    from flash_attention_factory_b200.lib import paged_attention_diff as diff

    dev = cuda_device
    lens = [300, 0, 70, 999, 16]
    case = paged_case(7, lens, 8, 4, 64, 16, cache="int8")
    lam, _ = learned(4, 64)
    whole = run(case, dev, lam)
    c = to(case, dev)
    sc = diff.scratch(c["query"], c["key_cache"], 999)
    out = torch.full((5, 4, 128), 9.0, dtype=torch.float16, device=dev)
    lam_dev = lam.to(dev)
    p = diff.params(*sc, out, c["query"], c["key_cache"], c["value_cache"], c["block_tables"], c["context_lens"], lam_dev,
                    case["sm_scale"], 1.0, 16, 999, k_scale_per_block=c["k_scale"], v_scale_per_block=c["v_scale"])
    ids, offsets = (t.to(dev) for t in pack_block_tables(case["block_tables"], lens, 16))
    some = torch.tensor([3, 1, 4], dtype=torch.int32, device=dev)
    p.attn.block_tables, p.attn.block_table_offsets = ids.data_ptr(), offsets.data_ptr()
    p.attn.seq_indices, p.attn.num_seqs = some.data_ptr(), 3
    _cabi.check(_cabi.load_library().launch_kernels_diff(ctypes.byref(p), ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream), None))
    torch.cuda.synchronize(dev)
    assert torch.equal(out.cpu()[[3, 1, 4]], whole[[3, 1, 4]])
    assert (out.cpu()[[0, 2]] == 9.0).all()


def test_runs_are_bit_identical_and_overlap(cuda_device):
    """Two streams with scratch of their own, a captured and replayed call, and the blocking form."""
    from flash_attention_factory_b200.lib import paged_attention_diff as diff

    dev = cuda_device
    case = paged_case(8, [700] * 40, 16, 8, 128, 16, cache="e4m3", scale="block")
    lam, w = learned(8, 128)
    once = run(case, dev, lam, norm_weight=w)
    c = to(case, dev)
    lam, w = lam.to(dev), w.to(dev)
    sets = [(diff.scratch(c["query"], c["key_cache"], 700), torch.empty(40, 8, 256, dtype=torch.float16, device=dev)) for _ in range(3)]

    def go(sc, out, fn=diff.enqueue):
        return fn(*sc, out, c["query"], c["key_cache"], c["value_cache"], c["block_tables"], c["context_lens"], lam,
                  case["sm_scale"], 1.0, 16, 700, norm_weight=w, k_scale_per_block=c["k_scale"], v_scale_per_block=c["v_scale"])

    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    torch.cuda.synchronize(dev)
    for _ in range(5):
        for st, (sc, out) in zip(streams, sets):
            with torch.cuda.stream(st):
                go(sc, out)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize(dev)
    with torch.cuda.graph(graph):
        go(*sets[2])
    graph.replay()
    graph.replay()
    torch.cuda.synchronize(dev)
    for _, out in sets:
        assert torch.equal(out.cpu(), once)
    us = go(*sets[0], fn=diff.run)
    assert len(us) == 2 and all(t > 0 for t in us) and torch.equal(sets[0][1].cpu(), once)


def test_empty_batch_and_wide_groups_of_pairs(cuda_device):
    """No sequences at all; 16 KV heads (4 head groups) with the largest group."""
    from flash_attention_factory_b200.lib import paged_attention_diff as diff

    dev = cuda_device
    q = torch.empty(0, 8, 64, dtype=torch.float16, device=dev)
    kc = torch.zeros(2, 16, 4, 64, dtype=torch.float16, device=dev)
    diff.enqueue(*diff.scratch(q, kc, 0), torch.empty(0, 4, 128, dtype=torch.float16, device=dev), q, kc, kc,
                 torch.empty(0, 1, dtype=torch.int32, device=dev), torch.empty(0, dtype=torch.int32, device=dev),
                 torch.ones(4, device=dev), 0.1, 1.0, 16, 0)
    case = paged_case(30, [333, 1, 90], 128, 16, 64, 64, cache="e5m2", scale="block", spread=4.0)
    lam, w = learned(64, 64)
    check(run(case, dev, lam, norm_weight=w), *reference(case, lam, w), "16 KV heads")


def test_decode_step_after_the_rotating_append(cuda_device):
    """rope_and_cache fills the pairs' cache like any other: append, then differential attention over it."""
    from flash_attention_factory_b200.cache_ops import rope_and_cache
    from test_rope_cache_gpu import rotated64, table

    dev = cuda_device
    lens = [40, 7, 130]
    case = paged_case(31, lens, 8, 4, 64, 16, cache="fp16")
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(3, 4, 64, generator=g).half() for _ in range(2))
    pos = torch.tensor(lens) - 1
    slots = torch.tensor([int(case["block_tables"][i, p // 16]) * 16 + p % 16 for i, p in enumerate(pos.tolist())])
    c = to(case, dev)
    qo = torch.empty_like(c["query"])
    rope_and_cache(c["query"], k.to(dev), v.to(dev), pos.to(dev), table(200, 64).to(dev), qo, c["key_cache"], c["value_cache"], slots.to(dev))
    torch.cuda.synchronize(dev)
    turned, size = rotated64(k, table(200, 64), pos, False)
    held = c["key_cache"].cpu().flatten(0, 1)[slots].double()
    assert ((held - turned).abs() <= HALF * turned.abs() + 2.0 ** -25 + 4 * 2.0 ** -24 * size).all()
    after = dict(case, query=qo.cpu(), key_cache=c["key_cache"].cpu(), value_cache=c["value_cache"].cpu())
    lam, w = learned(4, 64)
    check(run(after, dev, lam, norm_weight=w), *reference(after, lam, w), "after the append")
