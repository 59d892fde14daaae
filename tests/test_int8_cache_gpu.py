"""Attention over an 8-bit integer cache: scalar, per-head and per-block scales, both variants."""
import pytest
import torch

from _fp64 import attention64, check, paged_case, to

pytestmark = pytest.mark.gpu


def _run(variant, case, device, scale=1.0, sinks=None, softcap=-1.0, alibi=None, **kw):
    from flash_attention_factory_b200 import lib

    c = to(case, device)
    s, h, d = c["query"].shape
    hk = c["key_cache"].size(2)
    max_ctx = int(case["context_lens"].max())
    npart = max(1, -(-max_ctx // (512 if d == 128 else 256)))
    ml = torch.full((s, h, npart), float("nan"), device=device)
    es = torch.full_like(ml, float("nan"))
    tmp = torch.full((s, h, npart, d), float("nan"), dtype=torch.float16, device=device)
    out = torch.full((s, h, d), float("nan"), dtype=torch.float16, device=device)
    mod = getattr(lib, f"paged_attention_int8_{variant}")
    mod.enqueue(ml, es, tmp, out, None, c["query"], c["key_cache"], c["value_cache"], c["block_tables"],
                c["context_lens"], h // hk, case["sm_scale"], scale, case["block_size"], max_ctx,
                alibi.to(device) if alibi is not None else torch.ones(h, device=device),
                sinks.to(device) if sinks is not None else None, softcap, use_alibi=alibi is not None,
                use_softcap=softcap > 0, **{k: v.to(device) for k, v in kw.items()})
    torch.cuda.synchronize(device)
    return out.cpu()


def _scales(case, kind):
    return {f"k_scale_per_{kind}": case["k_scale"], f"v_scale_per_{kind}": case["v_scale"]}


# every number of heads per CTA (1, 2, 4) and of tiles per stage, groups 1..8, contexts of nothing, one
# token, and around the block, partition and tile borders
@pytest.mark.parametrize("variant", ["loop", "reduce"])
@pytest.mark.parametrize("hk,group,d,bs", [(8, 4, 128, 16), (8, 5, 64, 64), (2, 8, 128, 32), (1, 3, 64, 128),
                                           (4, 1, 128, 64), (3, 2, 128, 16), (6, 7, 64, 16), (16, 2, 64, 32)])
def test_block_scales(cuda_device, variant, hk, group, d, bs):
    lens = [0, 1, 15, 16, 17, 513, 255, 1100, 512]
    case = paged_case(hk * 100 + group, lens, hk * group, hk, d, bs, spread=6.0)
    want, tol = attention64(case, case["k_scale"], case["v_scale"])
    check(_run(variant, case, cuda_device, scale=77.0, **_scales(case, "block")), want, tol, f"{variant} hk{hk} d{d} bs{bs}")


@pytest.mark.parametrize("variant", ["loop", "reduce"])
@pytest.mark.parametrize("kind", ["scalar", "head"])
def test_scalar_and_head_scales_with_sinks(cuda_device, variant, kind):
    case = paged_case(5, [700, 3, 64, 0, 2049], 12, 4, 128, 16, scale=kind)
    if kind == "scalar":
        case["k_scale"] = case["v_scale"] = max(case["k_scale"], case["v_scale"])
    sinks = torch.linspace(-2, 6, 12).half()
    want, tol = attention64(case, case["k_scale"], case["v_scale"], sinks=sinks)
    kw = dict(scale=case["k_scale"]) if kind == "scalar" else _scales(case, "head")
    check(_run(variant, case, cuda_device, sinks=sinks, **kw), want, tol, f"{variant} {kind}")


@pytest.mark.parametrize("variant", ["loop", "reduce"])
def test_score_modifiers_and_block_scales(cuda_device, variant):
    case = paged_case(6, [700, 33, 1025], 8, 2, 64, 16, spread=4.0)
    alibi = torch.linspace(0.01, 0.2, 8)
    want, tol = attention64(case, case["k_scale"], case["v_scale"], softcap=20.0, alibi=alibi)
    check(_run(variant, case, cuda_device, softcap=20.0, alibi=alibi, **_scales(case, "block")), want, tol, variant)


@pytest.mark.parametrize("variant", ["loop", "reduce"])
def test_values_of_very_different_size(cuda_device, variant):
    """Blocks whose values differ by 2^24, tiny values throughout (codes times 1e-6 are below what fp16
    holds exactly), blocks of zeros with a scale of 0, and codes of -128."""
    case = paged_case(8, [600, 31, 1300], 8, 4, 128, 16, spread=24.0)
    case["k_scale"] = case["k_scale"].clamp(max=0.05)
    case["v_scale"][::5] = 0.0
    case["value_cache"][::5] = 0
    case["k_scale"][1::7] = 0.0
    case["value_cache"][3, 4, 1, 5] = -128
    want, tol = attention64(case, case["k_scale"], case["v_scale"])
    check(_run(variant, case, cuda_device, **_scales(case, "block")), want, tol, "wide range")
    case = paged_case(9, [600, 31, 1300], 8, 4, 128, 16, spread=2.0)
    case["v_scale"] *= 1e-4
    want, tol = attention64(case, case["k_scale"], case["v_scale"])
    # results near 1e-4: the bound is carried by the values' size, not by an absolute term (2^-24 is half a subnormal step)
    check(_run(variant, case, cuda_device, **_scales(case, "block")), want, tol, "small values")
    assert float(want.abs().max()) < 1e-3


@pytest.mark.parametrize("variant", ["loop", "reduce"])
def test_subnormal_value_scales(cuda_device, variant):
    """Scales whose reciprocal is infinite, alone (the result is below every fp16 number) and beside ordinary ones."""
    case = paged_case(14, [300, 20], 4, 2, 64, 16)
    case["v_scale"][:] = 1e-40
    assert (_run(variant, case, cuda_device, **_scales(case, "block")) == 0).all()
    case = paged_case(14, [300, 20], 4, 2, 64, 16)
    case["v_scale"][::2] = 1e-40
    want, tol = attention64(case, case["k_scale"], case["v_scale"])
    check(_run(variant, case, cuda_device, **_scales(case, "block")), want, tol, variant)


def test_scales_of_blocks_outside_the_context_are_not_used(cuda_device):
    case = paged_case(10, [40, 16], 4, 2, 128, 16)
    used = {int(b) for i, n in enumerate([40, 16]) for b in case["block_tables"][i, : -(-n // 16)]}
    idle = [b for b in range(case["key_cache"].size(0)) if b not in used]
    case["k_scale"][idle] = float("nan")
    case["v_scale"][idle] = float("inf")
    want, tol = attention64(case, case["k_scale"], case["v_scale"])
    for variant in ("loop", "reduce"):
        check(_run(variant, case, cuda_device, **_scales(case, "block")), want, tol, variant)


def test_wide_launch_gives_the_bits_of_the_narrow_one(cuda_device):
    """A sequence alone (4-warp CTAs) and inside a batch that fills the GPU twice (8-warp CTAs)."""
    lens = [1024] * 160
    case = paged_case(12, lens, 8, 8, 64, 64, spread=3.0)
    batch = _run("reduce", case, cuda_device, **_scales(case, "block"))
    one = {**case, "query": case["query"][7:8], "block_tables": case["block_tables"][7:8], "context_lens": case["context_lens"][7:8]}
    assert torch.equal(_run("reduce", one, cuda_device, **_scales(case, "block"))[0], batch[7])


def test_through_the_other_entry_points(cuda_device):
    """serving, torch custom ops and the host-buffer step run the int8 operators."""
    import flash_attention_factory_b200.torch_ops  # noqa: F401
    from flash_attention_factory_b200 import host_io, lib
    from flash_attention_factory_b200.serving import AutoDecodePlan, paged_attention_auto

    lens = [700, 40, 1500, 9]
    case = paged_case(13, lens, 8, 4, 128, 16)
    c = to(case, cuda_device)
    want, tol = attention64(case, case["k_scale"], case["v_scale"])
    direct = _run("reduce", case, cuda_device, **_scales(case, "block"))
    plan = AutoDecodePlan(lens, 8, 128, 16, c["block_tables"].size(1), cuda_device, fold_short_fraction=0.0)
    out = torch.empty(4, 8, 128, dtype=torch.float16, device=cuda_device)
    paged_attention_auto(plan, out, c["query"], c["key_cache"], c["value_cache"], c["block_tables"], c["context_lens"], 2,
                         case["sm_scale"], k_scale_per_block=c["k_scale"], v_scale_per_block=c["v_scale"])
    check(out, want, tol, "serving")
    ml = torch.empty(4, 8, 3, device=cuda_device)
    tmp = torch.empty(4, 8, 3, 128, dtype=torch.float16, device=cuda_device)
    args = (c["query"], c["key_cache"], c["value_cache"], c["block_tables"], c["context_lens"], 2, case["sm_scale"], 1.0, 16,
            1500, torch.ones(8, device=cuda_device), None, -1.0)
    for name in ("int8_loop", "int8_reduce"):
        out.zero_()
        getattr(torch.ops.paged_attention_b200, name)(ml, ml.clone(), tmp, out, *args, c["k_scale"], c["v_scale"])
        check(out, want, tol, name)
    io = host_io.DecodeStepIO(4, 8, 128, c["block_tables"].size(1), cuda_device)
    io.query_host.copy_(case["query"])
    io.block_tables_host.copy_(case["block_tables"])
    io.context_lens_host.copy_(case["context_lens"])
    p = lib.paged_attention_int8_reduce.params(ml, ml.clone(), tmp, io.out, None, io.query, c["key_cache"], c["value_cache"],
                                               io.block_tables, io.context_lens, 2, case["sm_scale"], 1.0, 16, 1500,
                                               torch.ones(8, device=cuda_device), None, -1.0,
                                               k_scale_per_block=c["k_scale"], v_scale_per_block=c["v_scale"])
    assert torch.equal(io.bind(lib.paged_attention_int8_reduce.ENTRY, p).run(), direct)


@pytest.mark.parametrize("scales", ["scalar", "head", "block"])
def test_writer_stores_rounded_integers(cuda_device, scales):
    """reshape_and_cache on an int8 cache: round(x / s), ties to even, clamped to +-127; NaN -> 0."""
    from flash_attention_factory_b200.cache_ops import reshape_and_cache

    g = torch.Generator().manual_seed(3)
    t, hk, d, bs, nb = 21, 3, 64, 16, 4
    key = (torch.randn(t, hk, d, generator=g) * 3).half()
    value = (torch.randn(t, hk, d, generator=g) * 3).half()
    key[0, 0, :4] = torch.tensor([float("inf"), -float("inf"), float("nan"), 65504.0]).half()
    kc = torch.randint(-127, 128, (nb, bs, hk, d), generator=g).to(torch.int8)
    vc = kc.flip(0).contiguous()
    slots = torch.randperm(nb * bs, generator=g)[:t]
    slots[4] = -1
    s = {"scalar": torch.tensor(0.043), "head": torch.rand(2, hk, generator=g) * 0.1 + 0.01,
         "block": torch.rand(2, nb, hk, generator=g) * 0.1 + 0.01}[scales]
    want = [kc.clone(), vc.clone()]
    for w, x, of in zip(want, (key, value), (s, s) if scales == "scalar" else s):
        flat = w.view(-1, hk, d)
        for i, slot in enumerate(slots.tolist()):
            if slot >= 0:
                by = of if scales == "scalar" else of[:, None] if scales == "head" else of[slot // bs][:, None]
                flat[slot] = (x[i].float() / by).nan_to_num(0.0, 1e9, -1e9).round().clamp(-127, 127).to(torch.int8)
    dk, dv = kc.to(cuda_device), vc.to(cuda_device)
    kw = {} if scales == "scalar" else {f"k_scale_per_{scales}": s[0].contiguous().to(cuda_device), f"v_scale_per_{scales}": s[1].contiguous().to(cuda_device)}
    reshape_and_cache(key.to(cuda_device), value.to(cuda_device), dk, dv, slots.to(cuda_device),
                      float(s) if scales == "scalar" else 1.0, **kw)
    torch.cuda.synchronize(cuda_device)
    assert torch.equal(dk.cpu(), want[0]) and torch.equal(dv.cpu(), want[1])


@pytest.mark.parametrize("hk,group", [(4, 2), (1, 3)])
def test_many_short_sequences_run_the_persistent_form(cuda_device, hk, group):
    """At least four units per SM and a known, short maximum: whole-context items, with a warp per head and with
    warps that share one, empty contexts among them."""
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(0, 90, (700,), generator=g).tolist()
    case = paged_case(14, lens, hk * group, hk, 64, 16, spread=6.0)
    want, tol = attention64(case, case["k_scale"], case["v_scale"])
    check(_run("loop", case, cuda_device, **_scales(case, "block")), want, tol, f"hk{hk}")


def test_host_batch_step(cuda_device):
    """The pipelined host-buffer step takes the int8 entry points; cut into sub-batches it gives the same bits."""
    from flash_attention_factory_b200 import _cabi

    lens = [700, 40, 1500, 9, 300, 0, 513, 77]
    case = paged_case(15, lens, 8, 4, 128, 16)
    direct = _run("reduce", case, cuda_device, **_scales(case, "block"))
    c = to(case, cuda_device)
    ml, es = (torch.empty(8, 8, 3, device=cuda_device) for _ in range(2))
    tmp = torch.empty(8, 8, 3, 128, dtype=torch.float16, device=cuda_device)
    out = torch.zeros(8, 8, 128, dtype=torch.float16, device=cuda_device)
    q, bt, cl = (torch.empty_like(c[n]) for n in ("query", "block_tables", "context_lens"))
    from flash_attention_factory_b200.lib import paged_attention_int8_reduce as mod

    p = mod.params(ml, es, tmp, out, None, q, c["key_cache"], c["value_cache"], bt, cl, 2, case["sm_scale"], 1.0, 16, 1500,
                   torch.ones(8, device=cuda_device), None, -1.0, **{k: v.to(cuda_device) for k, v in _scales(c, "block").items()})
    host = [case[n].pin_memory() for n in ("query", "block_tables", "context_lens")]
    for n in (1, 3):
        host_out = torch.zeros(8, 8, 128, dtype=torch.float16).pin_memory()
        io = _cabi.PaHostBatch()
        io.host_query, io.host_block_tables, io.host_context_lens = (t.data_ptr() for t in host)
        io.host_out, io.sub_batches = host_out.data_ptr(), n
        import ctypes

        _cabi.check(_cabi.load_library().pa_decode_step_host_batch(
            _cabi.ENTRY_IDS[mod.ENTRY], ctypes.byref(p), ctypes.byref(io),
            ctypes.c_void_p(torch.cuda.current_stream(cuda_device).cuda_stream), 1))
        assert torch.equal(host_out, direct), n


def test_overlapping_and_captured_launches(cuda_device):
    """Two streams with scratch of their own and a captured, replayed launch, bit for bit against a solitary one."""
    from flash_attention_factory_b200.lib import paged_attention_int8_reduce as mod

    dev = cuda_device
    case = paged_case(16, [900] * 40, 16, 8, 128, 16, spread=3.0)
    once = _run("reduce", case, dev, **_scales(case, "block"))
    c = to(case, dev)
    alibi = torch.ones(16, device=dev)
    sets = [(torch.empty(40, 16, 2, device=dev), torch.empty(40, 16, 2, device=dev),
             torch.empty(40, 16, 2, 128, dtype=torch.float16, device=dev), torch.empty(40, 16, 128, dtype=torch.float16, device=dev))
            for _ in range(3)]

    def go(s):
        mod.enqueue(*s, None, c["query"], c["key_cache"], c["value_cache"], c["block_tables"], c["context_lens"], 2,
                    case["sm_scale"], 1.0, 16, 900, alibi, None, -1.0, k_scale_per_block=c["k_scale"], v_scale_per_block=c["v_scale"])

    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    torch.cuda.synchronize(dev)
    for _ in range(6):
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                go(s)
    torch.cuda.synchronize(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go(sets[2])
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize(dev)
    for s in sets:
        assert torch.equal(s[3].cpu(), once)


def test_block_ids_outside_the_cache_read_zeros(cuda_device):
    """As in the FP8 operators: such a block is zeros (under the scale of the last block)."""
    case = paged_case(17, [40], 4, 4, 64, 16)
    zeroed = {k: (v.clone() if torch.is_tensor(v) else v) for k, v in case.items()}
    block = int(case["block_tables"][0, 1])
    zeroed["key_cache"][block] = 0
    zeroed["value_cache"][block] = 0
    want, tol = attention64(zeroed, case["k_scale"], case["v_scale"])
    case["block_tables"][0, 1] = case["key_cache"].size(0) + 7
    for variant in ("loop", "reduce"):
        check(_run(variant, case, cuda_device, **_scales(case, "block")), want, tol, variant)


@pytest.mark.parametrize("scheme,parts", [("lpt", 3), ("heads", 2)])
def test_shards_of_a_batch(cuda_device, scheme, parts):
    """The multi-GPU driver on logical shards of an int8 batch: gathered, the bits of the whole batch."""
    from flash_attention_factory_b200.multi_gpu import shard_reference_batch

    case = paged_case(15, [900, 17, 2100, 640, 333], 16, 8, 128, 16, scale="scalar")
    scale = case["k_scale"] = case["v_scale"] = max(case["k_scale"], case["v_scale"])
    job = shard_reference_batch({**case, "fp8_scale": scale}, [cuda_device] * parts, scheme, "reduce")
    job.run()
    got = job.gather(torch.empty(5, 16, 128, dtype=torch.float16, device=cuda_device))
    want, tol = attention64(case, scale, scale)
    check(got, want, tol, scheme)
    assert torch.equal(got.cpu(), _run("reduce", case, cuda_device, scale=scale))
