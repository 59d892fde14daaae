"""The operators beside the reference's four refuse bad arguments on the host, before any device work."""
import ctypes

import pytest
import torch

import flash_attention_factory_b200 as pkg
from flash_attention_factory_b200 import _cabi


@pytest.fixture(scope="module")
def lib():
    from flash_attention_factory_b200 import build

    build.build()
    return pkg.load_library()


def _attn(**kw):
    p = _cabi.PaParams()
    base = dict(out=0x1000, max_logits=0x2000, exp_sums=0x3000, tmp_out=0x4000, query=0x5000, key_cache=0x6000,
                value_cache=0x7000, block_tables=0x8000, context_lens=0x9000, num_seqs=2, num_heads=8, head_size=128,
                num_kv_heads=2, max_num_partitions=1, max_blocks_per_seq=4, block_size=16, num_queries_per_tokens=4,
                num_blocks=8, sm_scale=0.1, fp8_scale=1.0, kv_dtype=_cabi.KV_INT8)
    base.update(kw)
    for k, v in base.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("entry", ["launch_kernels_int8_loop", "launch_kernels_int8_reduce"])
def test_int8_entries(lib, entry):
    def call(**kw):
        p = _attn(**kw)
        return getattr(lib, entry)(ctypes.byref(p), None, None), lib.pa_last_error().decode()

    for kv in (_cabi.KV_F16, _cabi.KV_FP8_E5M2, _cabi.KV_FP8_E4M3, 4, -1):
        rc, msg = call(kv_dtype=kv)
        assert rc == _cabi.PA_ERR_BAD_ARG and "kv_dtype" in msg
    assert call(head_size=96)[0] == _cabi.PA_ERR_UNSUPPORTED
    assert call(fp8_scale=0.0)[0] == _cabi.PA_ERR_BAD_ARG
    assert call(query=0)[0] == _cabi.PA_ERR_BAD_ARG
    assert "together" in call(k_scale_per_block=0x1000)[1]
    assert "exclude" in call(k_scale_per_block=0x1000, v_scale_per_block=0x1000, k_scale_per_head=0x1000)[1]
    assert call(num_seqs=0)[0] == _cabi.PA_OK
    assert getattr(lib, entry)(None, None, None) == _cabi.PA_ERR_BAD_ARG


def test_fp8_entries_refuse_an_int8_cache(lib):
    for entry in ("launch_kernels_loop", "launch_kernels_reduce", "launch_kernels_fp8_loop", "launch_kernels_fp8_reduce"):
        assert getattr(lib, entry)(ctypes.byref(_attn()), None, None) == _cabi.PA_ERR_BAD_ARG


def test_int8_modules_mirror_the_fp8_surface():
    import inspect

    from flash_attention_factory_b200 import lib as shim

    for variant in ("loop", "reduce"):
        for fn in ("run", "params", "enqueue"):
            a = inspect.signature(getattr(getattr(shim, f"paged_attention_int8_{variant}"), fn))
            b = inspect.signature(getattr(getattr(shim, f"paged_attention_fp8_{variant}"), fn))
            assert [n.replace("int8_scale", "fp8_scale") for n in a.parameters] == list(b.parameters)


def test_int8_modules_refuse_cpu_tensors():
    from flash_attention_factory_b200 import lib as shim

    c = torch.zeros(1, 16, 1, 128, dtype=torch.int8)
    with pytest.raises(RuntimeError, match="CUDA"):
        shim.paged_attention_int8_loop.run(torch.zeros(1, 2, 1), torch.zeros(1, 2, 1), torch.zeros(1, 2, 1, 128).half(),
                                           torch.zeros(1, 2, 128).half(), torch.zeros(1), torch.zeros(1, 2, 128).half(), c, c,
                                           torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32), 2, 0.1,
                                           1.0, 16, 1, torch.ones(2), None, -1.0)


def _cache_write(p, **kw):
    base = dict(key=0x1000, value=0x2000, key_cache=0x3000, value_cache=0x4000, slot_mapping=0x5000, num_tokens=3,
                num_kv_heads=2, head_size=128, block_size=16, num_blocks=4, fp8_scale=1.0, kv_dtype=_cabi.KV_INT8)
    base.update(kw)
    for k, v in base.items():
        setattr(p, k, v)


def test_rope_and_cache(lib):
    def call(cache=None, **kw):
        p = _cabi.PaRopeCacheParams()
        _cache_write(p.cache, **(cache or {}))
        base = dict(query=0x6000, query_out=0x7000, positions=0x8000, cos_sin=0x9000, max_position=64, rotary_dim=128,
                    num_heads=4, query_token_stride=512, key_token_stride=256, value_token_stride=256)
        base.update(kw)
        for k, v in base.items():
            setattr(p, k, v)
        return lib.pa_rope_and_cache(ctypes.byref(p), None), lib.pa_last_error().decode()

    bad, unsupported = _cabi.PA_ERR_BAD_ARG, _cabi.PA_ERR_UNSUPPORTED
    assert lib.pa_rope_and_cache(None, None) == bad
    assert call(cache=dict(num_tokens=0))[0] == _cabi.PA_OK
    assert call(cache=dict(kv_dtype=9))[0] == bad
    assert call(cache=dict(key=0x1008))[0] == bad
    assert call(cache=dict(fp8_scale=0.0))[0] == bad
    assert call(cache=dict(head_size=72))[0] == unsupported
    assert call(cache=dict(head_size=528))[0] == unsupported
    for r in (0, 8, 24, 144):
        assert call(rotary_dim=r)[0] == unsupported
    assert call(max_position=0)[0] == bad
    assert call(positions=0)[0] == bad
    assert call(cos_sin=0)[0] == bad
    assert call(cos_sin=0x9004)[0] == bad
    assert "together" in call(query=0)[1]
    assert "together" in call(query_out=0)[1]
    assert call(num_heads=0)[0] == bad
    assert call(query=0x6004)[0] == bad
    assert call(key_token_stride=260)[0] == bad


def test_cache_ops_refuse_cpu_tensors_and_odd_layouts():
    from flash_attention_factory_b200 import cache_ops

    k = torch.zeros(2, 1, 64).half()
    kc = torch.zeros(1, 16, 1, 64, dtype=torch.int8)
    i = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        cache_ops.rope_and_cache(None, k, k, i, torch.zeros(4, 64), None, kc, kc, i)


def test_append_block_scaled(lib):
    def call(**kw):
        p = _cabi.PaBlockScaledParams()
        base = dict(key=0x1000, value=0x2000, key_cache=0x3000, value_cache=0x4000, k_scale_per_block=0x5000,
                    v_scale_per_block=0x6000, block_tables=0x7000, context_lens=0x8000, num_seqs=3, num_tokens=3,
                    num_kv_heads=2, head_size=128, block_size=16, max_blocks_per_seq=4, num_blocks=8, kv_dtype=_cabi.KV_INT8,
                    key_token_stride=256, value_token_stride=256)
        base.update(kw)
        for k, v in base.items():
            setattr(p, k, v)
        return lib.pa_append_block_scaled(ctypes.byref(p), None), lib.pa_last_error().decode()

    bad, unsupported = _cabi.PA_ERR_BAD_ARG, _cabi.PA_ERR_UNSUPPORTED
    assert lib.pa_append_block_scaled(None, None) == bad
    assert call(num_tokens=0)[0] == _cabi.PA_OK and call(num_seqs=0)[0] == _cabi.PA_OK
    assert call(kv_dtype=_cabi.KV_F16)[0] == bad and call(kv_dtype=7)[0] == bad
    assert call(head_size=72)[0] == unsupported
    assert call(block_size=24)[0] == unsupported and call(block_size=2048)[0] == unsupported
    assert call(num_kv_heads=0)[0] == bad
    for name in ("key", "value", "key_cache", "value_cache", "k_scale_per_block", "v_scale_per_block", "block_tables", "context_lens"):
        rc, msg = call(**{name: 0})
        assert rc == bad and "null" in msg, name
    assert "num_tokens must equal" in call(num_tokens=4)[1]
    assert call(key=0x1008)[0] == bad
    assert call(num_blocks=0)[0] == bad
    assert call(cos_sin=0x9000, max_position=8, rotary_dim=40)[0] == unsupported
    assert "together" in call(query=0xa000)[1]


def test_differential_attention(lib):
    def call(lambdas=0x1000, norm_weight=0, norm_eps=1e-5, **kw):
        p = _cabi.PaDiffParams()
        src = _attn(**{"kv_dtype": _cabi.KV_F16, **kw})
        ctypes.memmove(ctypes.byref(p.attn), ctypes.byref(src), ctypes.sizeof(src))
        p.lambdas, p.norm_weight, p.norm_eps, p.norm_scale = lambdas, norm_weight, norm_eps, 1.0
        return lib.launch_kernels_diff(ctypes.byref(p), None, None), lib.pa_last_error().decode()

    bad, unsupported = _cabi.PA_ERR_BAD_ARG, _cabi.PA_ERR_UNSUPPORTED
    assert lib.launch_kernels_diff(None, None, None) == bad
    assert call(num_seqs=0)[0] == _cabi.PA_OK
    assert call(kv_dtype=8)[0] == bad
    assert call(head_size=96)[0] == unsupported
    assert call(num_queries_per_tokens=9, num_heads=18)[0] == unsupported
    rc, msg = call(num_heads=12, num_kv_heads=3)
    assert rc == bad and "pairs" in msg
    assert call(lambdas=0)[0] == bad
    assert call(norm_weight=0x1000, norm_eps=0.0)[0] == bad
    assert call(norm_weight=0x1004)[0] == bad
    for extra in (dict(sinks=0x1000), dict(alibi_slopes=0x1000), dict(softcap=3.0)):
        assert call(**extra)[0] == unsupported
    assert call(max_logits=0)[0] == bad and call(max_num_partitions=0)[0] == bad
    assert call(k_scale_per_head=0x1000, v_scale_per_head=0x1000)[0] == bad  # an fp16 cache has no scales


def test_diff_partition_counts(lib):
    n = lib.pa_diff_num_partitions
    f16, e4m3 = _cabi.KV_F16, _cabi.KV_FP8_E4M3
    assert n(1, 3, 128, 1000, f16) == 0 and n(1, 2, 96, 1000, f16) == 0 and n(1, 0, 128, 1000, f16) == 0 and n(1, 2, 64, 9, 7) == 0
    assert n(4, 8, 128, 0, f16) == 1 and n(4, 8, 128, 1, f16) == 1
    assert n(3000, 8, 128, 1024, e4m3) == 2 and n(3000, 8, 128, 1024, f16) == 4  # a large batch: items of 512 KB
    assert n(1, 2, 64, 1000, e4m3) == 16          # a lone short sequence: 64 tokens
    assert n(2, 8, 128, 65536, e4m3) == 74        # 4 units: 296 items, one for every resident CTA
    assert n(1000, 4, 128, 2 ** 27, f16) == 65535
    for seqs in (1, 3, 40, 500):
        for ctx in (1, 63, 700, 9000, 200000):
            assert 1 <= n(seqs, 8, 64, ctx, e4m3) <= -(-ctx // 64)
