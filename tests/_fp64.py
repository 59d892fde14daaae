"""Plain fp64 statements of the operators that have no reference counterpart, and the error that
fp16 storage of their intermediates allows."""
from __future__ import annotations

import math

import torch

HALF = 2.0 ** -11  # half a step of fp16, relative


def cache_values(cache, scale=None):
    """fp64 values of a cache [num_blocks, block_size, heads, head_size]; scale None, a number, [heads] or [num_blocks, heads]."""
    x = cache.to(torch.float16).double() if cache.dtype != torch.int8 else cache.double()
    if scale is None:
        return x
    if not torch.is_tensor(scale):
        return x * scale
    s = scale.double()
    return x * (s[:, None, :, None] if s.dim() == 2 else s[:, None])


def sequence(values, table_row, n):
    bs = values.shape[1]
    ids = table_row[: -(-n // bs)].long()
    return values[ids].flatten(0, 1)[:n]


def attention64(case, k_scale=None, v_scale=None, sinks=None, softcap=0.0, alibi=None, weighted_code=0.0):
    """(result, allowed error) [S, H, D] of decode attention in fp64.

    Allowed error, |v| weighted by the softmax being a = sum_t p_t |v_t|: the weights are rounded
    to fp16 before the value product (HALF a), the split variant stores partial rows in fp16 (HALF a),
    the result is fp16 (HALF a at most), and the fp32 chains (dot products of at most 128 terms,
    exponentials, sums) stay below another HALF a; a weight under 2^-14 of the reference is
    subnormal and off by up to 2^-25 absolute, of a reference of at least 1: n 2^-25 max|v|.
    `weighted_code`: the largest code where a block's V scale is multiplied into the weights as it is
    (the FP8 operators): the product p scale is then what is rounded, off by up to 2^-25 absolute where
    it is subnormal, and meets a code c instead of a value: n 2^-25 max|c|, 448 for e4m3."""
    q, bt, lens = case["query"].double(), case["block_tables"], [int(c) for c in case["context_lens"]]
    kv, vv = cache_values(case["key_cache"], k_scale), cache_values(case["value_cache"], v_scale)
    s, h, d = q.shape
    hk = kv.shape[2]
    out, tol = torch.zeros(s, h, d).double(), torch.full((s, h, d), 2.0 ** -24).double()
    for i, n in enumerate(lens):
        if n == 0:
            continue
        k, v = sequence(kv, bt[i], n), sequence(vv, bt[i], n)
        sc = torch.einsum("kgd,tkd->kgt", q[i].view(hk, h // hk, d), k) * case["sm_scale"]
        if softcap > 0:
            sc = softcap * torch.tanh(sc / softcap)
        if alibi is not None:
            sc = sc + alibi.double().view(hk, h // hk, 1) * (torch.arange(n) - (n - 1)).double()
        if sinks is not None:
            sc = torch.cat([sc, sinks.double().view(hk, h // hk, 1)], dim=-1)
        p = torch.softmax(sc, dim=-1)[..., :n]
        out[i] = torch.einsum("kgt,tkd->kgd", p, v).reshape(h, d)
        a = torch.einsum("kgt,tkd->kgd", p, v.abs()).reshape(h, d)
        tol[i] += 4 * HALF * a + n * 2.0 ** -25 * max(float(v.abs().max()), weighted_code)
    return out, tol


def check(got, want, tol, what=""):
    got = got.double().cpu()
    assert got.shape == want.shape, f"{what}: {got.shape} vs {want.shape}"
    assert torch.isfinite(got).all(), f"{what}: non-finite result"
    off = (got - want).abs() - tol
    assert (off <= 0).all(), (f"{what}: {int((off > 0).sum())} of {off.numel()} values beyond the bound, worst "
                              f"{(got - want).abs().flatten()[off.argmax()]:.3e} against {tol.flatten()[off.argmax()]:.3e}")


def paged_case(seed, lens, heads, kv_heads, head_size, block_size, cache="int8", scale="block", spread=1.0):
    """Random paged inputs (CPU); an 8-bit cache is quantised from fp16 pages with amax scales of the asked
    kind, and `spread` (log2) varies the size of the pages from block to block."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // block_size) for n in lens]
    nb, mb = sum(counts) + 3, max([1] + counts)
    perm = torch.randperm(nb, generator=g)
    bt = torch.zeros(len(lens), mb, dtype=torch.int32)
    at = 0
    for i, c in enumerate(counts):
        bt[i, :c] = perm[at:at + c].int()
        at += c
    case = dict(query=torch.randn(len(lens), heads, head_size, generator=g).half(), block_tables=bt,
                context_lens=torch.tensor(lens, dtype=torch.int32), sm_scale=1.0 / math.sqrt(head_size),
                block_size=block_size, k_scale=None, v_scale=None)
    qmax = {"int8": 127.0, "e4m3": 448.0, "e5m2": 57344.0}.get(cache)
    dtype = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}.get(cache)
    for name in ("key", "value"):
        x = torch.randn(nb, block_size, kv_heads, head_size, generator=g)
        if scale == "block" and spread:
            x = x * 2.0 ** (torch.rand(nb, 1, kv_heads, 1, generator=g) * spread - spread / 2)
        if cache == "fp16":
            case[f"{name}_cache"] = x.half()
            continue
        s = {"block": x.abs().amax((1, 3)), "head": x.abs().amax((0, 1, 3)), "scalar": x.abs().max()}[scale] / qmax
        by = s[:, None, :, None] if s.dim() == 2 else s[:, None] if s.dim() == 1 else s
        y = (x / by).clamp(-qmax, qmax)
        case[f"{name}_cache"] = y.round().to(torch.int8) if cache == "int8" else y.to(dtype)
        case[f"{name[0]}_scale"] = s if s.dim() else float(s)
    return case


def to(case, device):
    return {k: v.to(device) if torch.is_tensor(v) else v for k, v in case.items()}
