"""The cache and attention operators on real work: what is called, on what, and what it costs at least.

Four operators of a decode step on a paged KV cache:
  rope    cache_ops.rope_and_cache        queries and keys rotated by position, K/V appended to the cache
  append  cache_ops.append_block_scaled   K/V appended to an 8-bit cache that keeps a scale per block and head
  int8    lib.paged_attention_int8_*      decode attention over an int8 cache with a scale per block and head
  diff    lib.paged_attention_diff        differential attention (difference of two softmax maps), decode

`run` computes the plain form where `own` is false (elementary torch operations in fp32) and calls
the library where it is true; `exact` restates each operator in fp64.
"""
import math
import random

import torch

own = False

MAX_POSITION = 65536
QMAX = {"int8": 127.0, "e4m3": 448.0, "e5m2": 57344.0}
DTYPES = {"fp16": torch.float16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
DEVICE = "cuda"


# ------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one user, one token: nothing but latency
        dict(name="rope: one token", op="rope", tokens=1, heads=32, kv_heads=8, head_size=128, rotary=128,
             interleaved=False, cache="fp16", scales="none", block=16, padded=0, strided=True, prompt=False),
        # a mixed step of 2053 tokens with padding rows, part of the head rotated, FP8 cache with per-head scales
        dict(name="rope: mixed step, e4m3", op="rope", tokens=2053, heads=40, kv_heads=8, head_size=64, rotary=32,
             interleaved=True, cache="e4m3", scales="head", block=64, padded=37, strided=True, prompt=False),
        # a long prompt, everything moved once
        dict(name="rope: prefill 32768", op="rope", tokens=32768, heads=32, kv_heads=8, head_size=128, rotary=128,
             interleaved=False, cache="fp16", scales="none", block=16, padded=0, strided=True, prompt=True),
        # one new token for each of 256 sequences, int8 blocks that are partly full
        dict(name="append: decode 256, int8", op="append", seqs=256, new_lo=1, new_hi=1, old_lo=0, old_hi=4096,
             lens_seed=11, heads=0, kv_heads=8, head_size=128, rotary=0, interleaved=False, cache="int8", block=16),
        # speculative tokens and prompt chunks together, rotated on the way, queries too
        dict(name="append: chunks, e4m3", op="append", seqs=37, new_lo=1, new_hi=512, old_lo=0, old_hi=2000,
             lens_seed=12, heads=40, kv_heads=8, head_size=64, rotary=64, interleaved=False, cache="e4m3", block=64),
        # prompts of a batch
        dict(name="append: prefill, e4m3", op="append", seqs=8, new_lo=2048, new_hi=8192, old_lo=0, old_hi=0,
             lens_seed=13, heads=0, kv_heads=8, head_size=128, rotary=128, interleaved=False, cache="e4m3", block=16),
        # a handful of short sequences
        dict(name="int8: 4 short", op="int8", seqs=4, ctx_lo=129, ctx_hi=512, lens_seed=21, heads=32, kv_heads=8,
             head_size=128, block=16, variant="loop"),
        # the small-head serving shape, blocks of 64 tokens
        dict(name="int8: 64 x 1500, head 64", op="int8", seqs=64, ctx_lo=1500, ctx_hi=1500, lens_seed=22, heads=40,
             kv_heads=8, head_size=64, block=64, variant="loop"),
        # a ragged batch
        dict(name="int8: 128 ragged to 8192", op="int8", seqs=128, ctx_lo=1024, ctx_hi=8192, lens_seed=23, heads=32,
             kv_heads=8, head_size=128, block=16, variant="reduce"),
        # a few short sequences, no norm
        dict(name="diff: 3 short, fp16", op="diff", seqs=3, ctx_lo=60, ctx_hi=509, lens_seed=31, heads=16, kv_heads=4,
             head_size=64, block=16, cache="fp16", scales="none", norm=False),
        # a ragged batch with the per-head norm
        dict(name="diff: 48 ragged to 8192, fp16", op="diff", seqs=48, ctx_lo=1024, ctx_hi=8192, lens_seed=32, heads=16,
             kv_heads=4, head_size=128, block=16, cache="fp16", scales="none", norm=True),
        # two very long sequences, FP8 cache, the widest group
        dict(name="diff: 2 x 65536, e4m3", op="diff", seqs=2, ctx_lo=65536, ctx_hi=65536, lens_seed=33, heads=32,
             kv_heads=4, head_size=128, block=16, cache="e4m3", scales="head", norm=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "int8", "diff"])
    head_size = rng.choice([64, 128])
    block = rng.choice([16, 32, 64, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    group = rng.randint(1, 8)
    if op == "rope":
        cache = rng.choice(["fp16", "e5m2", "e4m3", "int8"])
        tokens = _log(rng, 1, 12000)
        return dict(op=op, tokens=tokens, heads=kv_heads * group, kv_heads=kv_heads, head_size=head_size,
                    rotary=rng.choice([head_size, head_size, head_size // 2, 16]), interleaved=rng.random() < 0.5,
                    cache=cache, scales="none" if cache == "fp16" else rng.choice(["head", "block"]), block=block,
                    padded=rng.randint(0, tokens // 4), strided=rng.random() < 0.5, prompt=rng.random() < 0.5)
    if op == "append":
        rotary = rng.choice([0, head_size, head_size // 2])
        seqs = _log(rng, 1, 300)
        return dict(op=op, seqs=seqs, new_lo=1, new_hi=_log(rng, 1, max(1, 20000 // seqs)), old_lo=0,
                    old_hi=_log(rng, 1, 3000), lens_seed=rng.randrange(1 << 20), heads=kv_heads * group if rotary else 0,
                    kv_heads=kv_heads, head_size=head_size, rotary=rotary, interleaved=rng.random() < 0.5,
                    cache=rng.choice(["e5m2", "e4m3", "int8"]), block=block)
    # attention: the KV tokens of a draw stay below those of the largest listed case
    hi = _log(rng, 1, 40000)
    seqs = _log(rng, 1, max(1, min(200, 160000 // hi)))
    if op == "int8":
        return dict(op=op, seqs=seqs, ctx_lo=rng.choice([0, 1, max(1, hi // 4)]), ctx_hi=hi, lens_seed=rng.randrange(1 << 20),
                    heads=kv_heads * group, kv_heads=kv_heads, head_size=head_size, block=block,
                    variant=rng.choice(["loop", "reduce"]))
    cache = rng.choice(["fp16", "e5m2", "e4m3", "int8"])
    pairs = rng.choice([1, 2, 3, 4])
    return dict(op=op, seqs=seqs, ctx_lo=rng.choice([0, 1, max(1, hi // 4)]), ctx_hi=hi, lens_seed=rng.randrange(1 << 20),
                heads=pairs * group, kv_heads=pairs, head_size=head_size, block=block, cache=cache,
                scales="none" if cache == "fp16" else rng.choice(["head", "block"]), norm=rng.random() < 0.5)


def _spread(lens_seed, n, lo, hi):
    """n lengths between lo and hi, log-normal in the middle of the range, the first one hi: part of the case, not of the seed."""
    if lo >= hi:
        return [hi] * n
    r = random.Random(lens_seed)
    out = [hi]
    for _ in range(n - 1):
        out.append(min(hi, max(lo, int(round(math.exp(r.gauss(math.log(max(1.0, (lo + hi) / 3)), 0.6)))))))
    return out


def _append_lens(case):
    """(tokens held, tokens appended) per sequence."""
    new = _spread(case["lens_seed"], case["seqs"], case["new_lo"], case["new_hi"])
    r = random.Random(case["lens_seed"] + 1)
    old = [r.randint(case["old_lo"], case["old_hi"]) for _ in new]
    return old, new


def _ctx_lens(case):
    return _spread(case["lens_seed"], case["seqs"], case["ctx_lo"], case["ctx_hi"])


def _size(cache):
    return 2 if cache == "fp16" else 1


def work(case):
    op, d, hk = case["op"], case["head_size"], case["kv_heads"]
    if op == "rope":
        t = case["tokens"] - case["padded"]
        n = t * (2 * case["heads"] * d * 2 + 2 * hk * d * (2 + _size(case["cache"])) + case["rotary"] * 4 + 16)
        return {"bytes": n, "flops": 3 * t * (case["heads"] + hk) * case["rotary"]}
    if op == "append":
        old, new = _append_lens(case)
        bs, t = case["block"], sum(new)
        held = sum(o % bs for o in old)  # rows of a started block: read and written once where a scale grows
        blocks = sum(-(-(o + n) // bs) - o // bs for o, n in zip(old, new))
        n = t * (2 * hk * d * 3 + 2 * case["heads"] * d * 2 + case["rotary"] * 4) + held * 2 * hk * d + blocks * hk * 16
        return {"bytes": n, "flops": 3 * t * (case["heads"] + hk) * case["rotary"] + 4 * t * hk * d}
    tokens, bs = sum(_ctx_lens(case)), case["block"]
    if op == "int8":
        n = tokens * hk * d * 2 + (tokens // bs) * (hk * 8 + 4) + case["seqs"] * case["heads"] * d * 4
        return {"bytes": n, "flops": 4 * tokens * case["heads"] * d}
    n = tokens * 2 * hk * d * 2 * _size(case["cache"]) + (tokens // bs) * 4 + case["seqs"] * case["heads"] * 2 * d * 4
    if case["scales"] == "block":
        n += (tokens // bs) * 2 * hk * 8
    return {"bytes": n, "flops": 2 * tokens * case["heads"] * (2 * d + 4 * d)}


# ------------------------------------------------------------------------------------ the inputs
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float16)


def _rows_to_codes(x, cache, scale):
    """fp16 rows [..., heads, head size] -> what the cache holds; scale broadcasts over the last dim."""
    if cache == "fp16":
        return x
    y = (x.float() / scale).clamp(-QMAX[cache], QMAX[cache])
    return y.round().to(torch.int8) if cache == "int8" else y.to(DTYPES[cache])


def _pool(g, case, blocks, heads):
    """A cache of `blocks` blocks and its scale: None, per head [heads] or per block and head [blocks, heads]."""
    cache, bs, d = case["cache"], case["block"], case["head_size"]
    x = _randn(g, blocks, bs, heads, d)
    kind = case.get("scales", "block")
    if cache == "fp16":
        return x, None
    if kind == "head":
        amax = x.abs().amax(dim=(0, 1, 3)).float()
        scale = amax / QMAX[cache]
        return _rows_to_codes(x, cache, scale.view(1, 1, heads, 1)), scale
    x *= torch.rand(blocks, 1, heads, 1, generator=g, device=DEVICE).half() * 2 + 0.25  # blocks differ in size
    scale = x.abs().amax(dim=(1, 3)).float() / QMAX[cache]
    return _rows_to_codes(x, cache, scale.view(blocks, 1, heads, 1)), scale


def _tables(g, lens, bs, spare):
    """Block tables [S, MB] of rows of distinct blocks in random order, and the number of blocks."""
    counts = [-(-n // bs) for n in lens]
    total = sum(counts) + spare
    ids = torch.randperm(total, generator=g, device=DEVICE).int()
    mb = max(1, max(counts))
    at = torch.zeros(len(lens), mb, dtype=torch.int64)
    mask = torch.zeros(len(lens), mb, dtype=torch.bool)
    start = 0
    for i, n in enumerate(counts):
        at[i, :n] = torch.arange(start, start + n)
        mask[i, :n] = True
        start += n
    return torch.where(mask.to(DEVICE), ids[at.to(DEVICE)], torch.zeros((), dtype=torch.int32, device=DEVICE)).contiguous(), total


def _cos_sin(rotary):
    """[MAX_POSITION, rotary]: cosines, then sines, of position / 10000^(2i / rotary); angles in fp64."""
    i = torch.arange(rotary // 2, dtype=torch.float64, device=DEVICE)
    angle = torch.arange(MAX_POSITION, dtype=torch.float64, device=DEVICE)[:, None] * 10000.0 ** (-2.0 * i / rotary)
    return torch.cat([angle.cos(), angle.sin()], dim=1).float().contiguous()


def _qkv(g, case, tokens):
    """query, key, value of `tokens` tokens: slices of one projection's output, or tensors of their own."""
    h, hk, d = case["heads"], case["kv_heads"], case["head_size"]
    if case.get("strided", True):
        qkv = _randn(g, tokens, h + 2 * hk, d)
        return qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
    return _randn(g, tokens, h, d), _randn(g, tokens, hk, d), _randn(g, tokens, hk, d)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    op, bs = case["op"], case["block"]
    s = {"case": case}
    if op == "rope":
        t = case["tokens"]
        s["query"], s["key"], s["value"] = _qkv(g, case, t)
        blocks = -(-t // bs) + 8
        s["key_cache"], s["k_scale"] = _pool(g, case, blocks, case["kv_heads"])
        s["value_cache"], s["v_scale"] = _pool(g, case, blocks, case["kv_heads"])
        if case["prompt"]:  # consecutive positions, block after block
            at = torch.arange(t, device=DEVICE)
            s["slots"] = torch.randperm(blocks, generator=g, device=DEVICE)[at // bs] * bs + at % bs
            s["positions"] = (at + int(torch.randint(0, MAX_POSITION - t, (1,), generator=g, device=DEVICE))).contiguous()
        else:  # one token each of many sequences
            s["slots"] = torch.randperm(blocks * bs, generator=g, device=DEVICE)[:t].contiguous()
            s["positions"] = torch.randint(0, MAX_POSITION, (t,), generator=g, device=DEVICE)
        if case["padded"]:
            s["slots"][t - case["padded"]:] = -1
        s["cos_sin"] = _cos_sin(case["rotary"])
        s["query_out"] = torch.zeros(t, case["heads"], case["head_size"], dtype=torch.float16, device=DEVICE)
        return s
    if op == "append":
        old, new = _append_lens(case)
        t = sum(new)
        s["query"], s["key"], s["value"] = _qkv(g, case, t)
        # the pool holds the blocks that the call can touch: those from the first new token on
        held = [o % bs for o in old]
        tails, total = _tables(g, [h + n for h, n in zip(held, new)], bs, 4)
        skip = torch.tensor([o // bs for o in old])
        mb = int((skip + torch.tensor([-(-(h + n) // bs) for h, n in zip(held, new)])).max())
        col = torch.arange(mb)[None, :] - skip[:, None]
        inside = (col >= 0) & (col < tails.size(1))
        picked = tails.cpu().gather(1, col.clamp(0, tails.size(1) - 1))
        s["block_tables"] = torch.where(inside, picked, torch.zeros((), dtype=torch.int32)).to(DEVICE).contiguous()
        s["context_lens"] = torch.tensor([o + n for o, n in zip(old, new)], dtype=torch.int32, device=DEVICE)
        s["cu_tokens"] = torch.tensor([0] + new, device=DEVICE).cumsum(0).int()
        s["one_each"] = case["new_hi"] == 1
        s["key_cache"], s["k_scale"] = _pool(g, case, total, case["kv_heads"])
        s["value_cache"], s["v_scale"] = _pool(g, case, total, case["kv_heads"])
        s["cos_sin"] = _cos_sin(case["rotary"]) if case["rotary"] else None
        s["query_out"] = torch.zeros(t, case["heads"], case["head_size"], dtype=torch.float16, device=DEVICE) if case["heads"] else None
        if case["cache"] == "int8":
            s["values"] = torch.empty(2, *s["key_cache"].shape, dtype=torch.float16, device=DEVICE)
        return s
    lens = _ctx_lens(case)
    n, d, h, hk = len(lens), case["head_size"], case["heads"], case["kv_heads"]
    s["context_lens"] = torch.tensor(lens, dtype=torch.int32, device=DEVICE)
    s["max_ctx"] = max(lens)
    s["block_tables"], total = _tables(g, lens, bs, 2)
    if op == "int8":
        kind = dict(case, cache="int8", scales="block")
        s["key_cache"], s["k_scale"] = _pool(g, kind, total, hk)
        s["value_cache"], s["v_scale"] = _pool(g, kind, total, hk)
        s["query"] = _randn(g, n, h, d)
        parts = max(1, -(-s["max_ctx"] // (512 if d == 128 else 256)))
        s["max_logits"] = torch.empty(n, h, parts, dtype=torch.float32, device=DEVICE)
        s["exp_sums"] = torch.empty(n, h, parts, dtype=torch.float32, device=DEVICE)
        s["tmp"] = torch.empty(n, h, parts, d, dtype=torch.float16, device=DEVICE)
        s["out"] = torch.empty(n, h, d, dtype=torch.float16, device=DEVICE)
        s["alibi"] = torch.ones(h, dtype=torch.float32, device=DEVICE)
        return s
    s["key_cache"], s["k_scale"] = _pool(g, case, total, 2 * hk)
    s["value_cache"], s["v_scale"] = _pool(g, case, total, 2 * hk)
    s["query"] = _randn(g, n, 2 * h, d)
    s["lambdas"] = torch.rand(h, generator=g, device=DEVICE) * 0.6 + 0.2
    s["norm_weight"] = torch.rand(2 * d, generator=g, device=DEVICE) + 0.5 if case["norm"] else None
    s["out"] = torch.empty(n, h, 2 * d, dtype=torch.float16, device=DEVICE)
    return s


# ------------------------------------------------------------------------------------ the plain forms
NORM_EPS, NORM_SCALE = 1e-5, 0.2


def _rotated(x, cos_sin, positions, interleaved):
    """x [T, heads, D] with its first `rotary` dims rotated, in fp32."""
    r = cos_sin.size(1)
    cs = cos_sin[positions]
    cos, sin = cs[:, None, :r // 2], cs[:, None, r // 2:]
    y = x.float()
    if interleaved:
        a, b = y[..., 0:r:2], y[..., 1:r:2]
    else:
        a, b = y[..., :r // 2], y[..., r // 2:r]
    c, e = a * cos - b * sin, b * cos + a * sin
    front = torch.stack([c, e], dim=-1).flatten(-2) if interleaved else torch.cat([c, e], dim=-1)
    return torch.cat([front, y[..., r:]], dim=-1)


def _bytes(t):
    return t if t.dtype == torch.float16 else t.view(torch.uint8)


def _plain_rope(s):
    case, cache = s["case"], s["case"]["cache"]
    live = s["slots"][:case["tokens"] - case["padded"]]  # padding rows come last in these cases
    n, pos = live.numel(), s["positions"][:live.numel()]
    if case["heads"]:
        s["query_out"][:n] = _rotated(s["query"][:n], s["cos_sin"], pos, case["interleaved"]).half()
    rows = (_rotated(s["key"][:n], s["cos_sin"], pos, case["interleaved"]), s["value"][:n].float())
    for x, pool, scale in zip(rows, (s["key_cache"], s["value_cache"]), (s["k_scale"], s["v_scale"])):
        if cache == "fp16":
            codes = x.half()
        else:
            of = scale[None] if case["scales"] == "head" else scale[live // case["block"]]
            codes = _rows_to_codes(x, cache, of[..., None])
        _bytes(pool).view(-1, *pool.shape[2:])[live] = _bytes(codes)


def _plain_append(s):
    case, cache, bs = s["case"], s["case"]["cache"], s["case"]["block"]
    cu, ctx, bt = s["cu_tokens"].long(), s["context_lens"].long(), s["block_tables"].long()
    t = torch.arange(s["key"].size(0), device=DEVICE)
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    pos = ctx[seq] - cu[seq + 1] + t
    block, row = bt[seq, pos // bs], pos % bs
    k, v = s["key"].float(), s["value"].float()
    if s["cos_sin"] is not None:
        k = _rotated(s["key"], s["cos_sin"], pos, case["interleaved"])
        if case["heads"]:
            s["query_out"].copy_(_rotated(s["query"], s["cos_sin"], pos, case["interleaved"]))
    qmax = torch.full((), QMAX[cache], device=DEVICE)
    for x, pool, scale in ((k, s["key_cache"], s["k_scale"]), (v, s["value_cache"], s["v_scale"])):
        nb, hk = scale.shape
        first = torch.full((nb,), bs, device=DEVICE).scatter_reduce(0, block, row, "amin")
        amax = torch.zeros(nb, hk, device=DEVICE).scatter_reduce(0, block[:, None].expand(-1, hk), x.abs().amax(-1), "amax")
        held = torch.where((first == 0)[:, None], torch.zeros_like(scale), scale)
        grown = torch.where((first < bs)[:, None], torch.maximum(held, amax / qmax), scale)
        # rows that a touched block held before are stored again under its new scale
        old = (torch.arange(bs, device=DEVICE)[None] < first[:, None]) & (first < bs)[:, None] & (first > 0)[:, None]
        again = pool.float() * scale[:, None, :, None] / torch.where(grown == 0, torch.ones_like(grown), grown)[:, None, :, None]
        again = again.clamp(-QMAX[cache], QMAX[cache])
        again = again.round().to(torch.int8) if cache == "int8" else again.to(DTYPES[cache])
        codes = _bytes(pool)
        codes.copy_(torch.where(old[:, :, None, None], _bytes(again), codes))
        of = grown[block][..., None]
        codes.view(-1, *pool.shape[2:])[block * bs + row] = _bytes(_rows_to_codes(x, cache, torch.where(of == 0, torch.ones_like(of), of)))
        scale.copy_(grown)


def _gathered(s, pool, scale):
    """[S, T, heads, D] fp32: the first T = longest context tokens of every sequence."""
    bs = pool.size(1)
    ids = s["block_tables"][:, :max(1, -(-s["max_ctx"] // bs))].long()
    x = _bytes(pool)[ids]
    x = (x if pool.dtype == torch.float16 else x.view(pool.dtype)).float()  # [S, MB, bs, heads, D]
    if scale is not None:
        x *= scale[ids][:, :, None, :, None] if scale.dim() == 2 else scale[:, None]
    return x.flatten(1, 2)


def _weights(scores, context_lens):
    """softmax over the tokens inside each context; an empty context has no weights (zeros)."""
    inside = torch.arange(scores.size(-1), device=DEVICE) < context_lens.view(-1, *[1] * (scores.dim() - 1))
    scores = torch.where(inside, scores, torch.full((), -math.inf, device=DEVICE))
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _plain_int8(s):
    q = s["query"]
    n, h, d = q.shape
    k, v = _gathered(s, s["key_cache"], s["k_scale"]), _gathered(s, s["value_cache"], s["v_scale"])
    hk = k.size(2)
    scores = torch.matmul(q.float().view(n, hk, h // hk, d) * d ** -0.5, k.permute(0, 2, 3, 1))
    return torch.matmul(_weights(scores, s["context_lens"]), v.transpose(1, 2)).reshape(n, h, d).half()


def _plain_diff(s):
    q, case = s["query"], s["case"]
    n, d, h, hk = q.size(0), case["head_size"], case["heads"], case["kv_heads"]
    k, v = _gathered(s, s["key_cache"], s["k_scale"]), _gathered(s, s["value_cache"], s["v_scale"])
    t = k.size(1)
    q = q.float().view(n, hk, h // hk, 2, d).transpose(2, 3) * d ** -0.5  # [S, pair, map, group, D]
    scores = torch.matmul(q, k.view(n, t, hk, 2, d).permute(0, 2, 3, 4, 1))
    maps = _weights(scores, s["context_lens"])
    p = maps[:, :, 0] - s["lambdas"].view(hk, h // hk, 1) * maps[:, :, 1]
    o = torch.matmul(p, v.view(n, t, hk, 2 * d).transpose(1, 2)).reshape(n, h, 2 * d)
    if s["norm_weight"] is not None:
        o = o * torch.rsqrt((o * o).mean(-1, keepdim=True) + NORM_EPS) * s["norm_weight"] * NORM_SCALE
    return o.half()


# ------------------------------------------------------------------------------------ one pass
def _scales(s, kind):
    if s["k_scale"] is None:
        return {}
    return {f"k_scale_per_{kind}": s["k_scale"], f"v_scale_per_{kind}": s["v_scale"]}


def _own(s):
    from flash_attention_factory_b200 import cache_ops
    from flash_attention_factory_b200.lib import paged_attention_diff, paged_attention_int8_loop, paged_attention_int8_reduce

    case = s["case"]
    if case["op"] == "rope":
        cache_ops.rope_and_cache(s["query"], s["key"], s["value"], s["positions"], s["cos_sin"], s["query_out"],
                                 s["key_cache"], s["value_cache"], s["slots"], interleaved=case["interleaved"],
                                 **_scales(s, case["scales"]))
        return None
    if case["op"] == "append":
        cache_ops.append_block_scaled(s["key"], s["value"], s["key_cache"], s["value_cache"], s["k_scale"], s["v_scale"],
                                      s["block_tables"], s["context_lens"],
                                      cu_tokens=None if s["one_each"] else s["cu_tokens"],
                                      query=s["query"] if case["heads"] else None, query_out=s["query_out"],
                                      cos_sin=s["cos_sin"], interleaved=case["interleaved"])
        return None
    d, bs = case["head_size"], case["block"]
    if case["op"] == "int8":
        module = paged_attention_int8_loop if case["variant"] == "loop" else paged_attention_int8_reduce
        module.enqueue(s["max_logits"], s["exp_sums"], s["tmp"], s["out"], None, s["query"], s["key_cache"],
                       s["value_cache"], s["block_tables"], s["context_lens"], case["heads"] // case["kv_heads"],
                       d ** -0.5, 1.0, bs, s["max_ctx"], s["alibi"], None, -1.0, **_scales(s, "block"))
        return s["out"]
    if "scratch" not in s:  # kept by a program for as long as its batch has this shape
        s["scratch"] = paged_attention_diff.scratch(s["query"], s["key_cache"], s["max_ctx"])
    paged_attention_diff.enqueue(*s["scratch"], s["out"], s["query"], s["key_cache"], s["value_cache"],
                                 s["block_tables"], s["context_lens"], s["lambdas"], d ** -0.5, 1.0, bs, s["max_ctx"],
                                 norm_weight=s["norm_weight"], norm_eps=NORM_EPS, norm_scale=NORM_SCALE,
                                 **_scales(s, case["scales"]))
    return s["out"]


def _standing(s, pool, scale, k):
    """What a cache holds: FP8 and fp16 values themselves (scales are outputs or inputs beside them), int8 codes times scale."""
    if pool.dtype != torch.int8:
        return pool
    of = scale[:, None, :, None] if scale.dim() == 2 else scale[:, None]
    if "values" in s:
        return torch.mul(pool, of, out=s["values"][k])
    return (pool * of).half()


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        out = _own(s)
    else:
        out = {"rope": _plain_rope, "append": _plain_append, "int8": _plain_int8, "diff": _plain_diff}[op](s)
    if op in ("int8", "diff"):
        return {"out": out}
    got = {"key_cache": _standing(s, s["key_cache"], s["k_scale"], 0), "value_cache": _standing(s, s["value_cache"], s["v_scale"], 1)}
    if s["query_out"] is not None:
        got["query"] = s["query_out"]
    if op == "append":
        got["k_scale"], got["v_scale"] = s["k_scale"], s["v_scale"]
    return got


# ------------------------------------------------------------------------------------ fp64
def _grid(x, cache):
    """fp64 values -> the nearest value that the type holds (ties to even), saturating."""
    if cache == "fp16":
        return x.half().double()
    if cache == "int8":
        return x.round().clamp(-127, 127)
    bits, low = (3, -6) if cache == "e4m3" else (2, -14)
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** low)))
    e = torch.where(2.0 ** e > x.abs().clamp(min=2.0 ** low), e - 1, e)
    step = 2.0 ** (e - bits)
    return ((x / step).round() * step).clamp(-QMAX[cache], QMAX[cache])


def _turned(x, rotary, positions, interleaved, cos_sin):
    """Rotation as a product of complex numbers, fp64."""
    x = x.double()
    unit = torch.complex(*cos_sin[positions].double().view(len(positions), 1, 2, rotary // 2).unbind(2))
    front = x[..., :rotary]
    pairs = front.unflatten(-1, (rotary // 2, 2)) if interleaved else front.unflatten(-1, (2, rotary // 2)).transpose(-1, -2)
    z = torch.view_as_complex(pairs.contiguous()) * unit
    z = torch.view_as_real(z)
    z = z.flatten(-2) if interleaved else z.transpose(-1, -2).flatten(-2)
    return torch.cat([z, x[..., rotary:]], dim=-1)


def _exact_rope(case, s):
    live = [i for i, slot in enumerate(s["slots"].tolist()) if slot >= 0]
    at = torch.tensor(live, device=DEVICE)
    slot, pos = s["slots"][at], s["positions"][at]
    q = s["query_out"].double()
    q[at] = _turned(s["query"][at], case["rotary"], pos, case["interleaved"], s["cos_sin"])
    got = {"query": q}
    rows = {"key_cache": _turned(s["key"][at], case["rotary"], pos, case["interleaved"], s["cos_sin"]), "value_cache": s["value"][at].double()}
    for name, x in rows.items():
        pool, scale = s[name], s[name[0] + "_scale"]
        whole = pool.double()
        if scale is not None:
            per = scale.double().expand(pool.size(0), -1) if scale.dim() == 1 else scale.double()
            x = _grid(x / per[slot // case["block"]][..., None], case["cache"])
        whole.view(-1, *pool.shape[2:])[slot] = x
        if case["cache"] == "int8":
            whole *= per[:, None, :, None]
        got[name] = whole
    return got


def _exact_append(case, s):
    old, new = _append_lens(case)
    bs, cache = case["block"], case["cache"]
    table, start, got = s["block_tables"].cpu(), 0, {}
    pools = {n: s[n + "_cache"].double() for n in ("key", "value")}
    scales = {n: s[n[0] + "_scale"].double() for n in ("key", "value")}
    pos = torch.cat([torch.arange(o, o + n) for o, n in zip(old, new)]).to(DEVICE)
    rows = {"key": s["key"].double(), "value": s["value"].double()}
    if case["rotary"]:
        rows["key"] = _turned(s["key"], case["rotary"], pos, case["interleaved"], s["cos_sin"])
        if case["heads"]:
            got["query"] = _turned(s["query"], case["rotary"], pos, case["interleaved"], s["cos_sin"])
    for i, (o, n) in enumerate(zip(old, new)):
        p = o
        while p < o + n:
            block, r0 = int(table[i, p // bs]), p % bs
            count = min(bs - r0, o + n - p)
            for name in ("key", "value"):
                x = rows[name][start + p - o:start + p - o + count]  # [count, HK, D]
                top = x.abs().amax(dim=(0, 2)) / QMAX[cache]
                before = scales[name][block].clone() if r0 else torch.zeros_like(top)
                after = torch.maximum(before, top)
                by = torch.where(after == 0, torch.ones_like(after), after)[:, None]
                pool = pools[name][block]
                if r0:
                    kept = _grid(pool[:r0] * before[:, None] / by, cache)
                    pool[:r0] = torch.where((after > before)[:, None], kept, pool[:r0])
                pool[r0:r0 + count] = _grid(x / by, cache)
                scales[name][block] = after
            p += count
        start += n
    for name in ("key", "value"):
        got[name + "_cache"] = pools[name] * scales[name][:, None, :, None] if cache == "int8" else pools[name]
        got[name[0] + "_scale"] = scales[name]
    return got


def _tokens(s, pool, scale, i, n):
    bs = pool.size(1)
    ids = s["block_tables"][i, :-(-n // bs)].long()
    x = (pool if pool.dtype == torch.float16 else pool.view(torch.uint8))[ids]
    x = (x if pool.dtype == torch.float16 else x.view(pool.dtype)).double()
    if scale is not None:
        x = x * (scale.double()[ids][:, None, :, None] if scale.dim() == 2 else scale.double()[:, None])
    return x.flatten(0, 1)[:n]


def _exact_attention(case, s):
    lens, d, h, hk = _ctx_lens(case), case["head_size"], case["heads"], case["kv_heads"]
    g = h // hk
    diff = case["op"] == "diff"
    out = torch.zeros(len(lens), h, 2 * d if diff else d, dtype=torch.float64, device=DEVICE)
    for i, n in enumerate(lens):
        if n == 0:
            continue
        k, v = _tokens(s, s["key_cache"], s["k_scale"], i, n), _tokens(s, s["value_cache"], s["v_scale"], i, n)
        q = s["query"][i].double() / math.sqrt(d)
        if not diff:
            p = torch.softmax(torch.einsum("kgd,tkd->kgt", q.view(hk, g, d), k), dim=-1)
            out[i] = torch.einsum("kgt,tkd->kgd", p, v).reshape(h, d)
            continue
        p = torch.softmax(torch.einsum("kgcd,tkcd->ckgt", q.view(hk, g, 2, d), k.view(n, hk, 2, d)), dim=-1)
        o = torch.einsum("ckgt,tke->ckge", p, v.view(n, hk, 2 * d)).reshape(2, h, 2 * d)
        out[i] = o[0] - s["lambdas"].double()[:, None] * o[1]
    if diff and case["norm"]:
        out = out / torch.sqrt(out.square().mean(-1, keepdim=True) + NORM_EPS) * s["norm_weight"].double() * NORM_SCALE
    return {"out": out}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rope(case, s)
    if case["op"] == "append":
        return _exact_append(case, s)
    return _exact_attention(case, s)
