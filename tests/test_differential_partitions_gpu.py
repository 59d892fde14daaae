"""Differential attention over blocks of 128 tokens: a partition may not begin inside a copied box.

With 8-bit caches of head size 64 and an odd number of pairs a box holds 128 rows of one block; a partition
that began at row 64 of one would read the first half of the physically next block."""
import pytest

from _fp64 import check, paged_case
from test_differential_attention_gpu import learned, reference, run

@pytest.mark.gpu
@pytest.mark.parametrize("cache,scale", [("int8", "block"), ("e4m3", "block"), ("e5m2", "block"), ("int8", "head"),
                                         ("e4m3", "head"), ("e5m2", "head")])
@pytest.mark.parametrize("pairs", [1, 3])
def test_blocks_of_128_with_an_odd_number_of_pairs(cuda_device, cache, scale, pairs):
    """Scratch of few partitions and hints whose even share is 192, 320, 448 or 576 tokens, and the proposed ones."""
    lens = [1100, 0, 129, 700, 64, 1344, 193]
    case = paged_case(40 + pairs, lens, 4 * pairs, 2 * pairs, 64, 128, cache=cache, scale=scale, spread=4.0)
    lam, w = learned(2 * pairs, 64)
    want = reference(case, lam)
    for npart, hint in ((2, None), (3, None), (5, None), (7, None), (7, 1344), (3, 1344), (3, 576), (4, 1280), (None, None)):
        check(run(case, cuda_device, lam, npart=npart, hint=hint), *want, f"{cache} {scale} NP {npart} hint {hint}")
    check(run(case, cuda_device, lam, npart=7, norm_weight=w), *reference(case, lam, w), "with norm")


@pytest.mark.gpu
def test_proposed_scratch_of_a_long_batch(cuda_device):
    """8 sequences of up to 5000 tokens, one pair: the proposed scratch has 37 partitions of 192 tokens."""
    case = paged_case(44, [5000, 4321, 17, 900, 128, 2500, 3000, 4999], 4, 2, 64, 128, cache="e4m3", scale="block", spread=4.0)
    lam, _ = learned(2, 64)
    check(run(case, cuda_device, lam), *reference(case, lam), "proposed scratch")


@pytest.mark.parametrize("kv", [0, 1, 2, 3])
@pytest.mark.parametrize("d", [64, 128])
def test_partitions_begin_where_a_box_does(kv, d):
    """The rule alone, for every shape, many scratch sizes and hints; the proposed scratch among them."""
    from flash_attention_factory_b200 import _cabi, _test_aids, build

    build.build()
    propose = _cabi.load_library().pa_diff_num_partitions
    most_tiles = {0: {64: 2, 128: 1}}.get(kv, {64: 4, 128: 2})[d]
    seen = set()
    for bs in (16, 32, 64, 128):
        for pairs in (1, 2, 3, 4, 6):
            heads = 4 if pairs % 2 == 0 else 2
            for hint in (0, 1, 700, 1344, 5000, 40000, 2 ** 31):
                for npart in (1, 2, 3, 5, 7, 37, 200, propose(8, 2 * pairs, d, max(hint, 1), kv)):
                    p = _cabi.PaParams()
                    for name, value in dict(out=16, max_logits=16, exp_sums=16, tmp_out=16, query=16, key_cache=16, value_cache=16,
                                            block_tables=16, context_lens=16, num_seqs=8, num_heads=2 * pairs, head_size=d,
                                            num_kv_heads=2 * pairs, max_num_partitions=npart, max_blocks_per_seq=2 ** 20,
                                            block_size=bs, num_queries_per_tokens=1, num_blocks=64, sm_scale=0.1, fp8_scale=1.0,
                                            kv_dtype=kv, max_context_len=hint).items():
                        setattr(p, name, value)
                    tokens, rows = _test_aids.diff_split(p)
                    tiles = most_tiles
                    while tiles > 1 and 64 // heads * tiles > bs:
                        tiles //= 2
                    assert rows == min(bs, 64 // heads * tiles), (bs, pairs)
                    assert tokens % 64 == 0 and tokens % rows == 0, (bs, pairs, hint, npart, tokens, rows)
                    longest = min(hint or 2 ** 20 * bs, 2 ** 20 * bs, 2 ** 30)
                    assert tokens * npart >= longest and (tokens - max(64, rows)) * npart < longest
                    seen.add(rows)
    assert (128 in seen) == (kv != 0 and d == 64)
