"""NaN and infinities where the work of a paged operator is cut, against the definition."""

import pytest
import torch

from megabake_b200 import paged_kv_attention, paged_prefill_attention
from tests import paged_reference as reference
from tests.test_gpu_paged import BF16, FP16, Cache, _check, _int32, _normal

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]

CUT = [(4, 2, 64), (8, 2, 128), (4, 1, 256)]   # in tables of some thousand tokens


def _put(cache, pool, positions, value):
    for position in positions:
        slot = cache.slots[0][position]
        cache.pools[pool][slot // cache.page, slot % cache.page] = value


@pytest.mark.parametrize("new", [4, 300])
@pytest.mark.parametrize("heads", CUT)
def test_prompt_queries_that_are_nan_where_units_are_cut(heads, new):
    count, kv_heads, dim = heads
    cache = Cache([4000], kv_heads, dim, 64, BF16, new)
    query = _normal((new, count, dim), cache.g, BF16)
    bad = [1, new - 2]
    query[bad, 0, 5] = float("nan")
    out = paged_prefill_attention(query, *cache.pools, cache.table, cache.lengths, _int32([0, new]))
    for t in sorted({0, 1, 2, new // 2, new - 3, new - 2, new - 1}):
        expected = reference.attend(query[t], *cache.pools, cache.table[0], 4000 - new + t + 1, dim ** -0.5)
        first = 1 if t in bad else 0
        if first:
            assert out[t, 0].isnan().all(), t
        _check(out[t, first:], tuple(x[first:] for x in expected), 4000, BF16, reference.prompt_rounding(BF16))


@pytest.mark.parametrize("first,end", [(256, 512), (256, 768), (1024, 2560), (0, 700), (3000, 3990)])
@pytest.mark.parametrize("heads", [(4, 1, 64), (8, 1, 128), (2, 1, 256), (4, 2, 64)])
def test_prompt_runs_of_nan_keys(heads, first, end):
    """A CTA's share of this unit is 256 keys: whole pieces have no other scores."""
    count, kv_heads, dim = heads
    cache = Cache([4000], kv_heads, dim, 64, BF16, first)
    _put(cache, 0, range(first, end), float("nan"))
    query = _normal((5, count, dim), cache.g, BF16)
    out = paged_prefill_attention(query, *cache.pools, cache.table, cache.lengths, _int32([0, 5]))
    assert out.isnan().all()
    assert paged_kv_attention(query[:1], None, None, *cache.pools, cache.table, cache.lengths).isnan().all()


@pytest.mark.parametrize("heads", CUT)
def test_prompt_pieces_without_weight(heads):
    """Scores of minus infinity all over whole pieces: keys without weight, as if they were not there."""
    count, kv_heads, dim = heads
    cache = Cache([4000], kv_heads, dim, 64, BF16, 3)
    query = _normal((5, count, dim), cache.g, BF16).abs() + 0.5
    entries = 20 * 64, 50 * 64
    without = cache.table.clone()
    without[0, 20:50] = -1
    _put(cache, 0, range(*entries), -float("inf"))
    out = paged_prefill_attention(query, *cache.pools, cache.table, cache.lengths, _int32([0, 5]))
    for t in range(5):
        expected = reference.attend(query[t], *cache.pools, without[0], 4000 - 5 + t + 1, dim ** -0.5)
        _check(out[t], expected, 4000, BF16, reference.prompt_rounding(BF16))


@pytest.mark.parametrize("heads,cached", [((4, 2, 64), 40), ((9, 3, 64), 4000), ((32, 8, 128), 300), ((24, 1, 128), 3000),
                                          ((8, 1, 256), 2000), ((12, 1, 256), 90)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_decode_values_that_are_no_numbers(heads, cached, dtype):
    """Infinities and NaN among the values reach all queries of their key head, in their columns, and nobody else's:
    infinities as such, unless there are both.  (Weights here are far above what 16 bits resolve.)"""
    count, kv_heads, dim = heads
    cache = Cache([cached, cached], kv_heads, dim, 16, dtype, cached)
    query = _normal((2, count, dim), cache.g, dtype)
    inf, nan = float("inf"), float("nan")
    odd = {0: {1: inf, 2: -inf, 3: nan, 4: inf}, cached // 2: {4: -inf, 1: inf}, cached // 2 + 1: {dim - 1: -inf},
           cached - 1: {7: inf, dim - 2: nan}}
    odd.update({cached // 3 + i: {10 + i: inf if i % 2 else -inf} for i in range(10)})
    seen = {}
    for position, columns in odd.items():
        slot = cache.slots[0][position]
        for column, value in columns.items():
            cache.pools[1][slot // 16, slot % 16, kv_heads - 1, column] = value
            seen[column] = seen.get(column, 0.0) + value
    finite = [p.clone() for p in cache.pools]
    finite[1].nan_to_num_(0.0, 0.0, 0.0)
    out = paged_kv_attention(query, None, None, *cache.pools, cache.table, cache.lengths)
    mine = torch.arange(count, device="cuda") // (count // kv_heads) == kv_heads - 1
    for t in range(2):
        got, expected = out[t].clone(), reference.attend(query[t], *finite, cache.table[t], cached, dim ** -0.5)
        for column, value in seen.items() if t == 0 else ():
            there = got[mine, column]
            assert bool(there.isnan().all() if value != value else there.eq(value).all()), column
            got[mine, column] = expected[0][mine, column].to(dtype)
        _check(got, expected, cached, dtype, reference.decode_rounding(dtype))
