"""Calls of the paged operators at the edges of what they take."""

import pytest
import torch

from megabake_b200 import paged_append, paged_kv_attention, paged_prefill_attention
from tests import paged_reference as reference
from tests.test_gpu_paged import BF16, FP16, Cache, _check, _int32, _normal

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]


@pytest.mark.parametrize("heads,width", [((4, 2, 64), 8), ((4, 2, 64), 60), ((5, 1, 128), 60), ((2, 1, 256), 60)])
@pytest.mark.parametrize("first", [1, 7, 300])
def test_prompt_queries_before_the_first_request(heads, width, first):
    """Queries of no request are zero in a new output on both sides of the requests, and stay in one that is given."""
    count, kv_heads, dim = heads
    cache = Cache([50, 33], kv_heads, dim, 16, BF16, first)
    cache.table = torch.nn.functional.pad(cache.table, (0, width - cache.table.shape[1]), value=-1).contiguous()
    tokens = first + 30 + 21 + 4
    query = _normal((tokens, count, dim), cache.g, BF16)
    offsets = _int32([first, first + 30, first + 51])
    junk = torch.full_like(query, float("nan"))   # what the allocator hands out next
    del junk
    new = paged_prefill_attention(query, *cache.pools, cache.table, cache.lengths, offsets)
    given = paged_prefill_attention(query, *cache.pools, cache.table, cache.lengths, offsets, out=torch.full_like(query, 5.0))
    assert new[:first].eq(0).all() and new[first + 51:].eq(0).all()
    assert given[:first].eq(5).all() and given[first + 51:].eq(5).all()
    assert torch.equal(new[first:first + 51], given[first:first + 51])
    for r, at, n, length in ((0, first, 30, 50), (1, first + 30, 21, 33)):
        for j in (0, n // 2, n - 1):
            keys = length - n + j + 1
            expected = reference.attend(query[at + j], *cache.pools, cache.table[r], keys, dim ** -0.5)
            _check(new[at + j], expected, keys, BF16, reference.prompt_rounding(BF16))


def test_prompt_requests_that_end_before_the_last_row():
    """Requests without queries at the end of the table; all queries belong to none."""
    cache = Cache([50, 33, 20], 2, 64, 16, BF16, 0)
    query = _normal((40, 4, 64), cache.g, BF16)
    out = paged_prefill_attention(query, *cache.pools, cache.table, cache.lengths, _int32([5, 9, 9, 9]))
    assert out[:5].eq(0).all() and out[9:].eq(0).all() and not out[5:9].eq(0).all(-1).any()
    out = paged_prefill_attention(query, *cache.pools, cache.table, cache.lengths, _int32([40, 40, 40, 40]))
    assert out.eq(0).all()
    out = paged_prefill_attention(query, *cache.pools, cache.table, cache.lengths, _int32([0, 0, 0, 0]))
    assert out.eq(0).all()


@pytest.mark.parametrize("heads", [(34, 2, 128), (9, 3, 64), (5, 1, 128), (24, 1, 64), (7, 1, 256)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_prompt_bits_do_not_depend_on_rows_of_no_query(heads, dtype):
    """128 rows of a tile are not a multiple of these groups, and requests end inside of tiles: what lies in the rows that are
    left over, from an earlier launch or of the next request, changes nothing."""
    count, kv_heads, dim = heads
    cache = Cache([5000, 700], kv_heads, dim, 16, dtype, count)
    query = _normal((59, count, dim), cache.g, dtype)
    offsets = _int32([0, 39, 59])
    full = _normal((600, 128 * kv_heads, dim), cache.g, dtype)     # fills every row of a tile
    results = []
    for factor in (0.0, 1.0, 30.0, -30.0, 1000.0):
        paged_prefill_attention(full * factor, *cache.pools, cache.table, cache.lengths, _int32([0, 600, 600]))
        results.append(paged_prefill_attention(query, *cache.pools, cache.table, cache.lengths, offsets))
        other = query.clone()
        other[39:] *= factor
        results.append(paged_prefill_attention(other, *cache.pools, cache.table, cache.lengths, offsets))
    for result in results[1:]:
        assert torch.equal(result[:39], results[0][:39])
    for result in results[2::2]:
        assert torch.equal(result, results[0])


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_strides_of_single_places_mean_nothing(dim):
    """One token of one request with one key head, on one page: strides of these dimensions are any numbers."""
    g = torch.Generator(device="cuda").manual_seed(dim)

    def odd(x, strides):
        flat = torch.empty(x.numel() + 64, dtype=x.dtype, device="cuda")
        return flat.as_strided(x.shape, strides).copy_(x)

    query, key, value = (_normal((1, n, dim), g, BF16) for n in (3, 1, 1))
    pools = [_normal((1, 16, 1, dim), g, BF16) for _ in range(2)]
    table, lengths, offsets, slots = _int32([[0]]), _int32([9]), _int32([0, 1]), torch.tensor([8], device="cuda")
    results = []
    for again in (False, True):
        p = [x.clone() for x in pools]
        q, k, v = query, key, value
        if again:
            p = [odd(x, (3, dim, 7, 1)) for x in p]
            q, k, v = odd(q, (3 * dim + 1, dim, 1)), odd(k, (5, 2 * dim + 3, 1)), odd(v, (1, 1, 1))
        out = paged_kv_attention(q, k, v, *p, table, lengths)
        paged_append(v, k, *p, slots)
        results.append([out, paged_prefill_attention(q, *p, table, lengths, offsets), *p])
    for one, other in zip(*results):
        assert torch.equal(one, other)


def test_queries_that_are_broadcast():
    """One query for all heads, or for all tokens: strides of zero."""
    cache = Cache([200, 700], 2, 64, 16, BF16, 1)
    offsets = _int32([0, 10, 30])
    for shape in ((1, 4, 64), (30, 1, 64)):
        query = _normal(shape, cache.g, BF16).expand(30, 4, 64)
        for call in (lambda q: paged_prefill_attention(q, *cache.pools, cache.table, cache.lengths, offsets),
                     lambda q: paged_kv_attention(q[:2], q[:2, :2], q[:2, 2:], *cache.clone(), cache.table, cache.lengths)):
            assert torch.equal(call(query), call(query.contiguous()))
