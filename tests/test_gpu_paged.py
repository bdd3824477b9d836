"""The operators around a paged key-value cache against their definition in 64 bits."""

import random

import pytest
import torch

from megabake_b200 import PagedState, paged_append, paged_kv_attention, paged_prefill_attention, paged_reserve
from megabake_b200.diagnostics import CompilerError
from tests import paged_reference as reference

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]

BF16, FP16 = torch.bfloat16, torch.float16
HEADS = [(9, 3, 64), (14, 2, 64), (4, 4, 64), (32, 8, 128), (5, 1, 128), (8, 1, 256), (34, 2, 128), (24, 1, 64),
         (16, 1, 256)]


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _normal(shape, g, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


class Cache:
    """Pools whose every unused place holds NaN, and a table of scattered pages."""

    def __init__(self, lengths, kv_heads, dim, page, dtype, seed, layout="nhd"):
        self.g = g = torch.Generator(device="cuda").manual_seed(seed)
        held = [reference.pages_of(n, page) for n in lengths]
        self.pages = sum(held) + 3
        shape = (self.pages, page, kv_heads, dim) if layout == "nhd" else (self.pages, kv_heads, page, dim)
        self.pools = [torch.full(shape, float("nan"), dtype=dtype, device="cuda") for _ in range(2)]
        if layout == "hnd":
            self.pools = [p.transpose(1, 2) for p in self.pools]
        width = max(held) + 2
        order = torch.randperm(self.pages, generator=g, device="cuda").tolist()
        rows, self.slots = [], []
        for n, count in zip(lengths, held):
            mine, order = order[:count], order[count:]
            rows.append(mine + [-1] * (width - count))
            self.slots.append([mine[i // page] * page + i % page for i in range(n)])
        self.table, self.lengths = _int32(rows), _int32(lengths)
        self.page = page
        every = torch.tensor(sum(self.slots, []), dtype=torch.int64, device="cuda")
        for pool in self.pools:
            pool[every // page, every % page] = _normal((every.numel(), kv_heads, dim), g, dtype)

    def clone(self):
        """The pools as they are, in the same layout."""
        return [torch.empty_strided(p.shape, p.stride(), dtype=p.dtype, device="cuda").copy_(p) for p in self.pools]


def _check(out, expected, keys, dtype, rounding):
    bound = reference.tolerance(expected, keys, dtype, rounding)
    error = (out.double() - expected[0]).abs()
    assert torch.isfinite(out).all()
    assert bool((error <= bound).all()), f"{float((error / bound).max()):.3f} of the bound"


# ---------------------------------------------------------------------------------------
# Pages and slots
# ---------------------------------------------------------------------------------------
def _run_reserve(counts, state, page, max_tokens):
    lengths, table, stack, free = state
    tensors = [_int32(lengths), _int32(table), _int32(stack), _int32([free])]
    batch = paged_reserve(_int32(counts), *tensors, page, max_tokens)
    return ([t.tolist() for t in tensors[:3]] + [tensors[3].item()], [t.tolist() for t in batch])


@pytest.mark.parametrize("requests,width,page,pages", [(1, 1, 8, 1), (1, 40, 16, 64), (7, 5, 8, 30), (33, 9, 64, 200),
                                                       (300, 6, 8, 900), (1024, 3, 16, 2500), (1025, 4, 8, 3000),
                                                       (2048, 2, 8, 2500)])
def test_reserve_against_the_definition(requests, width, page, pages):
    rng = random.Random(requests)
    stack = list(range(pages))
    rng.shuffle(stack)
    state = ([0] * requests, [[-1] * width for _ in range(requests)], stack, pages)
    for step in range(12):
        most = width * page + 3
        counts = [rng.choice((0, 1, 1, rng.randint(-most, most), rng.randint(-most, 0))) for _ in range(requests)]
        max_tokens = rng.choice((0, 1, requests, requests * page, sum(max(c, 0) for c in counts)))
        got, batch = _run_reserve(counts, state, page, max_tokens)
        state, expected = reference.reserve(counts, *state, page, max_tokens)
        assert got == [list(state[0]), state[1], state[2], state[3]], step
        assert batch == [list(x) for x in expected], step


def test_reserve_gives_pages_back_before_it_grants():
    state = PagedState(1, 2, 64, 1, 64, page_size=16, pages=4, device="cuda")
    first = state.reserve(_int32([64, 1]), 80)
    assert first.granted.tolist() == [64, 0] and state.free_count.item() == 0
    second = state.reserve(_int32([-64, 64]), 80)
    assert second.granted.tolist() == [-64, 64] and state.lengths.tolist() == [0, 64]
    assert second.rows.tolist() == [1] * 64 + [-1] * 16 and second.offsets.tolist() == [0, 0, 64]


def test_reserve_extreme_counts():
    low, high = -2 ** 31, 2 ** 31 - 1
    state = PagedState(1, 4, 32, 1, 64, page_size=8, device="cuda")
    state.reserve(_int32([9, 9, 9, 9]), 36)
    batch = state.reserve(_int32([low, high, high, 2]), 5)
    assert batch.granted.tolist() == [-9, 0, 0, 2] and state.lengths.tolist() == [0, 9, 9, 11]


def test_reserve_with_a_broken_state_stays_in_its_tensors():
    """Ids that name no page and a free count beyond the stack: entries without a page, slots -1."""
    lengths, table = _int32([20, 500, -7]), _int32([[7, -3], [1, 2], [0, 0]])
    stack, free = _int32([5, 99]), _int32([40])
    batch = paged_reserve(_int32([3, -1, 2]), lengths, table, stack, free, 16, 8)
    assert batch.granted.tolist() == [3, -1, 2] and lengths.tolist() == [23, 31, 2]
    assert batch.slots.tolist() == [-1] * 8
    assert batch.positions.tolist() == [20, 21, 22, 0, 1, 0, 0, 0]


# ---------------------------------------------------------------------------------------
# Append
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("layout", ["nhd", "hnd"])
@pytest.mark.parametrize("tokens,kv_heads,dim,page,dtype", [(1, 1, 64, 8, BF16), (5, 3, 64, 16, FP16), (77, 2, 128, 64, BF16),
                                                            (1000, 8, 256, 1024, FP16), (3001, 5, 128, 32, BF16)])
def test_append(tokens, kv_heads, dim, page, dtype, layout):
    cache = Cache([tokens + 9], kv_heads, dim, page, dtype, tokens, layout)
    rng = random.Random(tokens)
    slots = rng.sample(cache.slots[0], tokens)
    for i in rng.sample(range(tokens), tokens // 4):
        slots[i] = rng.choice((-1, -2 ** 63, cache.pages * page, 2 ** 62))
    fused = _normal((tokens, 2 * kv_heads + 1, dim), cache.g, dtype)
    key, value = fused[:, :kv_heads], fused[:, kv_heads + 1:]
    expected = cache.clone()
    for t, slot in enumerate(slots):
        if 0 <= slot < cache.pages * page:
            expected[0][slot // page, slot % page] = key[t]
            expected[1][slot // page, slot % page] = value[t]
    paged_append(key, value, *cache.pools, torch.tensor(slots, dtype=torch.int64, device="cuda"))
    for got, want in zip(cache.pools, expected):
        assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))


def test_append_of_values_that_are_no_numbers():
    cache = Cache([8], 1, 64, 8, BF16, 0)
    key = torch.tensor([float("nan"), float("inf"), -float("inf"), -0.0], device="cuda").to(BF16).repeat(16).view(1, 1, 64)
    paged_append(key, key, *cache.pools, torch.tensor([3], device="cuda"))
    assert torch.equal(cache.pools[0][0, 3].view(torch.int16), key[0].view(torch.int16))


# ---------------------------------------------------------------------------------------
# One new token a request
# ---------------------------------------------------------------------------------------
def _decode_case(lengths, heads, page, dtype, seed, layout="nhd", append=True, rows=None, scale=None):
    count, kv_heads, dim = heads
    cache = Cache(lengths, kv_heads, dim, page, dtype, seed, layout)
    tokens = len(lengths) if rows is None else len(rows)
    fused = _normal((tokens, count + 2 * kv_heads, dim), cache.g, dtype)
    query, key, value = fused.split((count, kv_heads, kv_heads), dim=1)
    key, value = (key, value) if append else (None, None)
    before = cache.clone()
    out = paged_kv_attention(query, key, value, *cache.pools, cache.table, cache.lengths,
                             None if rows is None else _int32(rows), scale=scale)
    scale = dim ** -0.5 if scale is None else scale
    for t in range(tokens):
        r = t if rows is None else rows[t]
        if not 0 <= r < len(lengths) or lengths[r] == 0:
            assert out[t].eq(0).all()
            continue
        n = lengths[r]
        expected = reference.attend(query[t], *before, cache.table[r], n, scale,
                                    new_key=key[t] if append else None, new_value=value[t] if append else None)
        _check(out[t], expected, n, dtype, reference.decode_rounding(dtype))
        if append:
            slot = cache.slots[r][-1]
            before[0][slot // page, slot % page] = key[t]
            before[1][slot // page, slot % page] = value[t]
    for got, want in zip(cache.pools, before):
        assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))
    return out


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads", HEADS)
def test_decode_head_layouts(heads, dtype):
    _decode_case([1, 64, 0, 65, 130, 700], heads, 16, dtype, heads[0])


@pytest.mark.parametrize("length", [1, 2, 7, 8, 9, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 1023, 1025])
def test_decode_lengths(length):
    for heads, page in (((6, 2, 64), 8), ((4, 4, 128), 64), ((3, 1, 256), 32)):
        _decode_case([length], heads, page, BF16, length)


@pytest.mark.parametrize("layout", ["nhd", "hnd"])
@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256, 512, 1024])
def test_decode_pages(page, layout):
    _decode_case([page - 1, page, page + 1, 3 * page + 5, 1], (14, 2, 64), page, FP16, page, layout)
    _decode_case([2 * page + 1, 5], (2, 1, 256), page, BF16, page, layout)


def test_decode_many_requests():
    lengths = [(i * 37) % 300 for i in range(500)]
    _decode_case(lengths, (3, 1, 64), 16, BF16, 1)


@pytest.mark.parametrize("heads", [(4, 2, 64), (8, 1, 128), (2, 1, 256)])
def test_decode_long_contexts_are_shared_out(heads):
    _decode_case([20011, 3, 9001], heads, 64, BF16, 5)


def test_decode_rows_name_the_requests():
    _decode_case([5, 0, 90, 300, 17], (4, 2, 64), 16, BF16, 2, rows=[3, -1, 0, 4, 1, 5, 2, -2 ** 31, 2 ** 31 - 1])


def test_decode_without_new_keys_reads_a_request_twice():
    _decode_case([100, 33], (4, 2, 128), 16, BF16, 3, append=False, rows=[0, 1, 0, 0])


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 3.0])
def test_decode_scales(scale):
    _decode_case([200, 1], (4, 2, 64), 16, FP16, 4, scale=scale)


@pytest.mark.parametrize("append", [False, True])
def test_decode_skips_positions_without_a_page(append):
    lengths, heads, page = [200, 40, 16, 33], (4, 2, 64), 16
    cache = Cache(lengths, 2, 64, page, BF16, 8)
    cache.table[0, 2:5] = -1
    cache.table[0, 7] = cache.pages
    cache.table[0, 11] = 2 ** 31 - 1
    cache.table[1, 0] = -2 ** 31
    cache.table[2, 0] = -1             # nothing is left of this one
    cache.table[3, 2] = -1             # the last position, and with it the token's own key, has no place
    fused = _normal((4, 8, 64), cache.g, BF16)
    query, key, value = fused.split((4, 2, 2), dim=1)
    before = cache.clone()
    new = (key, value) if append else (None, None)
    out = paged_kv_attention(query, *new, *cache.pools, cache.table, cache.lengths)
    for t, n in enumerate(lengths):
        expected = reference.attend(query[t], *before, cache.table[t], n, 0.125,
                                    new_key=key[t] if append else None, new_value=value[t] if append else None)
        _check(out[t], expected, n, BF16, reference.decode_rounding(BF16))
    assert out[2].eq(0).all()
    for got, want, new_rows in zip(cache.pools, before, (key, value)):
        for t in (0, 1) if append else ():
            slot = cache.slots[t][-1]
            want[slot // page, slot % page] = new_rows[t]
        assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))


def test_decode_lengths_beyond_the_table():
    """More tokens than a row of the table can hold count as a full row; negative ones as none."""
    cache = Cache([64, 64], 1, 64, 16, BF16, 9)
    cache.table = cache.table[:, :4].contiguous()
    cache.lengths = _int32([2 ** 31 - 1, -5])
    query = _normal((2, 2, 64), cache.g, BF16)
    out = paged_kv_attention(query, None, None, *cache.pools, cache.table, cache.lengths)
    _check(out[0], reference.attend(query[0], *cache.pools, cache.table[0], 64, 0.125), 64, BF16,
           reference.decode_rounding(BF16))
    assert out[1].eq(0).all()


def test_decode_values_at_the_ends_of_the_range():
    """Scores far apart, equal scores, and the largest values: one key takes all, or all share."""
    cache = Cache([300], 1, 64, 16, BF16, 10)
    slots = torch.tensor(cache.slots[0], device="cuda")
    page, place = slots // 16, slots % 16
    query = torch.full((1, 1, 64), 100.0, dtype=BF16, device="cuda")
    for keys in (torch.linspace(-300, 300, 300, device="cuda"), torch.full((300,), -300.0, device="cuda")):
        cache.pools[0][page, place] = keys.to(BF16)[:, None, None].expand(300, 1, 64)
        cache.pools[1][page, place] = _normal((300, 1, 64), cache.g, BF16) * 1e37
        out = paged_kv_attention(query, None, None, *cache.pools, cache.table, cache.lengths)
        expected = reference.attend(query[0], *cache.pools, cache.table[0], 300, 0.125)
        if keys[0] != keys[-1]:
            assert torch.equal(out[0], expected[0].to(BF16))
        else:
            # equal scores, exactly: every weight is 1
            exact = (expected[0], expected[1], torch.zeros_like(expected[2]))
            _check(out[0], exact, 300, BF16, reference.decode_rounding(BF16))


def test_decode_infinities_and_nan():
    """A NaN among the keys makes the request's output NaN, and nobody else's; a score of minus infinity is a key
    without weight; a place behind the length has no say whatever it holds."""
    cache = Cache([20, 20, 20], 1, 64, 16, BF16, 11)
    query = _normal((3, 2, 64), cache.g, BF16).abs() + 0.5
    slots = [cache.slots[r][7] for r in range(3)]
    cache.pools[0][slots[0] // 16, slots[0] % 16] = float("nan")
    cache.pools[0][slots[1] // 16, slots[1] % 16] = -float("inf")
    behind = int(cache.table[2, 1]) * 16 + 20 % 16
    cache.pools[0][behind // 16, behind % 16] = float("inf")
    cache.pools[1][behind // 16, behind % 16] = -float("inf")
    out = paged_kv_attention(query, None, None, *cache.pools, cache.table, cache.lengths)
    assert out[0].isnan().all()
    finite = [p.clone() for p in cache.pools]
    kept = [i for i in range(20) if i != 7]
    order = [cache.slots[1][i] for i in kept]
    for pool, source in zip(finite, cache.pools):    # the same request without that key
        for i, slot in enumerate(order):
            at = cache.slots[1][i]
            pool[at // 16, at % 16] = source[slot // 16, slot % 16]
    _check(out[1], reference.attend(query[1], *finite, cache.table[1], 19, 0.125), 20, BF16,
           reference.decode_rounding(BF16))
    _check(out[2], reference.attend(query[2], *cache.pools, cache.table[2], 20, 0.125), 20, BF16,
           reference.decode_rounding(BF16))


# ---------------------------------------------------------------------------------------
# Several new tokens a request
# ---------------------------------------------------------------------------------------
def _prompt_case(new, cached, heads, page, dtype, seed, layout="nhd", extra=3, out=None, scale=None, holes=()):
    count, kv_heads, dim = heads
    lengths = [n + c for n, c in zip(new, cached)]
    cache = Cache(lengths, kv_heads, dim, page, dtype, seed, layout)
    for r, entry, value in holes:
        cache.table[r, entry] = value
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    query = _normal((offsets[-1] + extra, count + 1, dim), cache.g, dtype)[:, 1:]
    if out is not None:
        out = torch.full_like(query, out, memory_format=torch.contiguous_format)
    before = cache.clone()
    got = paged_prefill_attention(query, *cache.pools, cache.table, cache.lengths, _int32(offsets), scale=scale, out=out)
    scale = dim ** -0.5 if scale is None else scale
    for r, n in enumerate(new):
        for j in _some(n):
            keys = lengths[r] - n + j + 1
            expected = reference.attend(query[offsets[r] + j], *before, cache.table[r], keys, scale)
            _check(got[offsets[r] + j], expected, keys, dtype, reference.prompt_rounding(dtype))
    assert got[offsets[-1]:].eq(0.0 if out is None else out[-1, 0, 0]).all()
    for pool, want in zip(cache.pools, before):
        assert torch.equal(pool.nan_to_num(7.0), want.nan_to_num(7.0))
    return got


def _some(n):
    """All queries of a short prompt; of a long one those around the edges of tiles."""
    if n <= 40:
        return range(n)
    near = {e + d for e in range(0, n + 1, 16) for d in (-1, 0)} if n <= 300 else \
        {e + d for e in range(0, n + 1, 128) for d in (-1, 0, 1, 63, 64)}
    return sorted(i for i in near | {0, 1, n // 2, n - 2, n - 1} if 0 <= i < n)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads", HEADS)
def test_prompt_head_layouts(heads, dtype):
    _prompt_case([33, 1, 0, 150], [0, 70, 5, 200], heads, 16, dtype, heads[0])


@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 600])
def test_prompt_lengths(tokens):
    for heads, page in (((6, 2, 64), 8), ((4, 4, 128), 64), ((3, 1, 256), 32)):
        _prompt_case([tokens], [0], heads, page, BF16, tokens)


@pytest.mark.parametrize("cached", [1, 63, 64, 65, 127, 128, 129, 1000, 9000])
def test_prompt_after_a_cached_prefix(cached):
    for heads, page in (((8, 2, 64), 64), ((5, 1, 128), 16), ((8, 1, 256), 128)):
        _prompt_case([70], [cached], heads, page, BF16, cached)


@pytest.mark.parametrize("layout", ["nhd", "hnd"])
@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256, 512, 1024])
def test_prompt_pages(page, layout):
    _prompt_case([page - 1, page + 1, 5], [3, 0, 2 * page], (14, 2, 64), page, FP16, page, layout)
    _prompt_case([page + 3], [page], (2, 1, 256), page, BF16, page, layout)


def test_prompt_many_requests():
    new = [(i * 13) % 40 for i in range(300)]
    cached = [(i * 29) % 150 for i in range(300)]
    _prompt_case(new, cached, (3, 1, 64), 16, BF16, 1)


def test_prompt_long():
    _prompt_case([2500], [0], (4, 1, 128), 64, BF16, 2)
    _prompt_case([1200, 1300], [700, 0], (8, 8, 64), 64, FP16, 3)


def test_prompt_rows_behind_the_last_request():
    _prompt_case([20, 3], [0, 9], (4, 2, 64), 16, BF16, 4, extra=300)
    _prompt_case([20, 3], [0, 9], (4, 2, 64), 16, BF16, 4, extra=300, out=5.0)
    _prompt_case([0, 0], [40, 9], (4, 2, 64), 16, BF16, 5, extra=300, out=-2.0)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 3.0])
def test_prompt_scales(scale):
    _prompt_case([50], [20], (4, 2, 64), 16, FP16, 6, scale=scale)


def test_prompt_skips_positions_without_a_page():
    holes = [(0, 0, -1), (0, 3, 2 ** 31 - 1), (0, 9, -2 ** 31), (0, 20, 10 ** 6), (1, 0, -1), (1, 1, -1), (2, 0, -5)]
    _prompt_case([60, 20, 300], [300, 12, 0], (4, 2, 64), 16, BF16, 7, holes=holes)
    _prompt_case([60, 20, 300], [300, 12, 0], (2, 1, 256), 16, BF16, 7, holes=holes)


def test_prompt_with_more_queries_than_keys():
    """Queries before position 0 have no key: zeros."""
    cache = Cache([5, 40], 2, 64, 16, BF16, 12)
    query = _normal((50, 4, 64), cache.g, BF16)
    out = paged_prefill_attention(query, *cache.pools, cache.table, cache.lengths, _int32([0, 9, 50]))
    assert out[:4].eq(0).all() and out[9:10].eq(0).all()
    for t, r, keys in ((4, 0, 1), (8, 0, 5), (10, 1, 1), (49, 1, 40)):
        _check(out[t], reference.attend(query[t], *cache.pools, cache.table[r], keys, 0.125), keys, BF16,
               reference.prompt_rounding(BF16))


def test_prompt_lengths_beyond_the_table():
    cache = Cache([64, 64], 1, 64, 16, BF16, 9)
    cache.table = cache.table[:, :4].contiguous()
    cache.lengths = _int32([2 ** 31 - 1, -5])
    query = _normal((6, 2, 64), cache.g, BF16)
    out = paged_prefill_attention(query, *cache.pools, cache.table, cache.lengths, _int32([0, 3, 6]))
    for j in range(3):
        _check(out[j], reference.attend(query[j], *cache.pools, cache.table[0], 62 + j, 0.125), 64, BF16,
               reference.prompt_rounding(BF16))
    assert out[3:].eq(0).all()


def test_prompt_infinities_and_nan():
    cache = Cache([200, 200], 1, 64, 16, BF16, 13)
    query = _normal((200, 2, 64), cache.g, BF16)
    slot = cache.slots[0][150]
    cache.pools[0][slot // 16, slot % 16] = float("nan")
    out = paged_prefill_attention(query, *cache.pools, cache.table, cache.lengths, _int32([0, 100, 200]))
    assert out[50:100].isnan().all()              # positions 150 .. 199 see it
    assert out[:50].isfinite().all() and out[100:].isfinite().all()


@pytest.mark.parametrize("heads,new,cached", [((4, 2, 64), 200, 0), ((2, 1, 128), 40, 500), ((8, 1, 256), 50, 3),
                                              ((1, 1, 64), 300, 5000), ((4, 4, 128), 20, 0)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_prompt_values_that_are_no_numbers(heads, new, cached, dtype):
    """Infinities and NaN among the values reach the queries that see them, in their columns, and no others."""
    count, kv_heads, dim = heads
    cache = Cache([new + cached], kv_heads, dim, 16, dtype, new)
    query = _normal((new, count, dim), cache.g, dtype)
    odd = {cached + new // 2: {0: float("inf"), 33: float("nan")}, cached + new // 2 + 3: {0: -float("inf"), dim - 1: -float("inf")},
           cached + new - 1: {7: float("nan")}}
    if cached:
        odd[cached // 2] = {40: float("inf")}
    for position, columns in odd.items():
        slot = cache.slots[0][position]
        for column, value in columns.items():
            cache.pools[1][slot // 16, slot % 16, kv_heads - 1, column] = value
    out = paged_prefill_attention(query, *cache.pools, cache.table, cache.lengths, _int32([0, new]))
    finite = [p.clone() for p in cache.pools]
    finite[1].nan_to_num_(0.0, 0.0, 0.0)
    group = count // kv_heads
    mine = torch.arange(count, device="cuda") // group == kv_heads - 1
    for t in _some(new):
        seen = {}
        for position, columns in odd.items():
            if position <= cached + t:
                for column, value in columns.items():
                    seen[column] = seen.get(column, 0.0) + value
        got, expected = out[t].clone(), reference.attend(query[t], *finite, cache.table[0], cached + t + 1, dim ** -0.5)
        for column, value in seen.items():
            there = got[mine, column]
            assert bool(there.isnan().all() if value != value else there.eq(value).all()), (t, column)
            got[mine, column] = expected[0][mine, column].to(dtype)
        _check(got, expected, cached + t + 1, dtype, reference.prompt_rounding(dtype))


# ---------------------------------------------------------------------------------------
# Streams, graphs, devices, refusals
# ---------------------------------------------------------------------------------------
def test_offsets_beyond_32_bits():
    """Pages whose elements lie past 2^32 bytes and 2^31 elements of a pool."""
    page, kv_heads, dim = 1024, 8, 128
    pages = 2 ** 31 // (page * kv_heads * dim) + 70
    pools = [torch.zeros(pages, page, kv_heads, dim, dtype=BF16, device="cuda") for _ in range(2)]
    g = torch.Generator(device="cuda").manual_seed(0)
    high = pages - 3
    for pool in pools:
        pool[high:high + 2] = _normal((2, page, kv_heads, dim), g, BF16)
    table, lengths = _int32([[high + 1, high]]), _int32([1500])
    query = _normal((1, 8, dim), g, BF16)
    key, value = (_normal((1, kv_heads, dim), g, BF16) for _ in range(2))
    out = paged_kv_attention(query, key, value, *pools, table, lengths)
    assert torch.equal(pools[0][high, 1499 - 1024], key[0]) and torch.equal(pools[1][high, 1499 - 1024], value[0])
    _check(out[0], reference.attend(query[0], *pools, table[0], 1500, dim ** -0.5), 1500, BF16,
           reference.decode_rounding(BF16))
    out = paged_prefill_attention(query, *pools, table, lengths, _int32([0, 1]))
    _check(out[0], reference.attend(query[0], *pools, table[0], 1500, dim ** -0.5), 1500, BF16,
           reference.prompt_rounding(BF16))
    paged_append(value, key, *pools, torch.tensor([pages * page - 1], device="cuda"))
    assert torch.equal(pools[0][-1, -1], value[0]) and torch.equal(pools[1][-1, -1], key[0])


def _step_inputs(seed, lengths=(70, 9000, 0, 300), heads=(8, 2, 64)):
    cache = Cache(list(lengths), heads[1], heads[2], 16, BF16, seed)
    query = _normal((len(lengths), heads[0], heads[2]), cache.g, BF16)
    return cache, query


def test_other_streams():
    cache, query = _step_inputs(1)
    expected = paged_kv_attention(query, None, None, *cache.pools, cache.table, cache.lengths)
    prompt = paged_prefill_attention(query, *cache.pools, cache.table, cache.lengths, _int32([0, 1, 2, 2, 4]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(5):
        for stream in streams:
            with torch.cuda.stream(stream):
                got.append((paged_kv_attention(query, None, None, *cache.pools, cache.table, cache.lengths),
                            paged_prefill_attention(query, *cache.pools, cache.table, cache.lengths,
                                                    _int32([0, 1, 2, 2, 4]))))
    torch.cuda.synchronize()
    for a, b in got:
        assert torch.equal(a, expected) and torch.equal(b, prompt)


def test_the_same_call_gives_the_same_bits():
    cache, query = _step_inputs(2, lengths=(5000, 77, 131, 20000))
    first = paged_kv_attention(query, None, None, *cache.pools, cache.table, cache.lengths)
    prompt = paged_prefill_attention(query, *cache.pools, cache.table, cache.lengths, _int32([0, 1, 2, 2, 4]))
    for _ in range(5):
        assert torch.equal(first, paged_kv_attention(query, None, None, *cache.pools, cache.table, cache.lengths))
        assert torch.equal(prompt, paged_prefill_attention(query, *cache.pools, cache.table, cache.lengths,
                                                           _int32([0, 1, 2, 2, 4])))


def test_captured_steps_follow_the_lengths_and_overlap():
    """Two captured steps, each with its own cache, replayed on two streams at once, with other lengths each time."""
    parts = []
    for seed in (3, 4):
        cache, query = _step_inputs(seed)
        offsets = _int32([0, 1, 2, 2, 4])

        def call(cache=cache, query=query, offsets=offsets):
            return (paged_kv_attention(query, None, None, *cache.pools, cache.table, cache.lengths),
                    paged_prefill_attention(query, *cache.pools, cache.table, cache.lengths, offsets))

        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            call()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = call()
        parts.append((cache, query, call, graph, out, stream))
    torch.cuda.synchronize()
    full = [[70, 9000, 0, 300], [70, 9000, 0, 300]]
    for step in range(4):
        for (cache, *_), lengths in zip(parts, full):
            cache.lengths.copy_(_int32([max(0, n - 17 * step) for n in lengths]))
        torch.cuda.synchronize()
        for _ in range(3):
            for cache, query, call, graph, out, stream in parts:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for cache, query, call, graph, out, stream in parts:
            for got, want in zip(out, call()):
                assert torch.equal(got, want)
    for _, _, _, graph, _, _ in parts:
        graph.reset()


def test_captured_reserve():
    state = PagedState(1, 3, 64, 1, 64, page_size=8, device="cuda")
    counts = _int32([0, 0, 0])
    state.reserve(counts, 6)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        batch = state.reserve(counts, 6)
    total = [0, 0, 0]
    for step in ([1, 2, 3], [0, 0, 6], [3, 3, 1], [1, 0, 0]):
        counts.copy_(_int32(step))
        graph.replay()
        granted = batch.granted.tolist()
        assert granted == ([3, 3, 0] if step == [3, 3, 1] else step)
        total = [a + b for a, b in zip(total, granted)]
        assert state.lengths.tolist() == total


def test_refusals():
    cache, query = _step_inputs(5)
    good = dict(query=query, key=None, value=None, key_pages=cache.pools[0], value_pages=cache.pools[1],
                block_table=cache.table, lengths=cache.lengths)

    def refused(match, stage="input-binding", **changes):
        with pytest.raises(CompilerError, match=match) as info:
            paged_kv_attention(**{**good, **changes})
        assert info.value.diagnostic.stage == stage

    keys = torch.zeros(4, 2, 64, dtype=BF16, device="cuda")
    refused("heads a multiple", query=query[:, :3])
    refused("query must be", query=query[:, :, :32])
    refused("query must be torch.bfloat16", query=query.half())
    refused("16-byte", query=torch.zeros(4, 8, 72, dtype=BF16, device="cuda")[:, :, 4:68])
    refused("16-byte", query=torch.zeros(4, 8, 128, dtype=BF16, device="cuda")[:, :, ::2])
    refused("come together", key=keys)
    refused("value must be", key=keys, value=keys[:3])
    refused("value_pages must be", value_pages=cache.pools[1].half())
    refused("block_table must be", block_table=cache.table.long())
    refused("block_table must be", block_table=cache.table[0])
    refused("block_table must be a contiguous", block_table=cache.table[:, ::2])
    refused("a row of the table each", block_table=cache.table[:3])
    refused("lengths must be", lengths=cache.lengths[:3])
    refused("lengths must be", lengths=cache.lengths.cpu())
    refused("rows must be", rows=_int32([0, 1, 2]))
    refused("rows must be", rows=torch.tensor([0, 1, 2, 3], device="cuda"))
    refused("out must be", out=torch.empty_like(query, dtype=FP16))
    refused("status must be", status=torch.zeros(2, dtype=torch.int32, device="cuda"))
    with pytest.raises(CompilerError, match="offsets must be"):
        paged_prefill_attention(query, *cache.pools, cache.table, cache.lengths, _int32([0, 1, 2]))
    with pytest.raises(CompilerError, match="slots must be"):
        paged_append(keys, keys, *cache.pools, _int32([0, 1, 2, 3]))
    with pytest.raises(CompilerError, match="counts must be"):
        paged_reserve(torch.tensor([1, 2, 3, 4], device="cuda"), cache.lengths, cache.table, _int32([0]), _int32([1]), 16, 4)
    with pytest.raises(CompilerError, match="max_tokens"):
        paged_reserve(_int32([1, 2, 3, 4]), cache.lengths, cache.table, _int32([0]), _int32([1]), 16, -1)
    with pytest.raises(RuntimeError, match="inference only"):
        paged_kv_attention(**{**good, "query": query.clone().requires_grad_()})
    with torch.no_grad():
        paged_kv_attention(**{**good, "query": query.clone().requires_grad_()})


def test_no_tokens():
    cache, query = _step_inputs(6)
    empty = query[:0]
    rows = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert paged_kv_attention(empty, None, None, *cache.pools, cache.table, cache.lengths, rows).shape == (0, 8, 64)
    assert paged_prefill_attention(empty, *cache.pools, cache.table, cache.lengths, _int32([0] * 5)).shape == (0, 8, 64)
    paged_append(torch.zeros(0, 2, 64, dtype=BF16, device="cuda"), torch.zeros(0, 2, 64, dtype=BF16, device="cuda"),
                 *cache.pools, torch.zeros(0, dtype=torch.int64, device="cuda"))


def test_status_stays_when_nothing_went_wrong():
    cache, query = _step_inputs(7)
    status = _int32([0])
    paged_kv_attention(query, None, None, *cache.pools, cache.table, cache.lengths, status=status)
    paged_prefill_attention(query, *cache.pools, cache.table, cache.lengths, _int32([0, 1, 2, 2, 4]), status=status)
    assert status.item() == 0


@pytest.mark.parametrize("heads", [(3, 1, 64), (9, 1, 256)])
def test_the_most_requests(heads):
    """2,048 rows, of which every 50th is compared: the tables of the kernels take shared memory from their rings."""
    count, kv_heads, dim = heads
    new = [(i * 7) % 5 for i in range(2048)]
    lengths = [n + (i * 31) % 150 for i, n in enumerate(new)]
    cache = Cache(lengths, kv_heads, dim, 16, BF16, 1)
    query = _normal((2048, count, dim), cache.g, BF16)
    out = paged_kv_attention(query, None, None, *cache.pools, cache.table, cache.lengths)
    for r in range(0, 2048, 50):
        expected = reference.attend(query[r], *cache.pools, cache.table[r], lengths[r], dim ** -0.5)
        _check(out[r], expected, lengths[r], BF16, reference.decode_rounding(BF16))
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    query = _normal((offsets[-1], count, dim), cache.g, BF16)
    out = paged_prefill_attention(query, *cache.pools, cache.table, cache.lengths, _int32(offsets))
    for r in range(0, 2048, 50):
        for j in range(new[r]):
            keys = lengths[r] - new[r] + j + 1
            expected = reference.attend(query[offsets[r] + j], *cache.pools, cache.table[r], keys, dim ** -0.5)
            _check(out[offsets[r] + j], expected, keys, BF16, reference.prompt_rounding(BF16))
    rows = torch.zeros(2049, dtype=torch.int32, device="cuda")
    with pytest.raises(CompilerError, match="2048"):
        paged_kv_attention(_normal((2049, count, dim), cache.g, BF16), None, None, *cache.pools, cache.table, cache.lengths, rows)


def test_query_heads_per_key_head():
    """Up to 128 for prompts; single tokens take any number."""
    cache = Cache([70], 1, 64, 16, BF16, 2)
    for count in (128, 130):
        query = _normal((1, count, 64), cache.g, BF16)
        expected = reference.attend(query[0], *cache.pools, cache.table[0], 70, 0.125)
        out = paged_kv_attention(query, None, None, *cache.pools, cache.table, cache.lengths)
        _check(out[0], expected, 70, BF16, reference.decode_rounding(BF16))
        if count == 128:
            out = paged_prefill_attention(query, *cache.pools, cache.table, cache.lengths, _int32([0, 1]))
            _check(out[0], expected, 70, BF16, reference.prompt_rounding(BF16))
        else:
            with pytest.raises(CompilerError):
                paged_prefill_attention(query, *cache.pools, cache.table, cache.lengths, _int32([0, 1]))


def test_output_in_the_place_of_the_queries():
    cache, query = _step_inputs(8, lengths=(5000, 77, 131, 20000))
    offsets = _int32([0, 1, 2, 2, 4])
    for call in (lambda q, out: paged_kv_attention(q, None, None, *cache.pools, cache.table, cache.lengths, out=out),
                 lambda q, out: paged_prefill_attention(q, *cache.pools, cache.table, cache.lengths, offsets, out=out)):
        expected, q = call(query, None), query.clone()
        assert call(q, q) is q and torch.equal(q, expected)


FIRST_CALL = """
import torch
from megabake_b200 import PagedState, paged_append, paged_kv_attention, paged_prefill_attention
state = PagedState(1, 2, 4096, 1, 64, device="cuda")
counts = torch.ones(2, dtype=torch.int32, device="cuda")
rows = torch.ones(2, 1, 64, dtype=torch.bfloat16, device="cuda")
pools = (state.key_pages[0], state.value_pages[0])
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    batch = state.reserve(counts, 2)
    a = paged_kv_attention(rows, rows, rows, *pools, state.block_table, state.lengths, batch.rows)
    paged_append(rows, rows, *pools, batch.slots)
    b = paged_prefill_attention(rows, *pools, state.block_table, state.lengths, batch.offsets)
for step in range(3):
    graph.replay()
torch.cuda.synchronize()
assert state.lengths.tolist() == [3, 3] and bool((a == 1).all()) and bool((b == 1).all())
print("captured")
"""


def test_the_first_call_of_a_process_is_captured():
    import subprocess
    import sys

    done = subprocess.run([sys.executable, "-c", FIRST_CALL], capture_output=True, text=True, timeout=250)
    assert done.returncode == 0 and "captured" in done.stdout, done.stderr[-2000:]


# ---------------------------------------------------------------------------------------
# Together, as a server uses them
# ---------------------------------------------------------------------------------------
def test_requests_come_and_go():
    """Prompts are reserved, appended and attended; then every request decodes; one ends and another takes its place.
    Every output against the definition on what the request has seen."""
    heads, kv_heads, dim, page = 4, 2, 64, 8
    g = torch.Generator(device="cuda").manual_seed(0)
    state = PagedState(1, 3, 96, kv_heads, dim, page_size=page, pages=30, device="cuda")
    pools = (state.key_pages[0], state.value_pages[0])
    history = [None] * 3

    def step(counts, prompt):
        batch = state.reserve(_int32(counts), 64)
        tokens = batch.slots.numel()
        fused = _normal((tokens, heads + 2 * kv_heads, dim), g, BF16)
        query, key, value = fused.split((heads, kv_heads, kv_heads), dim=1)
        if prompt:
            paged_append(key, value, *pools, batch.slots)
            out = paged_prefill_attention(query, *pools, state.block_table, state.lengths, batch.offsets)
        else:
            out = paged_kv_attention(query, key, value, *pools, state.block_table, state.lengths, batch.rows)
        for r, got in enumerate(batch.granted.tolist()):
            if got < 0:
                history[r] = None
        for t, r in enumerate(batch.rows.tolist()):
            if r < 0:
                assert out[t].eq(0).all()
                continue
            seen = history[r] or ([], [])
            history[r] = (seen[0] + [key[t]], seen[1] + [value[t]])
            k, v = (torch.stack(x)[None] for x in history[r])
            expected = reference.attend(query[t], k, v, _int32([0]), k.shape[1], dim ** -0.5)
            _check(out[t], expected, k.shape[1], BF16, reference.prompt_rounding(BF16))
        return batch

    step([20, 3, 0], True)
    for _ in range(6):
        step([1, 1, 0], False)
    step([0, 0, 41], True)
    step([1, 1, 1], False)
    step([-27, 1, 1], False)
    step([17, 0, 9], True)
    for _ in range(9):
        batch = step([1, 1, 1], False)
    assert state.lengths.tolist() == [26, 20, 61] and batch.granted.tolist() == [1, 1, 1]
    held = [e for row in state.block_table.tolist() for e in row if e >= 0]
    assert sorted(held + state.free_pages[:state.free_count.item()].tolist()) == list(range(30))
