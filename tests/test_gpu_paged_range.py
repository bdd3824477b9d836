"""Scores and values at the ends of what 16-bit numbers hold."""

import pytest
import torch

from megabake_b200 import paged_kv_attention, paged_prefill_attention
from tests import paged_reference as reference
from tests.test_gpu_paged import BF16, FP16, Cache, _check, _int32, _normal

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]


def _fill(cache, keys, values):
    slots = torch.tensor(cache.slots[0], device="cuda")
    page, place = slots // cache.page, slots % cache.page
    for pool, content in zip(cache.pools, (keys, values)):
        pool[page, place] = content.to(pool.dtype)


@pytest.mark.parametrize("scale", [None, -0.125])
@pytest.mark.parametrize("dtype,query,most,value", [
    (BF16, 100.0, 3e5, 1e37), (BF16, 100.0, 3e9, 1e37), (BF16, 1e10, 1e20, 1e37), (BF16, -1e4, 3e7, 3e38),
    (FP16, 100.0, 300.0, 6e4), (FP16, 1000.0, 3e3, 6e4), (FP16, 3e4, 3e4, 6e4), (FP16, -6e4, 6e4, 6e4)])
@pytest.mark.parametrize("heads", [(1, 1, 64), (3, 1, 128), (2, 1, 256)])
@pytest.mark.parametrize("length", [300, 3000])
def test_scores_far_from_zero(heads, length, dtype, query, most, value, scale):
    """The highest score takes all, exactly, where the next one is hundreds below; equal scores share, whatever they are; and the
    largest values are not too large to be summed.  300 keys that rise, then stay."""
    count, kv_heads, dim = heads
    cache = Cache([length], kv_heads, dim, 16, dtype, length)
    new = 200
    rising = torch.linspace(-most, most, 300, device="cuda").to(dtype)
    rising = rising.repeat_interleave(length // 300)
    values = _normal((length, kv_heads, dim), cache.g, dtype).float().clamp(-1, 1) * value
    q = torch.full((new, count, dim), query, device="cuda").to(dtype)
    ends = torch.finfo(dtype).max
    for keys in (rising, rising.flip(0), torch.full_like(rising, most), torch.full_like(rising, -most)):
        _fill(cache, keys[:, None, None].expand(length, kv_heads, dim), values)
        out = paged_prefill_attention(q, *cache.pools, cache.table, cache.lengths, _int32([0, new]), scale=scale)
        one = paged_kv_attention(q[-1:], None, None, *cache.pools, cache.table, cache.lengths, scale=scale)
        factor = query * (dim ** -0.5 if scale is None else scale) * dim
        for t, got, rounding in [(t, out[t], reference.prompt_rounding(dtype)) for t in (0, 1, 63, 64, 130, 198, 199)] + \
                                [(199, one[0], reference.decode_rounding(dtype))]:
            n = length - new + t + 1
            scores = keys[:n].double() * factor
            share = scores == scores.max()
            rest = scores[~share]
            assert not rest.numel() or float(scores.max() - rest.max()) > 200
            v = cache.pools[1].new_empty(0)
            slots = torch.tensor(cache.slots[0][:n], device="cuda")[share]
            v = cache.pools[1][slots // 16, slots % 16, 0].double()
            expected = (v.mean(0).expand(count, dim), v.abs().mean(0).expand(count, dim), torch.zeros(count, 1, device="cuda"))
            assert float(expected[1].max()) <= ends
            _check(got, expected, n, dtype, rounding)
