"""Arguments that the paged operators refuse, without a device."""

import ctypes

import pytest
import torch

from megabake_b200 import paged_append, paged_reserve
from megabake_b200 import runtime as rt
from megabake_b200.diagnostics import CompilerError

INT32 = torch.int32


def _refused(match, call):
    with pytest.raises(CompilerError, match=match) as info:
        call()
    assert info.value.diagnostic.stage == "input-binding"


@pytest.mark.parametrize("requests", [1, 4, 128, 2048])
@pytest.mark.parametrize("name", ["counts", "lengths", "free_pages"])
def test_reserve_takes_one_number_a_request(requests, name):
    """The result has one offset more than there are counts: a row of counts in a table of its own would make it two."""
    tensors = dict(counts=torch.zeros(requests, dtype=INT32), lengths=torch.zeros(requests, dtype=INT32),
                   block_table=torch.full((requests, 2), -1, dtype=INT32),
                   free_pages=torch.zeros(3, dtype=INT32), free_count=torch.zeros(1, dtype=INT32))
    if requests > 1 or name == "free_pages":
        _refused(f"{name} must be",
                 lambda: paged_reserve(**{**tensors, name: tensors[name][None]}, page_size=16, max_tokens=2))
        _refused(f"{name} must be",
                 lambda: paged_reserve(**{**tensors, name: tensors[name][:, None]}, page_size=16, max_tokens=2))
    _refused("CUDA", lambda: paged_reserve(**tensors, page_size=16, max_tokens=2))


@pytest.mark.parametrize("entry", ["mb_paged_attention", "mb_paged_prefill"])
def test_a_limit_below_zero_is_refused(entry):
    args = rt.PagedAttentionArgs(0, 4, 4, 4, 2, 64, 8, 32, 16, 0, 0.125, -1, 256, 64, 0, 0, 0, 0, 2048, 128, 64,
                                 2048, 128, 64, 4096, 0, 0, *[4096 * (i + 1) for i in range(6)], 0, 0)
    assert getattr(rt.load_library(), entry)(ctypes.byref(args), None) == 1   # MB_ERR_INVALID


@pytest.mark.parametrize("requests,width", [(2048, 1 << 20), (2048, (1 << 27) - 1), (17, 1 << 27)])
def test_reserve_takes_tables_whose_entries_an_int_counts(requests, width):
    """Pages of all rows together are counted in 32 bits."""
    args = rt.PagedReserveArgs(requests, width, 32, 8, 64, 0, *[4096 * (i + 1) for i in range(10)])
    assert rt.load_library().mb_paged_reserve(ctypes.byref(args), None) == 3   # MB_ERR_UNSUPPORTED


def test_strides_of_single_places_mean_nothing():
    """One token, one head or one page: what lies between it and the next is never looked at."""
    def one(shape, strides):
        return torch.zeros(4096, dtype=torch.bfloat16).as_strided(shape, strides)

    slots = torch.zeros(1, dtype=torch.int64)
    pool = one((1, 16, 1, 64), (3, 64, 5, 1))
    _refused("CUDA", lambda: paged_append(one((1, 1, 64), (195, 67, 1)), one((1, 1, 64), (1, 0, 1)), pool, pool, slots))
    _refused("16-byte", lambda: paged_append(one((1, 1, 64), (195, 67, 1)), one((1, 1, 64), (1, 0, 1)), pool,
                                             one((1, 16, 1, 64), (64, 68, 64, 1)), slots))
