"""Arguments that the paged operators refuse, without a device."""

import pytest
import torch

from megabake_b200 import PagedState, paged_append, paged_kv_attention, paged_prefill_attention, paged_reserve
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
