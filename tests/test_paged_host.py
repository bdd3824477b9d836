"""The paged operators without a device: refusals of the C entries and of the Python ones, the state's tensors, and the
definition that the GPU tests compare with."""

import ctypes
import random

import pytest
import torch

from megabake_b200 import PagedState, paged_append, paged_kv_attention, paged_prefill_attention, paged_reserve
from megabake_b200 import runtime as rt
from megabake_b200.diagnostics import CompilerError
from tests import paged_reference as reference

INVALID, UNSUPPORTED = 1, 3   # enum mb_error


def _reserve_args(**changes):
    args = rt.PagedReserveArgs(4, 8, 32, 16, 64, 0, *[4096 * (i + 1) for i in range(10)])
    for name, value in changes.items():
        setattr(args, name, value)
    return args


def _append_args(**changes):
    args = rt.PagedAppendArgs(4, 2, 64, 32, 16, 0, 128, 64, 128, 64, 2048, 128, 64, 2048, 128, 64,
                              *[4096 * (i + 1) for i in range(5)])
    for name, value in changes.items():
        setattr(args, name, value)
    return args


def _attention_args(**changes):
    args = rt.PagedAttentionArgs(0, 4, 4, 4, 2, 64, 8, 32, 16, 0, 0.125, 0, 256, 64, 128, 64, 128, 64, 2048, 128, 64,
                                 2048, 128, 64, *[4096 * (i + 1) for i in range(9)], 0, 0)
    for name, value in changes.items():
        setattr(args, name, value)
    return args


@pytest.mark.parametrize("changes,code", [
    (dict(requests=0), INVALID), (dict(width=0), INVALID), (dict(pages=0), INVALID), (dict(max_tokens=-1), INVALID),
    (dict(counts=0), INVALID), (dict(free_count=0), INVALID), (dict(slots=0), INVALID), (dict(rows=0), INVALID),
    (dict(slots=4100), INVALID), (dict(lengths=4097), INVALID), (dict(requests=2049), UNSUPPORTED),
    (dict(page_size=4), UNSUPPORTED), (dict(page_size=48), UNSUPPORTED), (dict(page_size=2048), UNSUPPORTED),
    (dict(width=1 << 27, page_size=16), UNSUPPORTED), (dict(width=(1 << 26) + 1, page_size=16), UNSUPPORTED),
    (dict(max_tokens=(1 << 30) + 1), UNSUPPORTED),
])
def test_reserve_entry_refuses(changes, code):
    assert rt.load_library().mb_paged_reserve(ctypes.byref(_reserve_args(**changes)), None) == code


@pytest.mark.parametrize("changes,code", [
    (dict(tokens=0), INVALID), (dict(kv_heads=0), INVALID), (dict(key=0), INVALID), (dict(slots=4), INVALID),
    (dict(key=4104), INVALID), (dict(value_token=4), INVALID), (dict(kpool_head=-64), INVALID),
    (dict(vpool_page=2049), INVALID), (dict(head_dim=96), UNSUPPORTED), (dict(page_size=0), UNSUPPORTED),
])
def test_append_entry_refuses(changes, code):
    assert rt.load_library().mb_paged_append(ctypes.byref(_append_args(**changes)), None) == code


@pytest.mark.parametrize("prefill", [False, True])
@pytest.mark.parametrize("changes,code", [
    (dict(tokens=0), INVALID), (dict(heads=3), INVALID), (dict(heads=0), INVALID), (dict(query=0), INVALID),
    (dict(value=0), INVALID), (dict(out=8), INVALID), (dict(query_head=4), INVALID), (dict(block_table=0), INVALID),
    (dict(block_table=4098), INVALID), (dict(key_pages=4104), INVALID), (dict(element=2), UNSUPPORTED),
    (dict(head_dim=80), UNSUPPORTED), (dict(page_size=24), UNSUPPORTED), (dict(width=1 << 27), UNSUPPORTED),
    (dict(width=(1 << 26) + 1), UNSUPPORTED),
])
def test_attention_entries_refuse(prefill, changes, code):
    lib = rt.load_library()
    if prefill and "value" not in changes:
        changes = {**dict(key=0, value=0), **changes}
    args = _attention_args(**changes)
    entry, size = ((lib.mb_paged_prefill, lib.mb_paged_prefill_workspace) if prefill else
                   (lib.mb_paged_attention, lib.mb_paged_attention_workspace))
    assert entry(ctypes.byref(args), None) == code
    assert size(ctypes.byref(args)) == -code


def test_prefill_entry_needs_offsets_and_appended_keys():
    lib = rt.load_library()
    assert lib.mb_paged_prefill(ctypes.byref(_attention_args()), None) == INVALID            # key and value given
    assert lib.mb_paged_prefill(ctypes.byref(_attention_args(key=0, value=0, index=0)), None) == INVALID


def test_addresses_follow_the_fields():
    from megabake_b200 import paged

    for struct_type, first, addresses in ((rt.PagedReserveArgs, "counts", paged._RESERVE_ADDRESSES),
                                          (rt.PagedAppendArgs, "key", paged._APPEND_ADDRESSES),
                                          (rt.PagedAttentionArgs, "query", paged._ATTENTION_ADDRESSES)):
        assert getattr(struct_type, first).offset + addresses.size == ctypes.sizeof(struct_type)


def test_entries_refuse_null():
    lib = rt.load_library()
    for name in ("mb_paged_reserve", "mb_paged_append", "mb_paged_attention", "mb_paged_prefill"):
        assert getattr(lib, name)(None, None) == INVALID


def _state(**changes):
    options = dict(layers=1, requests=3, capacity=40, kv_heads=2, head_dim=64, page_size=16, device="cpu")
    return PagedState(**{**options, **changes})


def test_state_tensors():
    state = _state(layers=2)
    assert state.capacity == 48 and state.block_table.shape == (3, 3) and len(state.key_pages) == 2
    assert state.key_pages[0].shape == (9, 16, 2, 64) and state.key_pages[0].dtype == torch.bfloat16
    assert state.free_pages.tolist() == list(range(8, -1, -1)) and state.free_count.tolist() == [9]
    assert state.block_table.eq(-1).all() and state.lengths.eq(0).all()


@pytest.mark.parametrize("changes", [dict(page_size=12), dict(page_size=4), dict(head_dim=96), dict(layers=0),
                                     dict(requests=0), dict(requests=2049), dict(capacity=0), dict(pages=0),
                                     dict(dtype=torch.float32)])
def test_state_refuses(changes):
    with pytest.raises(ValueError):
        _state(**changes)


def test_operators_refuse_the_cpu():
    state = _state()
    rows = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    one = torch.ones(3, dtype=torch.int32)
    pools = (state.key_pages[0], state.value_pages[0])
    for call in (lambda: state.reserve(one, 3),
                 lambda: paged_append(rows, rows, *pools, torch.zeros(3, dtype=torch.int64)),
                 lambda: paged_kv_attention(rows, rows, rows, *pools, state.block_table, state.lengths),
                 lambda: paged_prefill_attention(rows, *pools, state.block_table, state.lengths,
                                                 torch.zeros(4, dtype=torch.int32))):
        with pytest.raises(CompilerError) as info:
            call()
        assert info.value.diagnostic.stage == "input-binding" and "CUDA" in str(info.value)


@pytest.mark.parametrize("shape,dtype", [((9, 12, 2, 64), torch.bfloat16), ((9, 16, 2, 96), torch.bfloat16),
                                         ((9, 16, 2, 64), torch.float32), ((9, 16, 128), torch.bfloat16),
                                         ((0, 16, 2, 64), torch.float16)])
def test_pools_are_checked(shape, dtype):
    pool = torch.zeros(shape, dtype=dtype)
    rows = torch.zeros(3, 2, 64, dtype=dtype)
    with pytest.raises(CompilerError, match="key_pages"):
        paged_append(rows, rows, pool, pool, torch.zeros(3, dtype=torch.int64))


def test_pool_strides_are_checked():
    pool = torch.zeros(9, 16, 2, 68, dtype=torch.bfloat16)[..., :64]
    rows = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(CompilerError, match="16-byte"):
        paged_append(rows, rows, pool, pool, torch.zeros(3, dtype=torch.int64))


@pytest.mark.parametrize("seed", range(20))
def test_reserve_definition_keeps_pages(seed):
    """Whatever is asked for, every page is in one place: in one row of the table, or on the free part of the stack; and
    taking back what a call granted restores the tables."""
    rng = random.Random(seed)
    requests, width, page, pages = rng.randint(1, 9), rng.randint(1, 6), 8, rng.randint(1, 30)
    state = ([0] * requests, [[-1] * width for _ in range(requests)], list(range(pages)), pages)
    for _ in range(30):
        lengths, table, stack, free = state
        counts = [rng.choice((0, 1, rng.randint(-60, 60))) for _ in range(requests)]
        state, (offsets, slots, positions, rows, granted) = reference.reserve(
            counts, lengths, table, stack, free, page, rng.randint(0, 80))
        lengths, table, stack, free = state
        held = [e for row in table for e in row if e >= 0]
        assert sorted(held + stack[:free]) == list(range(pages))
        assert [sum(e >= 0 for e in row) for row in table] == [reference.pages_of(n, page) for n in lengths]
        assert len({s for s in slots if s >= 0}) == offsets[-1] == sum(max(g, 0) for g in granted)
        up = [max(g, 0) for g in granted]
        back, _ = reference.reserve([-n for n in up], lengths, table, stack, free, page, 0)
        again, _ = reference.reserve(up, *back, page, sum(up))
        assert again[0] == lengths and again[1] == table and again[3] == free
