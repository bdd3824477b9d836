"""Operators around a paged key-value cache.

A server that keeps many requests of unknown length holds keys and values in pages of a pool
``[pages, page_size, kv_heads, head_dim]`` (one pool each per layer) instead of one contiguous cache per
row.  One block table for all layers, int32 ``[requests, width]``, lists the pages of every request in
order (-1: none), ``lengths`` (int32 ``[requests]``) says how many tokens a request holds, and the unused pages
are the first ``free_count`` (int32 ``[1]``) entries of the stack ``free_pages`` (int32 ``[pages]``).
``PagedState`` makes these tensors; they are the caller's, as the contiguous state is.

``paged_reserve``            pages, slots and positions for the new tokens of every request, on the device
``paged_append``             keys and values of tokens into their slots
``paged_kv_attention``       one new token a request: append it and attend (the paged ``kv_attention``)
``paged_prefill_attention``  several new tokens a request, causal (the paged ``prefill_kv_attention``)

Each is one call into the native library on torch's current stream: nothing is synchronised, all of them can be
captured in a CUDA graph, and a scratch buffer is the call's own.  bf16 and fp16; heads of 64, 128 or 256;
any number of query heads per key head; pages of 8 to 1,024 tokens (a power of two); pools and rows may have any
strides that are multiples of 16 bytes.  Scores, softmax statistics and sums are fp32 and outputs are rounded
once -- unlike ``kv_attention``, whose rounding points are the reference's eager ones.  Inference only.

The reference has one contiguous cache and one length per batch (``fx_handler/hf_attention.py:194-196``);
per-request state is a step of its roadmap (``docs/roadmap.md:178``).
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import runtime as rt
from .diagnostics import fail

__all__ = ["PagedBatch", "PagedState", "paged_append", "paged_kv_attention", "paged_prefill_attention",
           "paged_reserve"]

_ELEMENTS = {torch.bfloat16: 0, torch.float16: 1}
_HEAD_DIMS = (64, 128, 256)
_MAX_REQUESTS = 2048
_ready: set[int] = set()   # devices that are known to be sm_100


class PagedBatch(NamedTuple):
    """Where the tokens of one ``paged_reserve`` go.  Row ``r`` of the table has the places ``offsets[r]`` ..
    ``offsets[r + 1] - 1``; places behind the last token hold slot -1, position 0 and row -1."""

    offsets: torch.Tensor     # int32 [requests + 1]
    slots: torch.Tensor       # int64 [max_tokens]: page * page_size + place in the page
    positions: torch.Tensor   # int64 [max_tokens]
    rows: torch.Tensor        # int32 [max_tokens]
    granted: torch.Tensor     # int32 [requests]: tokens granted, negative: dropped


class PagedState:
    """The tensors of a paged cache: pools per layer, one block table, lengths and the stack of free pages.

    ``pages`` defaults to enough for every request to grow to ``capacity`` tokens; fewer pages share the memory
    between requests that do not all grow that long."""

    def __init__(self, layers: int, requests: int, capacity: int, kv_heads: int, head_dim: int, *,
                 page_size: int = 64, pages: int | None = None, dtype: torch.dtype = torch.bfloat16, device=None):
        if min(layers, requests, capacity, kv_heads) < 1:
            raise ValueError("a paged state needs at least one layer, request, token and head")
        if dtype not in _ELEMENTS or head_dim not in _HEAD_DIMS or not _page_size_covered(page_size):
            raise ValueError("a paged state holds bf16 or fp16 heads of 64, 128 or 256 in pages of 8 to 1024 "
                             "tokens, a power of two")
        if requests > _MAX_REQUESTS:
            raise ValueError(f"a paged state holds at most {_MAX_REQUESTS} requests")
        width = -(-capacity // page_size)
        pages = requests * width if pages is None else pages
        if pages < 1:
            raise ValueError("a paged state needs at least one page")
        self.page_size, self.capacity = page_size, width * page_size
        shape = (pages, page_size, kv_heads, head_dim)
        self.key_pages = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(layers)]
        self.value_pages = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(layers)]
        self.block_table = torch.empty((requests, width), dtype=torch.int32, device=device)
        self.lengths = torch.empty(requests, dtype=torch.int32, device=device)
        self.free_pages = torch.empty(pages, dtype=torch.int32, device=device)
        self.free_count = torch.empty(1, dtype=torch.int32, device=device)
        self.reset()

    def reset(self) -> None:
        """Every request empty, every page free; page 0 is handed out first."""
        pages = self.free_pages.numel()
        self.block_table.fill_(-1)
        self.lengths.zero_()
        self.free_pages.copy_(torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=self.free_pages.device))
        self.free_count.fill_(pages)

    def reserve(self, counts: torch.Tensor, max_tokens: int) -> PagedBatch:
        """``paged_reserve`` on these tensors."""
        return paged_reserve(counts, self.lengths, self.block_table, self.free_pages, self.free_count,
                             self.page_size, max_tokens)


def _page_size_covered(page_size: int) -> bool:
    return 8 <= page_size <= 1024 and page_size & (page_size - 1) == 0


def _device_ready(device: torch.device) -> int:
    index = device.index
    if index not in _ready:
        from .engine import _require_native_device

        _require_native_device(device)
        _ready.add(index)
    return index


def _whole(name: str, tensor: torch.Tensor, dtype: torch.dtype, numel: int, device: torch.device) -> int:
    """Address of a contiguous tensor of whole numbers."""
    if tensor.dtype != dtype or tensor.device != device or tensor.numel() != numel or not tensor.is_contiguous():
        fail("input-binding", f"{name} must be a contiguous {dtype} tensor of {numel} on {device}, got "
                              f"{tensor.dtype} {tuple(tensor.shape)} on {tensor.device}")
    return tensor.data_ptr()


def _rows(name: str, tensor: torch.Tensor, shape: tuple, like: torch.Tensor) -> tuple:
    """Address and strides of ``[..., head_dim]`` values that are read 16 bytes at a time."""
    if tensor.dtype != like.dtype or tensor.device != like.device or tensor.shape != shape:
        fail("input-binding", f"{name} must be {like.dtype} {tuple(shape)} on {like.device}, got {tensor.dtype} "
                              f"{tuple(tensor.shape)} on {tensor.device}")
    return _strided(name, tensor)


def _strided(name: str, tensor: torch.Tensor) -> tuple:
    pointer, strides = tensor.data_ptr(), tensor.stride()
    bits = pointer >> 1
    for stride in strides[:-1]:
        bits |= stride
    if bits & 7 or pointer & 1 or strides[-1] != 1:
        fail("input-binding", f"{name} must have a contiguous last dimension and start, in every dimension, on "
                              "16-byte boundaries")
    return (pointer, *strides[:-1])


def _inference_only(*tensors) -> None:
    if torch.is_grad_enabled():
        for tensor in tensors:
            if tensor is not None and tensor.requires_grad:
                raise RuntimeError("MegaBake supports inference only")


def _pools(key_pages: torch.Tensor, value_pages: torch.Tensor) -> tuple:
    if key_pages.dtype not in _ELEMENTS or key_pages.dim() != 4 or key_pages.shape[3] not in _HEAD_DIMS or \
            not _page_size_covered(key_pages.shape[1]) or key_pages.shape[0] < 1 or key_pages.shape[2] < 1:
        fail("input-binding", "key_pages must be bf16 or fp16 [pages, page_size, kv_heads, head_dim] with head_dim 64, "
                              "128 or 256 and page_size a power of two from 8 to 1024, got "
                              f"{key_pages.dtype} {tuple(key_pages.shape)}")
    return _strided("key_pages", key_pages), _rows("value_pages", value_pages, key_pages.shape, key_pages)


def _call(function, args, index: int, what: str) -> None:
    lib = rt.load_library()
    stream = torch.cuda.current_stream(index).cuda_stream
    if index == torch.cuda.current_device():
        code = function(ctypes.byref(args), stream)
    else:
        with torch.cuda.device(index):
            code = function(ctypes.byref(args), stream)
    if code:
        rt._check(lib, code, "runtime", what)


def paged_reserve(counts: torch.Tensor, lengths: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                  free_count: torch.Tensor, page_size: int, max_tokens: int) -> PagedBatch:
    """Make room for ``counts[r]`` more tokens of every request ``r`` (int32 ``[requests]``), on the device.

    Requests are granted in row order, all or nothing: one is granted if its tokens fit its row of the table, if the
    tokens wanted up to it (by requests that fit their rows) are at most ``max_tokens``, and if the pages newly
    wanted up to it are free, or it wants none.  A negative count drops the request's last tokens instead (all of them at
    most): rejected speculation, or ``-length`` for a request that has ended; pages left without tokens are
    free again before anything is granted.  Dropping what a call granted restores the tables.

    ``lengths``, ``block_table``, ``free_pages`` and ``free_count`` are updated.  ``max_tokens`` fixes the shapes of the
    result, so that a captured step can be replayed with other counts."""
    if block_table.dim() != 2:
        fail("input-binding", f"block_table must be [requests, width], got {tuple(block_table.shape)}")
    device = counts.device
    requests, width = block_table.shape
    if device.type != "cuda" or not 1 <= requests <= _MAX_REQUESTS or width < 1 or not _page_size_covered(page_size) or \
            max_tokens < 0 or max_tokens > 0x7fffffff or width * page_size > 0x7fffffff or free_pages.numel() < 1:
        fail("input-binding", f"paged_reserve needs 1..{_MAX_REQUESTS} requests on a CUDA device, pages of 8 to 1024 tokens "
                              "(a power of two), rows below 2**31 tokens and max_tokens >= 0, got "
                              f"{tuple(block_table.shape)} pages of {page_size} on {device}, max_tokens {max_tokens}")
    index = _device_ready(device)
    int32 = torch.int32
    args = rt.PagedReserveArgs(
        requests, width, free_pages.numel(), page_size, max_tokens, 0,
        _whole("counts", counts, int32, requests, device), _whole("lengths", lengths, int32, requests, device),
        _whole("block_table", block_table, int32, requests * width, device),
        _whole("free_pages", free_pages, int32, free_pages.numel(), device),
        _whole("free_count", free_count, int32, 1, device))
    batch = PagedBatch(torch.empty(requests + 1, dtype=int32, device=device),
                       torch.empty(max_tokens, dtype=torch.int64, device=device),
                       torch.empty(max_tokens, dtype=torch.int64, device=device),
                       torch.empty(max_tokens, dtype=int32, device=device),
                       torch.empty(requests, dtype=int32, device=device))
    args.offsets, args.slots, args.positions, args.rows, args.granted = (t.data_ptr() for t in batch)
    _call(rt.load_library().mb_paged_reserve, args, index, "mb_paged_reserve")
    return batch


def paged_append(key: torch.Tensor, value: torch.Tensor, key_pages: torch.Tensor, value_pages: torch.Tensor,
                 slots: torch.Tensor) -> None:
    """Write ``key`` and ``value`` (``[tokens, kv_heads, head_dim]``) into the slots (int64 ``[tokens]``) of the pools.
    A slot outside the pool, as -1 behind the last token, is skipped; slots of one call are distinct (of two tokens
    with one slot either may be the one that stays)."""
    kpool, vpool = _pools(key_pages, value_pages)
    pages, page_size, kv_heads, head_dim = key_pages.shape
    if key.dim() != 3 or key.device.type != "cuda":
        fail("input-binding", f"key must be [tokens, kv_heads, head_dim] on a CUDA device, got {tuple(key.shape)} on "
                              f"{key.device}")
    tokens = key.shape[0]
    _inference_only(key, value, key_pages, value_pages)
    k = _rows("key", key, (tokens, kv_heads, head_dim), key_pages)
    v = _rows("value", value, (tokens, kv_heads, head_dim), key_pages)
    at = _whole("slots", slots, torch.int64, tokens, key.device)
    index = _device_ready(key.device)
    if tokens == 0:
        return
    args = rt.PagedAppendArgs(tokens, kv_heads, head_dim, pages, page_size, 0, k[1], k[2], v[1], v[2], *kpool[1:],
                              *vpool[1:], k[0], v[0], kpool[0], vpool[0], at)
    _call(rt.load_library().mb_paged_append, args, index, "mb_paged_append")


def _attention(what, function, workspace_of, query, key, value, key_pages, value_pages, block_table, lengths, index,
               index_name, index_numel, scale, out, status):
    kpool, vpool = _pools(key_pages, value_pages)
    pages, page_size, kv_heads, head_dim = key_pages.shape
    device = query.device
    if query.dim() != 3 or query.shape[2] != head_dim or query.shape[1] % kv_heads or query.shape[1] < 1 or \
            device.type != "cuda":
        fail("input-binding", f"query must be [tokens, heads, {head_dim}] on a CUDA device with heads a multiple of "
                              f"{kv_heads}, got {tuple(query.shape)} on {device}")
    if block_table.dim() != 2 or min(block_table.shape) < 1 or block_table.shape[1] * page_size > 0x7fffffff:
        fail("input-binding", f"block_table must be [requests, width] with rows below 2**31 tokens, got "
                              f"{tuple(block_table.shape)} pages of {page_size}")
    _inference_only(query, key, value, key_pages, value_pages)
    tokens, heads = query.shape[0], query.shape[1]
    requests, width = block_table.shape
    if index is None and requests != tokens:
        fail("input-binding", f"{tokens} queries need a row of the table each, or {index_name}; the table has {requests}")
    q = _rows("query", query, query.shape, key_pages)
    k = v = (0, 0, 0)
    if key is not None or value is not None:
        if key is None or value is None:
            fail("input-binding", "key and value come together")
        k = _rows("key", key, (tokens, kv_heads, head_dim), key_pages)
        v = _rows("value", value, (tokens, kv_heads, head_dim), key_pages)
    int32 = torch.int32
    table = _whole("block_table", block_table, int32, requests * width, device)
    held = _whole("lengths", lengths, int32, requests, device)
    at = 0 if index is None else _whole(index_name, index, int32, index_numel, device)
    zero_rest = out is None
    if out is None:
        out = torch.empty((tokens, heads, head_dim), dtype=query.dtype, device=device)
    elif out.dtype != query.dtype or out.shape != query.shape or out.device != device or not out.is_contiguous() or \
            out.data_ptr() % 16:
        fail("input-binding", f"out must be a contiguous {query.dtype} {tuple(query.shape)} tensor on {device} that "
                              "starts on a 16-byte boundary")
    device_index = _device_ready(device)
    if tokens == 0:
        return out
    args = rt.PagedAttentionArgs(
        _ELEMENTS[query.dtype], tokens, requests, heads, kv_heads, head_dim, width, pages, page_size, zero_rest,
        head_dim ** -0.5 if scale is None else scale, 0, q[1], q[2], k[1], k[2], v[1], v[2], *kpool[1:], *vpool[1:],
        q[0], k[0], v[0], kpool[0], vpool[0], table, held, at, out.data_ptr(), 0,
        0 if status is None else _whole("status", status, int32, 1, device))
    need = workspace_of(ctypes.byref(args))
    if need < 0:
        rt._check(rt.load_library(), -need, "resource-admission", what)
    if need:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
        args.workspace = workspace.data_ptr()
    _call(function, args, device_index, what)
    return out


def paged_kv_attention(query: torch.Tensor, key: torch.Tensor | None, value: torch.Tensor | None,
                       key_pages: torch.Tensor, value_pages: torch.Tensor, block_table: torch.Tensor,
                       lengths: torch.Tensor, rows: torch.Tensor | None = None, *, scale: float | None = None,
                       out: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one token a request over its paged cache: ``query`` ``[tokens, heads, head_dim]`` ->
    ``[tokens, heads, head_dim]``.

    Query ``t`` belongs to request ``rows[t]`` (int32 ``[tokens]``; ``t`` itself without ``rows``) and attends all
    ``lengths`` keys of that request; positions on pages outside the pool do not count.  Where nothing is left (an idle
    place with row -1, length 0) its output is zero.  With ``key`` and ``value`` (``[tokens, kv_heads, head_dim]``) the
    last position of the request is the token's own, appended first in the same call: ``lengths`` counts it already
    (``paged_reserve`` does), and ``rows`` names no request twice.  Without them several queries may read one
    request.  ``scale`` defaults to ``head_dim ** -0.5``.  ``status`` (int32 ``[1]``) receives a status code if a wait
    inside the kernel ran out."""
    lib = rt.load_library()
    return _attention("mb_paged_attention", lib.mb_paged_attention, lib.mb_paged_attention_workspace, query, key, value,
                      key_pages, value_pages, block_table, lengths, rows, "rows", query.shape[0], scale, out, status)


def paged_prefill_attention(query: torch.Tensor, key_pages: torch.Tensor, value_pages: torch.Tensor,
                            block_table: torch.Tensor, lengths: torch.Tensor, offsets: torch.Tensor, *,
                            scale: float | None = None, out: torch.Tensor | None = None,
                            status: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of several new tokens a request over its paged cache: ``query`` ``[tokens, heads, head_dim]``
    -> ``[tokens, heads, head_dim]``.

    Request ``r`` has the queries ``offsets[r] .. offsets[r + 1] - 1`` (int32 ``[requests + 1]``, as ``paged_reserve``
    gives them): its last positions, whose keys and values have been appended.  The one at position ``p`` attends the
    keys ``0 .. p`` that lie on pages of the pool: whole prompts, or a chunk after what is cached.  Queries behind
    the last request are zero in a new output; rows of an ``out`` that is given stay as they were there.  ``scale`` and
    ``status`` as for ``paged_kv_attention``."""
    lib = rt.load_library()
    return _attention("mb_paged_prefill", lib.mb_paged_prefill, lib.mb_paged_prefill_workspace, query, None, None,
                      key_pages, value_pages, block_table, lengths, offsets, "offsets", block_table.shape[0] + 1, scale,
                      out, status)
