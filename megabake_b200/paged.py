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
any number of query heads per key head (128 for prompts); pages of 8 to 1,024 tokens (a power of two); pools and rows may have any
strides that are multiples of 16 bytes.  Scores, softmax statistics and sums are fp32, weights meet the values as two 16-bit
numbers for single tokens (16 bits for bf16, 22 for fp16) and as one for prompts, and outputs are rounded once --
unlike ``kv_attention``, whose rounding points are the reference's eager ones.  Inference only.

The reference has one contiguous cache and one length per batch (``fx_handler/hf_attention.py:194-196``);
per-request state is a step of its roadmap (``docs/roadmap.md:178``).
"""

from __future__ import annotations

import struct
from typing import NamedTuple

import torch

from . import runtime as rt
from .diagnostics import fail

__all__ = ["PagedBatch", "PagedState", "paged_append", "paged_kv_attention", "paged_prefill_attention",
           "paged_reserve"]

_ELEMENTS = {torch.bfloat16: 0, torch.float16: 1}
_HEAD_DIMS = (64, 128, 256)
_MAX_REQUESTS = 2048
_MAX_TOKENS = 1 << 30     # of a row of the table, and places of a reservation
_MAX_COUNT = 0x7fffffff   # of pages, and of tokens


class PagedBatch(NamedTuple):
    """Where the tokens of one ``paged_reserve`` go.  Row ``r`` of the table has the places ``offsets[r]`` ..
    ``offsets[r + 1] - 1``; places behind the last token hold slot -1, position 0 and row -1."""

    offsets: torch.Tensor     # int32 [requests + 1]
    slots: torch.Tensor       # int64 [max_tokens]: page * page_size + place in the page
    positions: torch.Tensor   # int64 [max_tokens]
    rows: torch.Tensor        # int32 [max_tokens]
    granted: torch.Tensor     # int32 [requests]: tokens granted, negative: dropped


class PagedState:
    """The tensors of a paged cache: pools per layer, one block table, lengths, the stack of free pages, and a status word for
    the attention operators (``status=state.status``, read by ``check``).

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
        self.status = torch.empty(1, dtype=torch.int32, device=device)
        self.reset()

    def reset(self) -> None:
        """Every request empty, every page free; page 0 is handed out first.  No fault is on record."""
        pages = self.free_pages.numel()
        self.block_table.fill_(-1)
        self.lengths.zero_()
        self.free_pages.copy_(torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=self.free_pages.device))
        self.free_count.fill_(pages)
        self.status.zero_()

    def check(self) -> None:
        """Synchronise the device and raise ``CompilerError`` if a kernel that was given ``status`` recorded a fault (a wait
        that ran out): outputs since the last check are not valid, nor is what was appended of them."""
        if self.status.is_cuda:
            torch.cuda.synchronize(self.status.device)   # steps may run on any stream
        code = int(self.status)
        if code:
            self.status.zero_()
            fail("runtime", f"device status {rt.STATUS_NAMES.get(code, code)}: "
                            f"{rt.load_library().mb_status_string(code).decode()}")

    def reserve(self, counts: torch.Tensor, max_tokens: int) -> PagedBatch:
        """``paged_reserve`` on these tensors."""
        return paged_reserve(counts, self.lengths, self.block_table, self.free_pages, self.free_count,
                             self.page_size, max_tokens)


def _page_size_covered(page_size: int) -> bool:
    return 8 <= page_size <= 1024 and page_size & (page_size - 1) == 0


# ---------------------------------------------------------------------------------------
# What a call costs the host decides what a small one takes.  All that follows from the tensors' types, shapes, strides
# and devices -- whether they fit, the fields of the native arguments, the size of the scratch -- is worked out once for
# every combination of them and found again under it; what is left for a call are addresses.  (One
# token of one request, 9/3 heads of 64: 27.8 -> 12.4 us a call; 32 requests reserved: 19.6 -> 14.8.)
# ---------------------------------------------------------------------------------------
_known: dict[tuple, tuple] = {}
_MAX_KNOWN = 1024
_raw_stream = torch._C._cuda_getCurrentRawStream   # torch.cuda.current_stream(index).cuda_stream without its object


def _remember(signature: tuple, found: tuple) -> tuple:
    if len(_known) >= _MAX_KNOWN:   # a program whose shapes never come back
        _known.clear()
    _known[signature] = found
    return found


def _optional(tensor: torch.Tensor | None):
    return None if tensor is None else (tensor.dtype, tensor.get_device(), tensor.shape, tensor.stride())


def _native_device(device: torch.device) -> int:
    from .engine import _require_native_device

    _require_native_device(device)
    return device.index


def _whole(name: str, tensor: torch.Tensor, dtype: torch.dtype, shape: tuple, device: torch.device) -> None:
    """A contiguous tensor of whole numbers; the shape of a single one does not matter."""
    if tensor.dtype != dtype or tensor.device != device or not tensor.is_contiguous() or \
            tensor.shape != shape and not (shape == (1,) and tensor.numel() == 1):
        fail("input-binding", f"{name} must be a contiguous {dtype} tensor {list(shape)} on {device}, got "
                              f"{tensor.dtype} {list(tensor.shape)} on {tensor.device}")


def _rows(name: str, tensor: torch.Tensor, shape: tuple, like: torch.Tensor) -> tuple:
    """Strides of ``[..., head_dim]`` values that are read 16 bytes at a time; that of a single place, which is never gone
    along, as if the next one followed at once."""
    if tensor.dtype != like.dtype or tensor.device != like.device or tensor.shape != shape:
        fail("input-binding", f"{name} must be {like.dtype} {tuple(shape)} on {like.device}, got {tensor.dtype} "
                              f"{tuple(tensor.shape)} on {tensor.device}")
    strides = tuple(shape[-1] if places == 1 else stride for places, stride in zip(shape, tensor.stride()))
    if strides[-1] != 1 or any(stride % 8 for stride in strides[:-1]):
        _misaligned(name)
    return strides[:-1]


def _misaligned(name: str) -> None:
    fail("input-binding", f"{name} must have a contiguous last dimension and start, in every dimension, on 16-byte "
                          "boundaries")


def _check_aligned(**addresses: int) -> None:
    for name, address in addresses.items():
        if address & 15:
            _misaligned(name)


def _inference_only(*tensors) -> None:
    for tensor in tensors:
        if tensor is not None and tensor.requires_grad:
            raise RuntimeError("MegaBake supports inference only")


def _pools(key_pages: torch.Tensor, value_pages: torch.Tensor) -> tuple:
    if key_pages.dtype not in _ELEMENTS or key_pages.dim() != 4 or key_pages.shape[3] not in _HEAD_DIMS or \
            not _page_size_covered(key_pages.shape[1]) or not 1 <= key_pages.shape[0] <= _MAX_COUNT or \
            key_pages.shape[2] < 1:
        fail("input-binding", "key_pages must be bf16 or fp16 [pages, page_size, kv_heads, head_dim] with head_dim 64, "
                              "128 or 256 and page_size a power of two from 8 to 1024, got "
                              f"{key_pages.dtype} {tuple(key_pages.shape)}")
    return (_rows("key_pages", key_pages, key_pages.shape, key_pages),
            _rows("value_pages", value_pages, key_pages.shape, key_pages))


def _call(function, args: bytes, index: int, what: str) -> None:
    stream = _raw_stream(index)
    if index == torch.cuda.current_device():
        code = function(args, stream)
    else:
        with torch.cuda.device(index):
            code = function(args, stream)
    if code:
        rt._check(rt.load_library(), code, "runtime", what)


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
    page_size, max_tokens = int(page_size), int(max_tokens)
    signature = (counts.dtype, counts.get_device(), counts.shape, counts.stride(), lengths.dtype, lengths.get_device(),
                 lengths.shape, lengths.stride(), block_table.dtype, block_table.get_device(), block_table.shape,
                 block_table.stride(), free_pages.dtype, free_pages.get_device(), free_pages.shape, free_pages.stride(),
                 free_count.dtype, free_count.get_device(), free_count.shape, page_size, max_tokens)
    fields, index = _known.get(signature) or _remember(signature, _reserve_fields(
        counts, lengths, block_table, free_pages, free_count, page_size, max_tokens))
    slots = torch.empty(max_tokens, dtype=torch.int64, device=counts.device)
    batch = PagedBatch(counts.new_empty(counts.shape[0] + 1), slots, torch.empty_like(slots),
                       counts.new_empty(max_tokens), torch.empty_like(counts))
    args = fields + _RESERVE_ADDRESSES.pack(
        counts.data_ptr(), lengths.data_ptr(), block_table.data_ptr(), free_pages.data_ptr(), free_count.data_ptr(),
        batch[0].data_ptr(), slots.data_ptr(), batch[2].data_ptr(), batch[3].data_ptr(), batch[4].data_ptr())
    _call(rt.load_library().mb_paged_reserve, args, index, "mb_paged_reserve")
    return batch


_RESERVE_ADDRESSES = struct.Struct("=10Q")


def _reserve_fields(counts, lengths, block_table, free_pages, free_count, page_size, max_tokens) -> tuple:
    if block_table.dim() != 2:
        fail("input-binding", f"block_table must be [requests, width], got {tuple(block_table.shape)}")
    device = counts.device
    requests, width = block_table.shape
    for name, tensor, shape in (("counts", counts, (requests,)), ("lengths", lengths, (requests,)),
                                ("block_table", block_table, (requests, width)),
                                ("free_pages", free_pages, (free_pages.numel(),)), ("free_count", free_count, (1,))):
        _whole(name, tensor, torch.int32, shape, device)
    if device.type != "cuda" or not 1 <= requests <= _MAX_REQUESTS or width < 1 or not _page_size_covered(page_size) or \
            max_tokens < 0 or max_tokens > _MAX_TOKENS or width * page_size > _MAX_TOKENS or \
            requests * width > _MAX_COUNT or not 1 <= free_pages.numel() <= _MAX_COUNT:
        fail("input-binding", f"paged_reserve needs 1..{_MAX_REQUESTS} requests on a CUDA device, pages of 8 to 1024 tokens "
                              "(a power of two), rows of at most 2**30 tokens, max_tokens up to that and fewer than 2**31 "
                              "entries of the table, got "
                              f"{tuple(block_table.shape)} pages of {page_size} on {device}, max_tokens {max_tokens}")
    args = rt.PagedReserveArgs(requests, width, free_pages.numel(), page_size, max_tokens)
    return bytes(args)[:rt.PagedReserveArgs.counts.offset], _native_device(device)


def paged_append(key: torch.Tensor, value: torch.Tensor, key_pages: torch.Tensor, value_pages: torch.Tensor,
                 slots: torch.Tensor) -> None:
    """Write ``key`` and ``value`` (``[tokens, kv_heads, head_dim]``) into the slots (int64 ``[tokens]``) of the pools.
    A slot outside the pool, as -1 behind the last token, is skipped; slots of one call are distinct (where two tokens
    name one slot, its place holds parts of both)."""
    if torch.is_grad_enabled():
        _inference_only(key, value, key_pages, value_pages)
    signature = (key.dtype, key.get_device(), key.shape, key.stride(), value.dtype, value.get_device(), value.shape,
                 value.stride(), key_pages.dtype, key_pages.get_device(), key_pages.shape, key_pages.stride(),
                 value_pages.dtype, value_pages.get_device(), value_pages.shape, value_pages.stride(), slots.dtype,
                 slots.get_device(), slots.shape, slots.stride())
    fields, index = _known.get(signature) or _remember(signature, _append_fields(key, value, key_pages, value_pages, slots))
    if key.shape[0] == 0:
        return
    addresses = (key.data_ptr(), value.data_ptr(), key_pages.data_ptr(), value_pages.data_ptr())
    if (addresses[0] | addresses[1] | addresses[2] | addresses[3]) & 15:
        _check_aligned(key=addresses[0], value=addresses[1], key_pages=addresses[2], value_pages=addresses[3])
    _call(rt.load_library().mb_paged_append, fields + _APPEND_ADDRESSES.pack(*addresses, slots.data_ptr()), index,
          "mb_paged_append")


_APPEND_ADDRESSES = struct.Struct("=5Q")


def _append_fields(key, value, key_pages, value_pages, slots) -> tuple:
    kpool, vpool = _pools(key_pages, value_pages)
    pages, page_size, kv_heads, head_dim = key_pages.shape
    if key.dim() != 3 or key.shape[0] > _MAX_COUNT or key.device.type != "cuda":
        fail("input-binding", f"key must be [tokens, kv_heads, head_dim] on a CUDA device, got {tuple(key.shape)} on "
                              f"{key.device}")
    tokens = key.shape[0]
    k = _rows("key", key, (tokens, kv_heads, head_dim), key_pages)
    v = _rows("value", value, (tokens, kv_heads, head_dim), key_pages)
    _whole("slots", slots, torch.int64, (tokens,), key.device)
    args = rt.PagedAppendArgs(tokens, kv_heads, head_dim, pages, page_size, 0, *k, *v, *kpool, *vpool)
    return bytes(args)[:rt.PagedAppendArgs.key.offset], _native_device(key.device)


_ATTENTION_ADDRESSES = struct.Struct("=11Q")


def _attention(what, query, key, value, key_pages, value_pages, block_table, lengths, index, scale, out, status):
    if torch.is_grad_enabled():
        _inference_only(query, key, value, key_pages, value_pages)
    if scale is not None:
        scale = float(scale)
    signature = (what, query.dtype, query.get_device(), query.shape, query.stride(), key_pages.dtype,
                 key_pages.get_device(), key_pages.shape, key_pages.stride(), value_pages.dtype, value_pages.get_device(),
                 value_pages.shape, value_pages.stride(), block_table.dtype, block_table.get_device(), block_table.shape,
                 block_table.stride(), lengths.dtype, lengths.get_device(), lengths.shape, lengths.stride(), scale,
                 _optional(key), _optional(value), _optional(index), _optional(out), _optional(status))
    fields, workspace_bytes, device_index = _known.get(signature) or _remember(
        signature, _attention_fields(what, query, key, value, key_pages, value_pages, block_table, lengths, index, scale,
                                     out, status))
    if out is None:
        out = query.new_empty(query.shape)
    if query.shape[0] == 0:
        return out
    q, kpool, vpool, to = query.data_ptr(), key_pages.data_ptr(), value_pages.data_ptr(), out.data_ptr()
    k, v = (0, 0) if key is None else (key.data_ptr(), value.data_ptr())
    if (q | k | v | kpool | vpool | to) & 15:
        _check_aligned(query=q, key=k, value=v, key_pages=kpool, value_pages=vpool, out=to)
    workspace = query.new_empty(workspace_bytes, dtype=torch.uint8) if workspace_bytes else None
    args = fields + _ATTENTION_ADDRESSES.pack(
        q, k, v, kpool, vpool, block_table.data_ptr(), lengths.data_ptr(), 0 if index is None else index.data_ptr(), to,
        0 if workspace is None else workspace.data_ptr(), 0 if status is None else status.data_ptr())
    _call(getattr(rt.load_library(), what), args, device_index, what)
    return out


def _attention_fields(what, query, key, value, key_pages, value_pages, block_table, lengths, index, scale, out,
                      status) -> tuple:
    prefill = what == "mb_paged_prefill"
    index_name = "offsets" if prefill else "rows"
    kpool, vpool = _pools(key_pages, value_pages)
    pages, page_size, kv_heads, head_dim = key_pages.shape
    device = query.device
    if query.dim() != 3 or query.shape[2] != head_dim or query.shape[1] % kv_heads or query.shape[1] < 1 or \
            query.shape[0] > _MAX_COUNT or device.type != "cuda":
        fail("input-binding", f"query must be [tokens, heads, {head_dim}] on a CUDA device with heads a multiple of "
                              f"{kv_heads}, got {tuple(query.shape)} on {device}")
    tokens, heads = query.shape[0], query.shape[1]
    if block_table.dim() != 2 or min(block_table.shape) < 1 or block_table.shape[1] * page_size > _MAX_TOKENS:
        fail("input-binding", f"block_table must be [requests, width] with rows of at most 2**30 tokens, got "
                              f"{tuple(block_table.shape)} pages of {page_size}")
    requests, width = block_table.shape
    if requests > _MAX_REQUESTS or (not prefill and tokens > _MAX_REQUESTS):
        fail("input-binding", f"a call takes at most {_MAX_REQUESTS} requests, got {max(requests, tokens)}")
    if index is None and (prefill or requests != tokens):
        fail("input-binding", f"{tokens} queries need a row of the table each, or {index_name}; the table has {requests}")
    q = _rows("query", query, query.shape, key_pages)
    k = v = (0, 0)
    if key is not None or value is not None:
        if key is None or value is None:
            fail("input-binding", "key and value come together")
        k = _rows("key", key, (tokens, kv_heads, head_dim), key_pages)
        v = _rows("value", value, (tokens, kv_heads, head_dim), key_pages)
    _whole("block_table", block_table, torch.int32, (requests, width), device)
    _whole("lengths", lengths, torch.int32, (requests,), device)
    if index is not None:
        _whole(index_name, index, torch.int32, (requests + 1 if prefill else tokens,), device)
    if out is not None and (out.dtype != query.dtype or out.shape != query.shape or out.device != device or
                            not out.is_contiguous()):
        fail("input-binding", f"out must be a contiguous {query.dtype} {tuple(query.shape)} tensor on {device}")
    if status is not None:
        _whole("status", status, torch.int32, (1,), device)
    device_index = _native_device(device)
    args = rt.PagedAttentionArgs(_ELEMENTS[query.dtype], tokens, requests, heads, kv_heads, head_dim, width, pages, page_size,
                                 out is None, head_dim ** -0.5 if scale is None else scale, 0, *q, *k, *v, *kpool, *vpool)
    workspace_bytes = 0
    if tokens:
        # the size does not depend on addresses: any that are aligned as they have to be
        for name in ("query", "key_pages", "value_pages", "block_table", "lengths", "out"):
            setattr(args, name, 4096)
        args.key = args.value = 4096 if key is not None else 0
        args.index = 4096 if index is not None else 0
        lib = rt.load_library()
        with torch.cuda.device(device_index):
            workspace_bytes = getattr(lib, what + "_workspace")(bytes(args))
        if workspace_bytes < 0:
            rt._check(lib, -workspace_bytes, "resource-admission", what)
    fields = bytes(args)[:rt.PagedAttentionArgs.query.offset]
    return fields, workspace_bytes, device_index


def paged_kv_attention(query: torch.Tensor, key: torch.Tensor | None, value: torch.Tensor | None,
                       key_pages: torch.Tensor, value_pages: torch.Tensor, block_table: torch.Tensor,
                       lengths: torch.Tensor, rows: torch.Tensor | None = None, *, scale: float | None = None,
                       out: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one token a request over its paged cache: ``query`` ``[tokens, heads, head_dim]`` ->
    ``[tokens, heads, head_dim]``.

    Query ``t`` belongs to request ``rows[t]`` (int32 ``[tokens]``; ``t`` itself without ``rows``) and attends all
    ``lengths`` keys of that request (a row of the table at most); positions on pages outside the pool do not count.
    Where nothing is left (an idle place with row -1, length 0) its output is zero.  With ``key`` and ``value``
    (``[tokens, kv_heads, head_dim]``) the last position of the request is the token's own, appended first in the same
    call: ``lengths`` counts it already (``paged_reserve`` does), and ``rows`` names no request twice.  Without them several
    queries may read one request.  ``scale`` defaults to ``head_dim ** -0.5``.  ``status`` (int32 ``[1]``) receives a status
    code if a wait inside the kernel ran out."""
    return _attention("mb_paged_attention", query, key, value, key_pages, value_pages, block_table, lengths, rows, scale,
                      out, status)


def paged_prefill_attention(query: torch.Tensor, key_pages: torch.Tensor, value_pages: torch.Tensor,
                            block_table: torch.Tensor, lengths: torch.Tensor, offsets: torch.Tensor, *,
                            scale: float | None = None, out: torch.Tensor | None = None,
                            status: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of several new tokens a request over its paged cache: ``query`` ``[tokens, heads, head_dim]``
    -> ``[tokens, heads, head_dim]``.

    Request ``r`` has the queries ``offsets[r] .. offsets[r + 1] - 1`` (int32 ``[requests + 1]``, as ``paged_reserve``
    gives them, or any from 0 to ``tokens`` that do not fall): its last positions, whose keys and values have been appended.
    The one at position ``p`` attends the keys ``0 .. p`` that lie on pages of the pool: whole prompts, or a chunk after what
    is cached.  Queries before the first request and behind the last one are zero in a new output; rows of an ``out`` that is
    given stay as they were there.  ``scale`` and
    ``status`` as for ``paged_kv_attention``."""
    return _attention("mb_paged_prefill", query, None, None, key_pages, value_pages, block_table, lengths, offsets, scale,
                      out, status)
