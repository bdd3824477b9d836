"""The operators around a paged key-value cache, plain and in 64 bits, with bounds for what a kernel may be off by."""

from __future__ import annotations

import torch


def pages_of(tokens: int, page: int) -> int:
    return -(-tokens // page)


def reserve(counts, lengths, table, stack, free, page, max_tokens):
    """``paged_reserve`` on lists: new (lengths, table, stack, free), then (offsets, slots, positions, rows, granted)."""
    lengths, table, stack = list(lengths), [list(row) for row in table], list(stack)
    width, kept, granted = len(table[0]), [], [0] * len(counts)
    for r, count in enumerate(counts):
        kept.append(max(lengths[r] + count, 0) if count < 0 else lengths[r])
    for r in reversed(range(len(counts))):
        for j in reversed(range(pages_of(kept[r], page), pages_of(lengths[r], page))):
            stack[free] = table[r][j]
            free += 1
            table[r][j] = -1
        granted[r] = kept[r] - lengths[r]
    tokens = pages = 0
    available = free
    slots, positions, rows, offsets = [], [], [], [0]
    for r, count in enumerate(counts):
        if count > 0 and kept[r] + count <= width * page:
            need = pages_of(kept[r] + count, page) - pages_of(kept[r], page)
            tokens, pages = tokens + count, pages + need
            if tokens <= max_tokens and (need == 0 or pages <= available):
                granted[r] = count
                for j in range(pages_of(kept[r], page), pages_of(kept[r] + count, page)):
                    free -= 1
                    table[r][j] = stack[free]
                for position in range(kept[r], kept[r] + count):
                    slots.append(table[r][position // page] * page + position % page)
                    positions.append(position)
                    rows.append(r)
        offsets.append(len(slots))
        lengths[r] = kept[r] + max(granted[r], 0)
    rest = max_tokens - len(slots)
    return (lengths, table, stack, free), (offsets, slots + [-1] * rest, positions + [0] * rest, rows + [-1] * rest,
                                           granted)


def attend(query, key_pages, value_pages, row, length, scale, *, new_key=None, new_value=None):
    """One query ``[heads, D]`` over the first ``length`` positions of a request (``row``: its line of the table), in 64
    bits.  ``new_key`` / ``new_value`` stand in for the last position, if it has a page.  Returns the output and what it is made of:
    the sum of weights times magnitudes of values, and the largest sum of magnitudes in a score."""
    pages, page, kv_heads, dim = key_pages.shape
    heads = query.shape[0]
    zero = torch.zeros(heads, dim, dtype=torch.float64, device=query.device)
    length = max(0, min(length, row.numel() * page))
    entries = row[:pages_of(length, page)].long()
    place = torch.arange(length, device=query.device)
    entry = entries[place // page] if length else entries
    keep = (entry >= 0) & (entry < pages)
    if not bool(keep.any()):
        return zero, zero, zero[:, :1]
    entry, place = entry.clamp(0, pages - 1), place % page
    keys, values = key_pages[entry, place].double(), value_pages[entry, place].double()
    if new_key is not None:
        keys[-1], values[-1] = new_key.double(), new_value.double()
    keys, values = (t[keep].repeat_interleave(heads // kv_heads, dim=1) for t in (keys, values))
    scores = torch.einsum("hd,lhd->hl", query.double(), keys) * scale
    magnitude = torch.einsum("hd,lhd->hl", query.double().abs(), keys.abs()) * abs(scale)
    weights = torch.softmax(scores, dim=-1)
    return (torch.einsum("hl,lhd->hd", weights, values), torch.einsum("hl,lhd->hd", weights, values.abs()),
            magnitude.amax(-1, keepdim=True))


def tolerance(result, keys: int, dtype: torch.dtype, weight_rounding: float):
    """What an output may be off by.

    A score is a sum of D products in 32 bits, every partial sum off by at most 2^-23 of the sum of magnitudes M (an
    addition inside the matrix unit may cut instead of round): D 2^-23 M; the factors of scale and log2 e add
    2^-22 |s| <= 2^-22 M.  A weight is then off by that, relatively, by 2.7e-6 at most for the exponential, and by
    39 2^-24 for the rounding of a maximum that is moved by up to 39, together less than 2^-17, in the numerator and in the
    denominator; sums over n keys add n 2^-23 each; ``weight_rounding`` is the relative error of a weight as
    the second product takes it.  All of it multiplies the sum of weights times magnitudes of values; the rounding of
    the output, half a step of its type, comes on top."""
    out, magnitude, score = result
    half = torch.finfo(dtype).eps / 2
    dim = out.shape[-1]
    relative = 2 * ((dim + 2) * 2.0 ** -23 * score + 2.0 ** -17 + keys * 2.0 ** -23) + weight_rounding
    before = relative * magnitude
    return before + half * (out.abs() + before) + torch.finfo(dtype).tiny * half


# A decode weight goes into the second product as two 16-bit numbers, a prompt's as one.
def decode_rounding(dtype: torch.dtype) -> float:
    return 2 * (torch.finfo(dtype).eps / 2) ** 2


def prompt_rounding(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2
