"""A paged cache's requests in plain Python and numpy: block tables with a ring of free blocks, and attention in 64 bits."""

from __future__ import annotations

import numpy as np
import torch

MOST = (1 << 31) - 1


def ceil(a, b):
    return -(-a // b)


def resize(tables, held, lengths, ring, cursor, *, blocks, block_size, capacity=None):
    """The outputs of one call, from lists: a dict of tables, free, kept, cursor, slots, starts."""
    tables, ring = [list(row) for row in tables], list(ring)
    size = len(ring)
    first, count = (cursor[0] % size, min(max(cursor[1], 0), size)) if size else (0, 0)
    front, end = first, first + count
    room, taken, given, full = size - count, 0, 0, False
    kept, slots, starts, returns = [], [], [], []
    for r, (h, x) in enumerate(zip(held, lengths)):
        starts.append(len(slots))
        most = min(len(tables[r]) * block_size, MOST)
        if not 0 <= h <= most:
            kept.append(0)
            continue
        if not 0 <= x <= most:
            kept.append(h)
            continue
        before, after = ceil(h, block_size), ceil(x, block_size)
        if x > h:
            full |= taken + after - before > count or capacity is not None and len(slots) + x - h > capacity
            if full:
                kept.append(h)
                continue
            for c in range(before, after):
                tables[r][c] = ring[(front + taken) % size]
                taken += 1
            for i in range(h, x):
                name = tables[r][i // block_size]
                slots.append(name * block_size + i % block_size if 0 <= name < blocks else -1)
        else:
            returns += tables[r][after:before]
        kept.append(x)
    starts.append(len(slots))
    for name in returns:
        if given < room:
            ring[(end + given) % size] = name
            given += 1
    if capacity is not None:
        slots += [-1] * (capacity - len(slots))
    return {"tables": tables, "free": ring, "kept": kept, "cursor": [(first + taken) % size if size else 0, count - taken + given],
            "slots": slots, "starts": starts}


def tokens_of(table, length, window, block_size, blocks):
    """(block, row) of the tokens that a request attends to."""
    length = max(0, min(length, len(table) * block_size))
    low = max(0, length - window) if window else 0
    at = [(table[i // block_size], i % block_size) for i in range(low, length)]
    return [(b, r) for b, r in at if 0 <= b < blocks]


def attend(layer, query, tables, lengths, *, block_size, value_dim, scale, window=0):
    """out [requests, query_heads, value_dim], lse, and how far the kernels may be from them: float64 arrays.

    layer: [planes] list of [blocks, block_size, heads, head_dim] tensors on the CPU. With u = 2^-24, a score of d products has an
    error of at most (d + 4) 2 u scale sum |q k| (products in 32 bits, added in any order, rounded either way), which
    is an error of that size relative to its weight; a weight 4 u more for its exponential; a sum of n weights or of n products n 2 u;
    16-bit weights 2^-11 (half) or 2^-15 (bfloat16 as the sum of two, each with 8 bits). The result is then rounded to its type."""
    keys, values = layer[0].double().numpy(), layer[-1].double().numpy()[..., :value_dim]
    dtype = layer[0].dtype
    blocks, _, heads, dim = keys.shape
    q = query.double().numpy()
    n, query_heads, _ = q.shape
    group = query_heads // heads
    out, lse = np.zeros((n, query_heads, value_dim)), np.full((n, query_heads), -np.inf)
    far, lse_far = np.zeros_like(out), np.zeros_like(lse)
    step = {torch.bfloat16: 2.0 ** -15, torch.float16: 2.0 ** -11, torch.float32: 0.0}[dtype]
    for r in range(n):
        at = tokens_of(tables[r], lengths[r], window, block_size, blocks)
        if not at:
            continue
        b, row = np.array(at).T
        for h in range(heads):
            mine = slice(h * group, (h + 1) * group)
            k, v = keys[b, row, h], values[b, row, h]
            s = scale * (q[r, mine] @ k.T)
            m = s.max(-1, keepdims=True)
            p = np.exp(s - m)
            total = p.sum(-1, keepdims=True)
            lse[r, mine] = (m + np.log(total))[:, 0]
            out[r, mine] = p @ v / total
            e = (dim + 4) * 2.0 ** -23 * abs(scale) * (np.abs(q[r, mine]) @ np.abs(k).T) + 2.0 ** -22
            sums = len(at) * 2.0 ** -23 + 2.0 ** -21
            weights = p / total
            # of the weights themselves, and of the sum that divides them
            own = (weights * (np.expm1(e) + step)) @ np.abs(v)
            lse_far[r, mine] = ((weights * np.expm1(e)).sum(-1) + sums) * 1.01 + np.abs(lse[r, mine]) * 2.0 ** -22
            far[r, mine] = (own + (weights @ np.abs(v)) * (lse_far[r, mine][:, None] + sums)) * 1.01
    half = torch.finfo(dtype).eps / 2
    far = far + (np.abs(out) + far) * half + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return out, lse, far, lse_far
