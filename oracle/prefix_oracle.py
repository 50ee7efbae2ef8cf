"""The prefix-sharing operators in plain 64-bit torch and Python, on the CPU.

Each function follows the operator's definition row by row; the page operators
work on lists of integers.
"""

from __future__ import annotations

import torch

PAGE = 128


def _spans(ends, rows: int):
    start = 0
    for end in ends.tolist():
        yield min(max(start, 0), rows), min(max(end, start, 0), rows)
        start = end


def slot_row(table_row, slot: int, pages: int) -> tuple[int, int] | None:
    """(page, row) of a slot, or None where it names nothing."""
    if slot < 0 or slot >= len(table_row) * PAGE:
        return None
    page = int(table_row[slot // PAGE])
    return (page, slot % PAGE) if 0 <= page < pages else None


def rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    out = torch.empty_like(x)
    out[..., 0::2] = x[..., 0::2] * cos[..., 0::2] - x[..., 1::2] * sin[..., 0::2]
    out[..., 1::2] = x[..., 1::2] * cos[..., 1::2] + x[..., 0::2] * sin[..., 1::2]
    return out


def rms(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight


def norm_rope(query, kv, cos, sin, kv_weight, ends, lengths, table, query_weight, eps):
    """(cache rows {(page, row): (latent, rope)}, query_rope, query_nope), all in 64 bits."""
    query, kv = query.double(), kv.double()
    cos, sin = cos.double()[:, :64], sin.double()[:, :64]
    rows = {}
    for b, (lo, hi) in enumerate(_spans(ends, kv.shape[0])):
        for t in range(lo, hi):
            at = slot_row(table[b], int(lengths[b]) - (hi - t), 1 << 62)
            if at is not None:
                rows[at] = (rms(kv[t, :512], kv_weight.double(), eps), rotate(kv[t, 512:], cos[t], sin[t]))
    nope = None
    if query_weight is not None:
        query = rms(query, query_weight.double(), eps)
        nope = query[..., :-64]
    return rows, rotate(query[..., -64:], cos[:, None], sin[:, None]), nope


def branch(lengths, new, table, refs, parents=None):
    """The operator on lists: (lengths, table, refs, copies, missing)."""
    batch, cols, pages = len(table), len(table[0]), len(refs)
    lengths, table, refs = list(lengths), [list(r) for r in table], list(refs)
    named = lambda p: 0 <= p < pages  # noqa: E731
    if parents is not None:
        old = [list(r) for r in table], list(lengths)
        for b, p in enumerate(parents):
            inside = 0 <= p < batch
            table[b], lengths[b] = (list(old[0][p]), old[1][p]) if inside else ([-1] * cols, 0)
        for sign, rows in ((1, table), (-1, old[0])):
            for row in rows:
                for p in row:
                    if named(p):
                        refs[p] += sign
    writes = []  # (first column, stop column, rows that stay in the first)
    for length, n in zip(lengths, new):
        length, end = max(length, 0), min(length + n, cols * PAGE)
        writes.append((length // PAGE, -(-end // PAGE), length % PAGE) if n > 0 and end > length else (0, 0, 0))
    takes = []
    for b, (first, stop, part) in enumerate(writes):
        for c in range(first, stop):
            p = table[b][c]
            if not named(p):
                takes.append((b, c, -1))
            elif refs[p] > 1:
                writers = [o for o, (f, _, older) in enumerate(writes) if older > 0 and table[o][f] == p]
                if not (c == first and part > 0 and refs[p] == len(writers) and writers[0] == b):
                    takes.append((b, c, p))
    free = [p for p, r in enumerate(refs) if r == 0]
    copies = [(-1, -1, 0)] * batch
    if len(takes) > len(free):
        return lengths, table, refs, copies, len(takes) - len(free)
    for (b, c, was), p in zip(takes, free):
        table[b][c], refs[p] = p, 1
        if was >= 0:
            refs[was] -= 1
            if c == writes[b][0] and writes[b][2] > 0:
                copies[b] = (was, p, writes[b][2])
    return lengths, table, refs, copies, 0


def compact(table, refs):
    """(table, refs, moves) on lists."""
    live = [p for p, r in enumerate(refs) if r > 0]
    below = set(p for p in live if p < len(live))
    moves = list(zip([p for p in live if p >= len(live)], [p for p in range(len(live)) if p not in below]))
    to, refs = dict(moves), list(refs)
    for src, dst in moves:
        refs[dst], refs[src] = refs[src], 0
    return [[to.get(p, p) for p in row] for row in table], refs, moves


def copy(cache: torch.Tensor, pairs, tokens=None) -> None:
    """In place; ``tokens`` for caches [P, 128, ...]."""
    rows = cache.dim() >= 3 and cache.shape[1] == PAGE
    for k, (src, dst) in enumerate(pairs):
        if not (0 <= src < cache.shape[0] and 0 <= dst < cache.shape[0]):
            continue
        n = PAGE if tokens is None else min(max(tokens[k], 0), PAGE)
        if rows:
            cache[dst, :n] = cache[src, :n]
        elif n > 0:
            cache[dst] = cache[src]


def attention(query_rope, query, ends, lengths, table, k_rope, kv_cache, scale):
    """(out, size, reach): the operator in 64 bits, and, for bounds, the sums of
    p |v| and the largest scale * sum |q| |k| of a row and head."""
    rows, heads, _ = query.shape
    pages = kv_cache.shape[0]
    q = torch.cat([query, query_rope], -1).double()
    out, size = (torch.zeros(rows, heads, 512, dtype=torch.float64) for _ in range(2))
    reach = torch.zeros(rows, heads, dtype=torch.float64)
    for b, (lo, hi) in enumerate(_spans(ends, rows)):
        cap, tokens = table.shape[1] * PAGE, int(lengths[b])
        length = min(max(tokens, 0), cap)
        row = table[b, : -(-length // PAGE)].long()
        named = ((row >= 0) & (row < pages)).repeat_interleave(PAGE)[:length]
        at = torch.where((row >= 0) & (row < pages), row, 0)
        keys = torch.cat([kv_cache[at].flatten(0, 2), k_rope[at].flatten(0, 2)], -1)[:length].double()
        for t in range(lo, hi):
            sees = min(max(0, tokens - (hi - 1 - t)), length)
            seen = keys[:sees][named[:sees]]
            if len(seen) == 0:
                continue
            p = torch.softmax(q[t] @ seen.T * scale, -1)
            out[t], size[t] = p @ seen[:, :512], p @ seen[:, :512].abs()
            reach[t] = (q[t].abs() @ seen.abs().T).amax(-1) * abs(scale)
    return out, size, reach
