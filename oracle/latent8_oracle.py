"""The 8-bit latent cache's operators, request by request on the CPU.

Rows are [.., 576] e4m3 codes with one scale per 128-token page and latent
head.  Codes are computed in fp32 as the operators define them (quotient or
product rounded once, then to nearest even), attention in fp64.  Nothing here
is fast; every rule is one line of its own.
"""

from __future__ import annotations

import math

import torch

PAGE, LATENT, ROPE = 128, 512, 64
F8 = torch.float8_e4m3fn


def spans(ends, rows: int):
    """Each request's packed rows (start, count); ends are clipped to [0, rows]."""
    out, lo = [], 0
    for e in ends:
        lo, hi = min(max(lo, 0), rows), min(max(int(e), 0), rows)
        hi = max(hi, lo)
        out.append((lo, hi - lo))
        lo = int(e)
    return out


def least_scale(amax: float) -> float:
    if amax <= 0:
        return 2.0 ** -126
    frac, power = math.frexp(amax)  # amax = frac * 2^power; 448 = 0.875 * 2^9
    power += -8 if frac > 0.875 else -9
    return 2.0 ** min(120, max(-126, power))


def append(kv, k_rope, ends, lengths, table, cache, scale, positions=None, entries=None, token_positions=None,
           token_weights=None) -> None:
    blocks, cols = cache.shape[0], table.shape[1]
    codes = cache.view(torch.uint8)
    for b, (start, n) in enumerate(spans(ends.tolist(), kv.shape[0])):
        pages: dict[int, list[int]] = {}
        for i in range(n):
            slot = int(lengths[b]) - n + i
            if 0 <= slot < cols * PAGE:
                pages.setdefault(slot // PAGE, []).append(i)
                e = int(entries[b]) if entries is not None else -1
                if token_positions is not None and 0 <= e < token_positions.shape[0]:
                    token_positions[e, slot] = positions[start + i]
                if token_weights is not None and 0 <= e < token_weights.shape[0]:
                    token_weights[e, slot] = 0.0
        for page, rows in pages.items():
            block = int(table[b, page])
            if not 0 <= block < blocks:
                continue
            first = (int(lengths[b]) - n + rows[0]) % PAGE
            for g in range(cache.shape[2]):
                x = torch.cat([kv[start + rows[0]:start + rows[-1] + 1, g],
                               k_rope[start + rows[0]:start + rows[-1] + 1, g]], -1).float()
                fine = x.isfinite()
                need = least_scale(float(torch.where(fine, x.abs(), 0.0).max()))
                old = scale[block, g].clone()
                now = old if first > 0 and float(old) >= need else torch.tensor(need, dtype=torch.float32)
                if first > 0 and not float(old) >= need:
                    older = cache[block, :first, g].float() * (old / now)
                    codes[block, :first, g] = older.to(F8).view(torch.uint8)
                new = torch.where(fine, x / now, math.nan).to(F8)
                codes[block, first:first + len(rows), g] = new.view(torch.uint8)
                scale[block, g] = now


def attention(query_rope, query, ends, lengths, table, cache, scale, softmax_scale, topk=None):
    """(out fp64 [T, N, 512], sums): sums[b] is the fp64 attention weight of
    each slot of request b's table, summed over its rows and heads.  Rows of no
    request are NaN in ``out`` (nothing says what they hold)."""
    rows, heads, _ = query.shape
    blocks, cols, g_count = cache.shape[0], table.shape[1], cache.shape[2]
    per = heads // g_count
    out = torch.full((rows, heads, LATENT), math.nan, dtype=torch.float64)
    size = torch.zeros(rows, heads, LATENT, dtype=torch.float64)   # sum of p |v|
    reach = torch.zeros(rows, heads, dtype=torch.float64)          # largest |q| . |k| * softmax_scale
    sums = torch.zeros(len(ends), cols * PAGE, dtype=torch.float64)
    q = torch.cat([query, query_rope], -1).double()
    for b, (start, n) in enumerate(spans(ends.tolist(), rows)):
        length = min(max(int(lengths[b]), 0), cols * PAGE)
        pages = table[b].long()
        good = (pages >= 0) & (pages < blocks)
        kv = cache.view(torch.uint8)[pages.clamp(0, blocks - 1)].view(F8).double()
        kv = kv * scale[pages.clamp(0, blocks - 1)].double()[:, None, :, None]
        kv = kv.flatten(0, 1)                                       # [slots, G, 576]
        good = good.repeat_interleave(PAGE)
        for i in range(n):
            sees = max(0, length - (n - 1 - i))
            if topk is None:
                keys = torch.arange(sees)[good[:sees]]
            else:
                ids = topk[start + i].long()
                ids = ids[(ids >= 0) & (ids < sees)]
                keys = ids[good[ids]]
            if len(keys) == 0:
                out[start + i] = 0.0
                continue
            for h in range(heads):
                k = kv[keys, h // per]
                p = torch.softmax((k @ q[start + i, h]) * softmax_scale, 0)
                out[start + i, h] = p @ k[:, :LATENT]
                size[start + i, h] = p @ k[:, :LATENT].abs()
                reach[start + i, h] = (k.abs() @ q[start + i, h].abs()).max() * softmax_scale
                if topk is None:
                    sums[b, keys] += p
    return out, sums, size, reach


def evict(lengths, budgets, table, entries, cache, scale, token_positions, token_weights, first, last):
    """(moves, kept): per request the list of (source, hole) slots and the new
    length; cache, scales and records are changed in place."""
    blocks, cols = cache.shape[0], table.shape[1]
    codes, before = cache.view(torch.uint8), scale.clone()
    moves, kept_lengths = [], []
    for b in range(len(lengths)):
        length = min(max(int(lengths[b]), 0), cols * PAGE)
        keep, e = min(length, max(int(budgets[b]), 0)), int(entries[b])
        if not 0 <= e < token_weights.shape[0]:
            keep = length
        kept_lengths.append(keep)
        if keep in (0, length):
            moves.append([])
            continue
        w, pos = token_weights[e, :length].tolist(), token_positions[e, :length].tolist()
        latest = max(pos)

        def order(t):
            held = pos[t] < first or pos[t] > latest - last
            return (-2 if held else -1 if math.isnan(w[t]) else 0, 0.0 if held or math.isnan(w[t]) else -w[t], t)

        kept = set(sorted(range(length), key=order)[:keep])
        holes = [t for t in range(keep) if t not in kept]
        sources = [t for t in range(keep, length) if t in kept]
        assert len(holes) == len(sources)
        moves.append(list(zip(sources, holes)))
        rows = {s: codes[int(table[b, s // PAGE]), s % PAGE].clone() for s in sources
                if 0 <= int(table[b, s // PAGE]) < blocks}
        for page in sorted({h // PAGE for h in holes}):
            block = int(table[b, page])
            mine = [(s, h) for s, h in moves[-1] if h // PAGE == page]
            if 0 <= block < blocks:
                froms = [int(table[b, s // PAGE]) for s, _ in mine]
                for g in range(cache.shape[2]):
                    old = before[block, g]
                    now = max([old] + [before[f, g] for f in froms if 0 <= f < blocks])
                    held = set(range(min(PAGE, keep - page * PAGE))) - {h % PAGE for _, h in mine}
                    if now != old:
                        at = torch.tensor(sorted(held), dtype=torch.long)
                        codes[block, at, g] = (cache[block].float()[at, g] * (old / now)).to(F8).view(torch.uint8)
                        scale[block, g] = now
                    for (s, h), f in zip(mine, froms):
                        if s in rows:
                            v = rows[s][g].view(F8).float() * (before[f, g] / now)
                            codes[block, h % PAGE, g] = v.to(F8).view(torch.uint8)
        for s, h in moves[-1]:
            token_weights[e, h], token_positions[e, h] = token_weights[e, s], token_positions[e, s]
    return moves, kept_lengths
