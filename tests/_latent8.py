"""Inputs and comparisons of the 8-bit latent cache's tests."""

from __future__ import annotations

import torch

from oracle import latent8_oracle as O

PAGE = 128
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SCALE = 576 ** -0.5


def i32(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32)


def make_cache(lengths, latent_heads, seed, spare=2, cols=None, exponents=(-7, -5)):
    """CPU cache, scales, table and pool records for requests of these
    lengths; page order shuffled, unused table entries 0."""
    g = torch.Generator().manual_seed(seed)
    counts = [max(0, -(-n // PAGE)) for n in lengths]
    cols = cols or max(1, max(counts, default=1))
    blocks = sum(counts) + spare
    order = torch.randperm(blocks, generator=g).tolist()
    table = torch.zeros(len(lengths), cols, dtype=torch.int32)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = i32(order[at:at + n])
        at += n
    cache = (torch.randn(blocks, PAGE, latent_heads, 576, generator=g) * 70).clamp(-448, 448).to(torch.float8_e4m3fn)
    scale = torch.exp2(torch.randint(*exponents, (blocks, latent_heads), generator=g).float())
    return {"cache": cache, "scale": scale, "table": table, "lengths": i32(lengths), "cols": cols, "blocks": blocks}


def queries(counts, heads, dtype, seed, pad=0, size=2.0):
    g = torch.Generator().manual_seed(seed + 1000)
    total = sum(counts) + pad
    q = (torch.randn(total, heads, 512, generator=g) * size).to(dtype)
    qr = (torch.randn(total, heads, 64, generator=g) * size).to(dtype)
    return qr, q, torch.tensor(counts).cumsum(0).to(torch.int32)


def same_codes(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Equal e4m3 codes; any NaN equals any NaN."""
    a, b = a.cpu().view(torch.uint8), b.cpu().view(torch.uint8)
    nan = ((a & 0x7F) == 0x7F) & ((b & 0x7F) == 0x7F)
    return bool(((a == b) | nan).all())


def attention_bound(out, size, reach, dtype, keys: int, scale):
    """How far an output may be from the 64-bit one.  The store rounds by half
    a step of the result; P is rounded to fp16 (2^-11 of each p); sums of
    ``keys`` terms in fp32; a score of 576 products in fp32 is off by at most
    578 * 2^-24 of |q| . |k|, which moves p (and its normaliser) by that factor
    each, and the exponential by 2^-22 of itself and 2^-23 of its argument.
    A page's scale enters p through its logarithm, which for other scales than
    powers of two is off by half a step of at most 126 (2^-18) and the
    logarithm's own 2^-21: below 2^-17.8, times ln 2, 2^-18 of p, and of the
    normaliser as much.
    Below fp16's normal range a P is off by 2^-25 next to a largest one of at
    least 1 in units of its page's scale: 2^-25 * 448 of the largest scale a
    key, twice that for a scale's fraction."""
    score = reach * (578 * 2.0 ** -24 + 2.0 ** -22)
    per = 2.0 ** -11 + keys * 2.0 ** -23 + 2 * score + 2.0 ** -21 + 2.0 ** -17
    tail = keys * 2.0 ** -25 * 896 * float(scale.max())
    return out.abs() * HALF_STEP[dtype] + size * per[..., None] + tail


def weights_bound(added, total, reach, keys: int, terms: int):
    """How far a token's accumulated weight may be from the 64-bit one: every p
    by its score's factor (its own and its normaliser's), the exponential and
    the logarithm; the normaliser's sum of ``keys`` and the sum of ``terms``
    (rows times heads) round in fp32, and the addition to the record.  The
    normaliser holds the logarithm of the pages' scales (2^-18, see above)."""
    off = float(reach.max()) * (2 * 578 * 2.0 ** -24 + 2.0 ** -21) + 2.0 ** -20 + keys * 2.0 ** -23 + terms * 2.0 ** -24 \
        + 2.0 ** -18
    return added.abs() * off + total.abs() * 2.0 ** -23


def oracle_attention(qr, q, ends, c, topk=None):
    return O.attention(qr, q, ends, c["lengths"], c["table"], c["cache"], c["scale"], SCALE, topk)


def wide_attention(qr, q, ends, c, topk=None):
    """The operator in fp64, heads together: (out, sums, size, reach, tail);
    ``tail`` is the part of the bound below for keys whose P may lie below
    fp16's normal range, the others are those of the oracle."""
    rows, heads, _ = q.shape
    groups = c["cache"].shape[2]
    per, cap = heads // groups, c["cols"] * PAGE
    out, size, tail = (torch.zeros(rows, heads, 512, dtype=torch.float64) for _ in range(3))
    reach = torch.zeros(rows, heads, dtype=torch.float64)
    sums = torch.zeros(len(ends), cap, dtype=torch.float64)
    queries_ = torch.cat([q, qr], -1).double()
    start = 0
    for b, end in enumerate(ends.tolist()):
        n, length = end - start, int(c["lengths"][b])
        pages = c["table"][b].long()
        scale = c["scale"][pages].double().repeat_interleave(PAGE, 0)                 # [slots, G]
        codes = c["cache"].view(torch.uint8)[pages].view(torch.float8_e4m3fn).double().flatten(0, 1)
        for i in range(n):
            sees = max(0, length - (n - 1 - i))
            at = torch.arange(sees) if topk is None else topk[start + i].long()
            at = at[(at >= 0) & (at < sees)]
            if len(at) == 0:
                continue
            for g in range(groups):
                mine = slice(g * per, (g + 1) * per)
                x, y = queries_[start + i, mine], codes[at, g] * scale[at, g, None]
                p = torch.softmax(x @ y.T * SCALE, -1)
                out[start + i, mine], size[start + i, mine] = p @ y[:, :512], p @ y[:, :512].abs()
                reach[start + i, mine] = (x.abs() @ y.abs().T).amax(-1) * SCALE
                weight = p * scale[at, g]
                top = weight.amax(-1, keepdim=True)
                tail[start + i, mine] = torch.where(weight < top * 2.0 ** -22, top * 2.0 ** -33, 0.0) @ codes[at, g, :512].abs()
                if topk is None:
                    sums[b, at] += p.sum(0)
        start = end
    return out, sums, size, reach, tail


def wide_bound(out, size, reach, tail, dtype, keys: int):
    """How far an output may be from the 64-bit one, scales of any size.  As in
    :func:`attention_bound`, but exponents hold the logarithms of the scales
    (below 2^9 with the scores of these tests): each of the eight sums that an
    exponent passes through rounds by 2^-16, times ln 2 below 2^-13 together.
    A row's largest P is at least 2^8, so that those from 2^-22 of the largest
    p times scale on lie in fp16's normal range (2^-14); one below is off by
    2^-25, which is 2^-33 of the largest p times scale, times its key's code.  A
    subnormal output rounds by half of its type's step."""
    score = reach * (578 * 2.0 ** -24 + 2.0 ** -22)
    per = 2.0 ** -11 + keys * 2.0 ** -23 + 2 * score + 2.0 ** -21 + 2.0 ** -13
    step = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}[dtype]
    return out.abs() * HALF_STEP[dtype] + size * per[..., None] + tail + step
