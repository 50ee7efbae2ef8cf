"""Inputs and bounds of the prefix-sharing operators' tests."""

from __future__ import annotations

import torch

from oracle import prefix_oracle as O

PAGE = 128
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}  # half a step of the smallest values
SCALE = 576 ** -0.5


def i32(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32)


def gpu(*tensors):
    return [None if t is None else t.cuda() for t in tensors]


def api():
    from nanovllm_amd import prefix_sharing

    return prefix_sharing


def norm_inputs(counts, past, heads, nope, dtype, seed, pad=0, cols=None, norm=None, stride=64):
    """CPU tensors of a norm_rope_append call: requests of ``counts`` new rows
    behind ``past`` tokens, ``pad`` rows behind the last."""
    g = torch.Generator().manual_seed(seed)
    total = sum(counts) + pad
    pages = [-(-(c + p) // PAGE) for c, p in zip(counts, past)]
    cols = cols or max(1, max(pages, default=1))
    blocks = sum(pages) + 2
    order, at = torch.randperm(blocks, generator=g).to(torch.int32), 0
    table = torch.full((len(counts), cols), -1, dtype=torch.int32)
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    angle = torch.rand(total, stride // 2, generator=g) * 6.283
    angle = angle.repeat_interleave(2, 1)
    size = torch.exp2(torch.rand(total, 1, generator=g) * 4 - 2)
    norm = nope > 0 if norm is None else norm
    return {
        "query": (size[..., None] * rand(total, heads, nope + 64)).to(dtype), "kv": (size * rand(total, 576)).to(dtype),
        "cos": angle.cos().to(dtype), "sin": angle.sin().to(dtype), "kv_weight": (1 + 0.3 * rand(512)).to(dtype),
        "ends": torch.tensor(counts).cumsum(0).to(torch.int32), "lengths": i32([c + p for c, p in zip(counts, past)]),
        "table": table, "k_rope": rand(blocks, PAGE, 1, 64).to(dtype), "kv_cache": rand(blocks, PAGE, 1, 512).to(dtype),
        "query_rope": torch.full((total, heads, 64), 7.0).to(dtype),
        "query_weight": (1 + 0.3 * rand(nope + 64)).to(dtype) if norm else None,
        "query_nope": torch.full((total, heads, nope), 7.0).to(dtype) if norm else None,
    }


NORM_ARGS = ("query", "kv", "cos", "sin", "kv_weight", "ends", "lengths", "table", "k_rope", "kv_cache", "query_rope")


def call_norm(d, eps=1e-6):
    api().norm_rope_append(*[d[k] for k in NORM_ARGS], query_norm_weight=d["query_weight"], query_nope=d["query_nope"],
                           eps=eps)


def near(got, want, dtype, factor, size=None):
    """|got - want| within the store's half step and ``factor`` of ``size``
    (the magnitudes that went into a value; the value's own without)."""
    got, want = got.double(), want.double()
    size = want.abs() if size is None else size
    bound = want.abs() * HALF_STEP[dtype] + size * factor + TINY[dtype]
    # (A NaN bound comes of a NaN or infinite value, which has to be there as it is.)
    same = (got == want) | (got.isnan() & want.isnan())
    return bool((same | ((got - want).abs() <= bound)).all())


def check_norm(got, d, eps=1e-6):
    """``got``: CPU copies after the call, ``d``: the inputs before it.

    fp32: a sum of n squares is off by at most n 2^-24 of itself, the root and
    its reciprocal by 2^-22, two products by 2^-24 each: below 2^-14 + 2^-21
    for 576 values.  A rotated value is two products and a sum: 3 2^-24 of the
    magnitudes, beside what the norm brought."""
    dtype = d["kv"].dtype
    rows, rope, nope = O.norm_rope(d["query"], d["kv"], d["cos"], d["sin"], d["kv_weight"], d["ends"], d["lengths"],
                                   d["table"], d["query_weight"], eps)
    off = 2.0 ** -14 + 2.0 ** -21 + 2.0 ** -22
    seen = torch.zeros(d["kv_cache"].shape[:2], dtype=torch.bool)
    size_rope = lambda x: x.abs() + x.unflatten(-1, (-1, 2)).flip(-1).flatten(-2).abs()  # noqa: E731
    pages = d["kv_cache"].shape[0]
    for (page, row), (latent, turned) in rows.items():
        if not 0 <= page < pages:
            continue
        seen[page, row] = True
        assert near(got["kv_cache"][page, row, 0], latent, dtype, off), (page, row)
        # (Rotation keeps a pair's length: its magnitudes are below sqrt(2) of the pair's, within size_rope twice.)
        assert near(got["k_rope"][page, row, 0], turned, dtype, 2.0 ** -21, 2 * size_rope(turned)), (page, row)
    for k in ("kv_cache", "k_rope"):  # every other row as it was
        assert torch.equal(got[k][~seen].view(torch.int16), d[k][~seen].view(torch.int16)), k
    last = min(max(int(d["ends"][-1]), 0), d["kv"].shape[0])
    assert near(got["query_rope"][:last], rope[:last], dtype, off, 2 * size_rope(rope[:last]))
    assert torch.equal(got["query_rope"][last:].view(torch.int16), d["query_rope"][last:].view(torch.int16))
    if nope is not None:
        assert near(got["query_nope"][:last], nope[:last], dtype, off)
        assert torch.equal(got["query_nope"][last:].view(torch.int16), d["query_nope"][last:].view(torch.int16))


def make_pages(lengths, pages, cols, seed, shared=()):
    """Table and counts (lists) of requests of these lengths; ``shared``:
    (request, other, columns) take the other's first pages."""
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table, at = [], 0
    for n in lengths:
        k = max(0, -(-n // PAGE))
        table.append(order[at:at + k] + [-1] * (cols - k))
        at += k
    for b, other, k in shared:
        table[b][:k] = table[other][:k]
    refs = [0] * pages
    for row in table:
        for p in row:
            if 0 <= p < pages:
                refs[p] += 1
    return table, refs
