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


def make_cache(prefixes, groups, own, seed, dtype, cols=None, spare=2, none=-1, size=1.0):
    """Caches, table and lengths of requests in groups: ``groups[s]`` requests
    share a prefix of ``prefixes[s]`` tokens (their whole pages), request b has
    ``own[b]`` more; requests behind the groups share nothing."""
    g = torch.Generator().manual_seed(seed)
    table, at, lengths = [], 0, []
    for n, tokens in zip(groups, prefixes):
        shared = list(range(at, at + tokens // PAGE))
        at += len(shared)
        for _ in range(n):
            lengths.append(tokens + own[len(lengths)])
            more = -(-lengths[-1] // PAGE) - len(shared)
            table.append(shared + list(range(at, at + max(0, more))))
            at += max(0, more)
    while len(lengths) < len(own):
        lengths.append(own[len(lengths)])
        more = -(-lengths[-1] // PAGE)
        table.append(list(range(at, at + more)))
        at += more
    blocks = at + spare
    order = torch.randperm(blocks, generator=g).tolist()
    cols = cols or max(1, max(len(r) for r in table))
    table = [[order[p] for p in r] + [none] * (cols - len(r)) for r in table]
    rand = lambda *s: (size * torch.randn(*s, generator=g)).to(dtype)  # noqa: E731
    return {"table": i32(table), "lengths": i32(lengths), "kv_cache": rand(blocks, PAGE, 1, 512),
            "k_rope": rand(blocks, PAGE, 1, 64), "group_ends": i32(list(torch.tensor(groups).cumsum(0))) if groups else i32([]),
            "prefix": i32(list(prefixes))}


def make_queries(c, counts, heads, seed, pad=0, size=2.0):
    g = torch.Generator().manual_seed(seed + 1000)
    total, dtype = sum(counts) + pad, c["kv_cache"].dtype
    c["query"] = (size * torch.randn(total, heads, 512, generator=g)).to(dtype)
    c["query_rope"] = (size * torch.randn(total, heads, 64, generator=g)).to(dtype)
    c["ends"] = torch.tensor(counts).cumsum(0).to(torch.int32)
    c["out"] = torch.full((total, heads, 512), 7.0).to(dtype)
    return c


def call_attention(d, scale=SCALE, groups=True):
    more = {"prefix_request_ends": d["group_ends"], "prefix_lengths": d["prefix"]} if groups else {}
    api().shared_prefix_attention(d["query_rope"], d["query"], d["ends"], d["lengths"], d["table"], d["k_rope"],
                                  d["kv_cache"], scale, d["out"], **more)


def attention_bound(c, out, size, reach):
    """How far an output may be from the 64-bit one.  The store rounds by half a
    step; so does P, each by half a step of its own (16 bits); sums of n terms
    in fp32 are off by n 2^-24 of their magnitudes, those of P and the output's
    each, and the join adds as many parts at most; a score of 576 products in
    fp32 is off by at most 578 2^-24 of |q| . |k|, with its factor 2^-22 of
    itself, and moves p and its normaliser by that each; the exponential is off
    by 2^-22 of itself.  fp16 holds P below its normal range to 2^-25, and a
    row's largest P is at least 2^8: 2^-33 of the largest |v| a key."""
    dtype = c["kv_cache"].dtype
    keys = int(c["lengths"].max())
    score = reach * (578 * 2.0 ** -24 + 2.0 ** -22)
    per = HALF_STEP[dtype] + keys * 2.0 ** -22 + 2 * score + 2.0 ** -20
    tail = keys * 2.0 ** -33 * float(torch.nan_to_num(c["kv_cache"].float(), 0, 0, 0).abs().max()) if dtype == torch.float16 else 0.0
    return out.abs() * HALF_STEP[dtype] + size * per[..., None] + tail + TINY[dtype]


def check_attention(got, c, scale=SCALE):
    out, size, reach = O.attention(c["query_rope"], c["query"], c["ends"], c["lengths"], c["table"], c["k_rope"],
                                   c["kv_cache"], scale)
    last = min(max(int(c["ends"][-1]), 0), out.shape[0])
    off = (got.double() - out).abs()[:last]
    worst = float((off / attention_bound(c, out, size, reach)[:last]).max()) if last else 0.0
    assert worst <= 1.0, worst
    assert torch.equal(got[last:].view(torch.int16), c["out"][last:].view(torch.int16))
    return worst


def shared_units(c, counts, heads):
    """What the call's groups save, in the half tiles that decide whether their
    prefixes are read once (2 for a tile of up to 32 pairs, 3 up to 64, 4 for 128)."""
    time = lambda pairs: 2 if pairs <= 32 else 3 if pairs <= 64 else 4 * -(-pairs // 128)  # noqa: E731
    at, saved = 0, 0
    for end, prefix in zip(c["group_ends"].tolist(), c["prefix"].tolist()):
        n, pairs = end - at, sum(counts[at:end]) * heads
        tiles = prefix // PAGE * 4
        less = tiles * (n * time(pairs // n) - time(pairs)) if n > 1 else 0
        if n > 1 and 0 < pairs < n * 128 and less > 16 * time(pairs):
            saved += less
        at = end
    return saved


READ_ONCE = 13 * 256  # half tiles saved from which a call's prefixes are read once
