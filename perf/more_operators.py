"""Measurable cases of serving many continuations of one prefix from the 16-bit latent cache.

One case is one call through ``nanovllm_amd.prefix_sharing``: attention of a
batch whose requests share a prefix's pages, the norms and rotation that make
new rows of the cache and the queries beside them, and the pages' own
bookkeeping (requests that branch off others with copies of the pages they
write to, and a cache brought together at its low pages).  Sizes come from
this repository's configurations and tests (128-token pages, 512 + 64 dims, 4
to 64 heads, one or four rows a request, up to 64 requests, prompts to 64K
tokens); ``draw`` gives more of the same ranges.

With ``own`` false, ``run`` computes each operator in elementary torch
operations in 32 bits; ``exact`` computes the definitions in 64 bits, request
by request.
"""

from __future__ import annotations

import functools
import math
import random
import sys
from pathlib import Path

import torch

own = False

PAGE, LATENT, ROPE = 128, 512, 64
ROW = LATENT + ROPE
SOFTMAX_SCALE = 1.0 / math.sqrt(ROW)
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


@functools.cache
def _framework():
    path = str(Path(__file__).resolve().parents[1] / "nanovllm-dsa-offload_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from nanovllm_amd import prefix_sharing

    return prefix_sharing


# ----------------------------------------------------------------- the cases
def _case(name: str | None, fields: dict) -> dict:
    return fields if name is None else {"name": name, **fields}


def _attend(name: str | None = None, **fields) -> dict:
    """``groups`` groups of requests that share a prefix of prefix_lo to
    prefix_hi tokens, ``loose`` requests without one, own_lo to own_hi tokens
    of their own each."""
    return _case(name, {"kind": "attend", "batch": 1, "groups": 1, "loose": 0, "rows": 1, "prefix_lo": 1, "prefix_hi": 1,
                        "own_lo": 1, "own_hi": 1, "heads": 64, "dtype": "bf16", **fields})


def _norm(name: str | None = None, **fields) -> dict:
    """Rows rows_lo to rows_hi of each request behind up to past_hi tokens;
    ``nope`` > 0: queries of nope + 64 dims are normalised per head too."""
    return _case(name, {"kind": "norm", "batch": 1, "rows_lo": 1, "rows_hi": 1, "past_hi": 0, "heads": 64, "nope": 0,
                        "dtype": "bf16", **fields})


def _branch(name: str | None = None, **fields) -> dict:
    """Every request continues a random one of ``parents`` requests, and gets
    room for ``new`` tokens."""
    return _case(name, {"kind": "branch", "batch": 1, "parents": 1, "lo": 1, "hi": 1, "new": 1, "pages": 64, "cols": 8,
                        "dtype": "bf16", **fields})


def _compact(name: str | None = None, **fields) -> dict:
    """A cache of ``pages`` of which requests of lo to hi tokens hold some."""
    return _case(name, {"kind": "compact", "batch": 1, "lo": 1, "hi": 1, "pages": 64, "dtype": "bf16", **fields})


def listed() -> list[dict]:
    return [
        # Two answers to one short prompt, one rank's heads: all latency.
        _attend("attend_b2_short", batch=2, prefix_lo=389, prefix_hi=389, own_lo=20, own_hi=37, heads=16),
        # Three system prompts, ragged questions behind them, one rank's heads, fp16.
        _attend("attend_b24_groups3_f16", batch=24, groups=3, prefix_lo=2049, prefix_hi=6007, own_lo=1, own_hi=901, heads=8,
                dtype="f16"),
        # Parallel sampling from one long prompt.
        _attend("attend_b32_16k", batch=32, prefix_lo=16384, prefix_hi=16384, own_lo=1, own_hi=513),
        # Speculative verify in two groups, and requests that share nothing.
        _attend("attend_mtp_b16", batch=16, groups=2, loose=3, rows=4, prefix_lo=8192, prefix_hi=12301, own_lo=130,
                own_hi=2050, heads=16),
        # A full batch over four documents of 32K.
        _attend("attend_b64_32k", batch=64, groups=4, prefix_lo=32768, prefix_hi=32768, own_lo=64, own_hi=1030),
        # One new token for each request of a full batch: keys into the cache, queries rotated.
        _norm("norm_decode_b64", batch=64, past_hi=32767),
        # A long prompt and the rest of a batch in chunks, queries normalised per head before their up-projection.
        _norm("norm_prompts_b6_f16", batch=6, rows_lo=301, rows_hi=4100, past_hi=4097, heads=16, nope=192, dtype="f16"),
        # One prompt, every head's rotation.
        _norm("norm_prompt_8k", rows_lo=8190, rows_hi=8190),
        # Eight beams that continue three of them.
        _branch("branch_b8", batch=8, parents=3, lo=900, hi=900, pages=200, cols=16),
        # A full batch whose requests split up: long histories, a large pool, room for verify rows.
        _branch("branch_b64_f16", batch=64, parents=24, lo=5000, hi=32700, new=4, pages=9001, cols=512, dtype="f16"),
        # A small cache after a few requests ended.
        _compact("compact_b8", batch=8, lo=300, hi=2100, pages=301),
        # A large cache brought together after most requests ended.
        _compact("compact_b48_8k", batch=48, lo=4000, hi=8320, pages=6007),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(("attend", "attend", "attend", "norm", "branch", "compact"))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    if kind == "norm":
        rows, nope, heads = rng.choice((1, 1, 4, _log(rng, 5, 8192))), rng.choice((0, 0, 64, 128, 192)), rng.choice((4, 8, 16, 64))
        batch = _log(rng, 1, max(1, min(64, 8192 * 64 // (rows * heads * (1 + nope // 32)))))
        return _norm(batch=batch, rows_lo=max(1, rows // 3), rows_hi=rows, past_hi=_log(rng, 1, 16384), heads=heads, nope=nope,
                     dtype=dtype)
    if kind == "branch":
        batch, hi = _log(rng, 1, 64), _log(rng, 100, 32000)
        cols, new = hi // PAGE + rng.choice((2, 5, 40)), rng.choice((1, 1, 4, 100))
        parents = rng.randrange(1, batch + 1)
        return _branch(batch=batch, parents=parents, lo=max(1, hi // 3), hi=hi, new=new,
                       pages=batch * 2 + parents * (hi // PAGE + 2) + _log(rng, 1, 3000), cols=cols, dtype=dtype)
    if kind == "compact":
        batch, hi = _log(rng, 1, 48), _log(rng, 100, 16000)
        hi = min(hi, 400_000 // batch)
        held = batch * -(-hi // PAGE)
        return _compact(batch=batch, lo=max(1, hi // 2), hi=hi, pages=held + rng.randrange(1, 1 + held), dtype=dtype)
    heads, rows = rng.choice((4, 8, 16, 32, 64)), rng.choice((1, 1, 1, 2, 4))
    prefix = _log(rng, 100, 32768)
    batch = _log(rng, 2, max(2, min(64, 2_000_000 * 64 // (prefix * heads * rows))))
    groups = rng.randrange(1, 1 + max(1, batch // 3))
    most = max(rows, _log(rng, 1, 2000))
    return _attend(batch=batch, groups=groups, loose=rng.choice((0, 0, 1)) if batch > groups else 0, rows=rows,
                   prefix_lo=max(1, int(prefix * rng.uniform(0.3, 1.0))), prefix_hi=prefix, own_lo=max(1, most // 4),
                   own_hi=most, heads=heads, dtype=dtype)


def _spread(lo: int, hi: int, count: int) -> list[int]:
    """``count`` sizes over [lo, hi], the largest first, the others in mixed order."""
    if count == 1:
        return [hi]
    step = next(s for s in (7, 5, 11, 13) if count % s)
    return [hi - (hi - lo) * ((i * step) % count) // (count - 1) for i in range(count)]


def _groups(case: dict) -> list[tuple[int, int, int]]:
    """(first request, end, prefix tokens) of every group."""
    count, inside = case["groups"], case["batch"] - case["loose"]
    at = [inside * i // count for i in range(count + 1)]
    return [(at[i], at[i + 1], p) for i, p in enumerate(_spread(case["prefix_lo"], case["prefix_hi"], count))]


def _sizes(case: dict) -> tuple[list[int], list[int]]:
    """(tokens, rows) of an attention case's requests."""
    own_tokens = _spread(case["own_lo"], case["own_hi"], case["batch"])
    prefix = [0] * case["batch"]
    for first, end, tokens in _groups(case):
        prefix[first:end] = [tokens] * (end - first)
    lengths = [p + o for p, o in zip(prefix, own_tokens)]
    return lengths, [min(case["rows"], n) for n in lengths]


# -------------------------------------------------------------- the inputs
def _rng(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g: torch.Generator, *shape) -> torch.Tensor:
    return torch.randn(*shape, generator=g, device="cuda")


def _ints(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32).cuda()


def _caches(g: torch.Generator, pages: int, dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """(kv_cache, k_rope) of that many pages, about unit size."""
    kv, rope = (torch.empty(pages, PAGE, 1, d, dtype=dtype, device="cuda") for d in (LATENT, ROPE))
    for cache in (kv, rope):
        for at in range(0, pages, 1024):
            part = cache[at:at + 1024]
            part.copy_(torch.randn(part.shape, generator=g, device="cuda", dtype=torch.float16))
    return kv, rope


def _table(g: torch.Generator, held: list[list[int]], pages: int, cols: int, none: int) -> tuple[torch.Tensor, torch.Tensor]:
    """The requests' page tables where request b holds the pages numbered
    held[b], at shuffled places of the cache, and how many hold each place."""
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    counts = torch.tensor([len(h) for h in held]).cuda()
    flat = torch.tensor([p for h in held for p in h]).cuda()
    inside = torch.arange(cols, device="cuda") < counts[:, None]
    table = torch.full((len(held), cols), none, dtype=torch.int32, device="cuda")
    table[inside] = order[flat]
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs.index_add_(0, order[flat], torch.ones(flat.shape[0], dtype=torch.int32, device="cuda"))
    return table, refs


def prepare(case: dict, seed: int) -> dict:
    g = _rng(seed)
    s = {"kind": case["kind"]}
    return {"attend": _prepare_attend, "norm": _prepare_norm, "branch": _prepare_branch,
            "compact": _prepare_compact}[case["kind"]](case, g, s)


def _prepare_attend(case: dict, g: torch.Generator, s: dict) -> dict:
    lengths, counts = _sizes(case)
    dtype, heads, total = DTYPES[case["dtype"]], case["heads"], sum(counts)
    held, next_page = [[] for _ in lengths], 0
    for first, end, tokens in _groups(case):
        shared = list(range(next_page, next_page + tokens // PAGE))
        next_page += len(shared)
        for b in range(first, end):
            held[b] = list(shared)
    for b, n in enumerate(lengths):
        more = -(-n // PAGE) - len(held[b])
        held[b] += range(next_page, next_page + more)
        next_page += more
    pages = next_page + 3
    s["table"], _ = _table(g, held, pages, max(len(h) for h in held), 0)
    s["kv_cache"], s["k_rope"] = _caches(g, pages, dtype)
    s["lengths"], s["ends"] = _ints(lengths), _ints(counts).cumsum(0).to(torch.int32)
    s["group_ends"] = _ints([end for _, end, _ in _groups(case)])
    s["group_tokens"] = _ints([tokens for _, _, tokens in _groups(case)])
    s["longest"], s["rows_most"] = max(lengths), max(counts)
    s["query"] = (2.0 * _randn(g, total, heads, LATENT)).to(dtype)
    s["query_rope"] = (2.0 * _randn(g, total, heads, ROPE)).to(dtype)
    s["out"] = torch.empty(total, heads, LATENT, dtype=dtype, device="cuda")
    return s


def _prepare_norm(case: dict, g: torch.Generator, s: dict) -> dict:
    rows = _spread(case["rows_lo"], case["rows_hi"], case["batch"])
    past = _spread(0, case["past_hi"], case["batch"])[::-1]
    lengths, total, dtype = [r + p for r, p in zip(rows, past)], sum(rows), DTYPES[case["dtype"]]
    counts = [-(-n // PAGE) for n in lengths]
    starts = [sum(counts[:b]) for b in range(len(counts))]
    pages = sum(counts) + 2
    s["table"], _ = _table(g, [list(range(a, a + c)) for a, c in zip(starts, counts)], pages, max(counts), 0)
    s["kv_cache"], s["k_rope"] = _caches(g, pages, dtype)
    s["lengths"], s["ends"] = _ints(lengths), _ints(rows).cumsum(0).to(torch.int32)
    # Rows of a projection: a size of their own each, a few dims above the rest.
    size = torch.exp2(2.0 * torch.rand(total, 1, generator=g, device="cuda") - 1.0)
    s["kv"] = (size * _randn(g, total, ROW)).to(dtype)
    s["query"] = (size[..., None] * _randn(g, total, case["heads"], case["nope"] + ROPE)).to(dtype)
    s["kv_weight"] = (1.0 + 0.2 * _randn(g, LATENT)).to(dtype)
    # Angles of positions to 64K, in 64 bits; the tables in the model's type, a pair's value twice.
    position = torch.cat([torch.arange(p, p + r) for p, r in zip(past, rows)]).cuda().double()
    inverse = 1e6 ** (-torch.arange(0, ROPE, 2, device="cuda").double() / ROPE)
    angle = (position[:, None] * inverse).repeat_interleave(2, 1)
    s["cos"], s["sin"] = angle.cos().to(dtype), angle.sin().to(dtype)
    s["query_rope"] = torch.empty(total, case["heads"], ROPE, dtype=dtype, device="cuda")
    s["query_weight"] = s["query_nope"] = None
    if case["nope"]:
        s["query_weight"] = (1.0 + 0.2 * _randn(g, case["nope"] + ROPE)).to(dtype)
        s["query_nope"] = torch.empty(total, case["heads"], case["nope"], dtype=dtype, device="cuda")
    return s


def _prepare_branch(case: dict, g: torch.Generator, s: dict) -> dict:
    batch, order = case["batch"], random.Random(int(torch.randint(0, 1 << 30, (1,), generator=g, device="cuda")))
    lengths = _spread(case["lo"], case["hi"], case["parents"]) + [0] * (batch - case["parents"])
    places = list(range(batch))
    order.shuffle(places)  # the requests that go on, at any rows of the batch
    lengths = [lengths[p] for p in places]
    alive = [b for b, n in enumerate(lengths) if n > 0]
    parents = [order.choice(alive) if n == 0 or order.random() < 0.7 else b for b, n in enumerate(lengths)]
    counts = [-(-n // PAGE) for n in lengths]
    starts = [sum(counts[:b]) for b in range(batch)]
    held = [list(range(a, a + c)) for a, c in zip(starts, counts)]
    table, refs = _table(g, held, case["pages"], case["cols"], -1)
    s["records"] = torch.cat([_ints(lengths), refs, table.flatten()])  # before the call, which changes them
    s["live"] = s["records"].clone()
    s["lengths"], s["refs"] = s["live"][:batch], s["live"][batch:batch + case["pages"]]
    s["table"] = s["live"][batch + case["pages"]:].view(batch, case["cols"])
    s["parents"], s["new"] = _ints(parents), _ints([case["new"]] * batch)
    s["copy_src"], s["copy_dst"], s["copy_tokens"] = (torch.empty(batch, dtype=torch.int32, device="cuda") for _ in range(3))
    s["missing"] = torch.empty(1, dtype=torch.int32, device="cuda")
    s["kv_cache"], s["k_rope"] = _caches(g, case["pages"], DTYPES[case["dtype"]])
    return s


def _prepare_compact(case: dict, g: torch.Generator, s: dict) -> dict:
    counts = [-(-n // PAGE) for n in _spread(case["lo"], case["hi"], case["batch"])]
    starts = [sum(counts[:b]) for b in range(len(counts))]
    held = [list(range(a, a + c)) for a, c in zip(starts, counts)]
    held[-1][0] = held[0][0]  # one page of two requests, and a place that nobody holds
    table, refs = _table(g, held, case["pages"], max(counts), -1)
    s["records"] = torch.cat([refs, table.flatten()])
    s["live"] = s["records"].clone()
    s["refs"], s["table"] = s["live"][:case["pages"]], s["live"][case["pages"]:].view(table.shape)
    s["move_src"], s["move_dst"] = (torch.full((case["pages"],), -1, dtype=torch.int32, device="cuda") for _ in range(2))
    s["move_count"] = torch.empty(1, dtype=torch.int32, device="cuda")
    s["kv_cache"], s["k_rope"] = _caches(g, case["pages"], DTYPES[case["dtype"]])
    return s


# ---------------------------------------------------------------- one pass
def run(s: dict):
    return {"attend": _run_attend, "norm": _run_norm, "branch": _run_branch, "compact": _run_compact}[s["kind"]](s)


def _run_attend(s: dict):
    if own:
        _framework().shared_prefix_attention(s["query_rope"], s["query"], s["ends"], s["lengths"], s["table"], s["k_rope"],
                                             s["kv_cache"], SOFTMAX_SCALE, s["out"], prefix_request_ends=s["group_ends"],
                                             prefix_lengths=s["group_tokens"])
    else:
        _plain_attend(s)
    return s["out"]


def _run_norm(s: dict):
    if own:
        _framework().norm_rope_append(s["query"], s["kv"], s["cos"], s["sin"], s["kv_weight"], s["ends"], s["lengths"],
                                      s["table"], s["k_rope"], s["kv_cache"], s["query_rope"],
                                      query_norm_weight=s["query_weight"], query_nope=s["query_nope"], eps=EPS)
    else:
        _plain_norm(s)
    out = {"query_rope": s["query_rope"], "kv_cache": s["kv_cache"], "k_rope": s["k_rope"]}
    return out if s["query_nope"] is None else out | {"query_nope": s["query_nope"]}


def _run_branch(s: dict):
    s["live"].copy_(s["records"])  # the tables before a step
    if own:
        api = _framework()
        api.pages_branch(s["lengths"], s["new"], s["table"], s["refs"], s["copy_src"], s["copy_dst"], s["copy_tokens"],
                         s["missing"], parents=s["parents"])
        api.pages_copy(s["copy_src"], s["copy_dst"], [s["kv_cache"], s["k_rope"]], tokens=s["copy_tokens"])
    else:
        _plain_branch(s)
        _plain_copy(s, s["copy_src"], s["copy_dst"], s["copy_tokens"])
    return {k: s[k] for k in ("lengths", "table", "refs", "copy_src", "copy_dst", "copy_tokens", "missing", "kv_cache",
                              "k_rope")}


def _run_compact(s: dict):
    s["live"].copy_(s["records"])
    if own:
        api = _framework()
        api.pages_compact(s["table"], s["refs"], s["move_src"], s["move_dst"], s["move_count"])
        api.pages_copy(s["move_src"], s["move_dst"], [s["kv_cache"], s["k_rope"]], count=s["move_count"])
    else:
        _plain_compact(s)
        listed_ = torch.arange(s["move_src"].shape[0], device="cuda") < s["move_count"]
        _plain_copy(s, s["move_src"], s["move_dst"], torch.where(listed_, PAGE, 0))
    return {k: s[k] for k in ("table", "refs", "move_src", "move_dst", "move_count", "kv_cache", "k_rope")}


# ------------------------------------------------------------- plain forms
def _plain_attend(s: dict) -> None:
    """Every request over all of its pages, padded to the longest."""
    batch, most, heads = s["lengths"].shape[0], s["rows_most"], s["query"].shape[1]
    ends, lengths = s["ends"].long(), s["lengths"].long()
    counts = torch.diff(ends, prepend=ends.new_zeros(1))
    turn = torch.arange(most, device="cuda")
    row = ((ends - counts)[:, None] + turn).clamp(max=s["query"].shape[0] - 1)
    slots = torch.arange(s["longest"], device="cuda")
    page = s["table"][:, slots // PAGE].long()
    kv = torch.cat([s["kv_cache"][page, slots % PAGE, 0], s["k_rope"][page, slots % PAGE, 0]], -1).float()
    q = torch.cat([s["query"], s["query_rope"]], -1).float()[row].view(batch, most * heads, ROW)
    visible = lengths[:, None] - (counts[:, None] - 1 - turn)
    seen = (slots < visible[..., None])[:, :, None].expand(-1, -1, heads, -1).reshape(batch, most * heads, -1)
    scores = torch.matmul(q, kv.transpose(1, 2).contiguous()) * SOFTMAX_SCALE
    scores = torch.where(seen, scores, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = torch.matmul(p, kv[..., :LATENT].contiguous()) / p.sum(-1, keepdim=True)
    real = turn < counts[:, None]
    s["out"][row[real]] = out.view(batch, most, heads, LATENT)[real].to(s["out"].dtype)


def _rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """Pairs (x0, x1) to (x0 cos - x1 sin, x1 cos + x0 sin)."""
    turned = torch.stack([-x[..., 1::2], x[..., 0::2]], -1).flatten(-2)
    return x * cos + turned * sin


def _rms(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight


def _plain_norm(s: dict) -> None:
    ends, lengths = s["ends"].long(), s["lengths"].long()
    t = torch.arange(s["kv"].shape[0], device="cuda")
    request = torch.searchsorted(ends, t, right=True)
    slot = lengths[request] - ends[request] + t
    page = s["table"][request, slot // PAGE].long()
    cos, sin, kv, query = (s[k].float() for k in ("cos", "sin", "kv", "query"))
    s["kv_cache"][page, slot % PAGE, 0] = _rms(kv[:, :LATENT], s["kv_weight"].float()).to(s["kv_cache"].dtype)
    s["k_rope"][page, slot % PAGE, 0] = _rotate(kv[:, LATENT:], cos, sin).to(s["k_rope"].dtype)
    if s["query_nope"] is not None:
        query = _rms(query, s["query_weight"].float())
        s["query_nope"].copy_(query[..., :-ROPE])
    s["query_rope"].copy_(_rotate(query[..., -ROPE:], cos[:, None], sin[:, None]))


def _plain_branch(s: dict) -> None:
    table, refs, parents = s["table"], s["refs"], s["parents"].long()
    batch, cols = table.shape
    rows, col = torch.arange(batch, device="cuda")[:, None], torch.arange(cols, device="cuda")
    one = torch.ones((), dtype=torch.int32, device="cuda")
    # Rows take over what their parents held; pages count their holders anew.
    before, after = table.clone(), table[parents]
    for held, sign in ((after, one), (before, -one)):
        refs.index_add_(0, held.clamp(min=0).flatten(), torch.where(held >= 0, sign, 0).to(torch.int32).flatten())
    lengths = s["lengths"].long()[parents]
    # Columns that the new tokens fall into: a page is kept by a row that holds it
    # alone, or by the lowest of the rows that all write to it.
    first, last = lengths // PAGE, (lengths + s["new"] - 1) // PAGE
    written = (col >= first[:, None]) & (col <= last[:, None]) & (s["new"] > 0)[:, None]
    named, at = after >= 0, after.clamp(min=0).long()
    part = written & named & (col == first[:, None]) & (lengths % PAGE > 0)[:, None]
    writers = torch.zeros_like(refs).index_add_(0, at.flatten(), part.to(torch.int32).flatten())
    lowest = torch.full_like(refs, batch).scatter_reduce_(
        0, at.flatten(), torch.where(part, rows, batch).to(torch.int32).flatten(), "amin")
    kept = named & ((refs[at] <= 1) | (part & (refs[at] == writers[at]) & (lowest[at] == rows)))
    takes = written & ~kept
    free = torch.where(refs == 0, torch.arange(refs.shape[0], device="cuda"), refs.shape[0]).sort().values
    lack = (takes.sum() - (refs == 0).sum()).clamp(min=0)
    takes = takes & (lack == 0)
    nth = takes.flatten().cumsum(0).view(batch, cols) - 1
    fresh = free[nth.clamp(0, refs.shape[0] - 1)].to(torch.int32)
    result = torch.where(takes, fresh, after)
    refs.index_add_(0, at.flatten(), torch.where(takes & named, -one, 0).to(torch.int32).flatten())
    refs.index_add_(0, result.clamp(min=0).flatten(), takes.to(torch.int32).flatten())
    copies = takes & part
    for name, values in (("copy_src", after), ("copy_dst", result)):
        s[name].copy_(torch.where(copies, values, -1).amax(1))
    s["copy_tokens"].copy_(torch.where(copies, (lengths % PAGE)[:, None], 0).amax(1))
    table.copy_(result)
    s["lengths"].copy_(lengths)
    s["missing"].copy_(lack)


def _plain_copy(s: dict, src: torch.Tensor, dst: torch.Tensor, tokens: torch.Tensor) -> None:
    """The first tokens[k] rows of page src[k] to page dst[k]."""
    k, row = (torch.arange(PAGE, device="cuda") < tokens[:, None]).nonzero(as_tuple=True)
    for cache in (s["kv_cache"], s["k_rope"]):
        cache[dst[k].long(), row] = cache[src[k].long(), row]


def _plain_compact(s: dict) -> None:
    refs, table, pages = s["refs"], s["table"], torch.arange(s["refs"].shape[0], device="cuda")
    live = refs > 0
    count = live.sum()
    src, dst = (live & (pages >= count)).nonzero()[:, 0], (~live & (pages < count)).nonzero()[:, 0]
    s["move_src"][:src.shape[0]], s["move_dst"][:dst.shape[0]] = src.to(torch.int32), dst.to(torch.int32)
    s["move_count"].fill_(src.shape[0])
    place = pages.scatter(0, src, dst)
    table.copy_(torch.where(table >= 0, place[table.clamp(min=0).long()], -1))
    refs[dst] = refs[src]
    refs[src] = 0


# --------------------------------------------------------- work and 64 bits
def work(case: dict) -> dict:
    if case["kind"] == "attend":
        lengths, counts = _sizes(case)
        heads, rows = case["heads"], sum(counts)
        once = sum((end - first - 1) * (tokens // PAGE * PAGE) for first, end, tokens in _groups(case))
        pairs = heads * sum(c * n - c * (c - 1) // 2 for n, c in zip(lengths, counts))
        return {"bytes": 2 * ROW * (sum(lengths) - once) + 2 * rows * heads * (ROW + LATENT),
                "flops": 2 * pairs * (ROW + LATENT)}
    if case["kind"] == "norm":
        rows, dims = sum(_spread(case["rows_lo"], case["rows_hi"], case["batch"])), case["nope"] + ROPE
        return {"bytes": 4 * rows * (ROW + case["heads"] * dims + ROPE), "flops": 6 * rows * (ROW + case["heads"] * dims)}
    token = 2 * ROW
    if case["kind"] == "branch":
        # About one copy of half a page for a request that shares its last page.
        held = sum(-(-n // PAGE) for n in _spread(case["lo"], case["hi"], case["parents"]))
        copies = max(1, case["batch"] - case["parents"])
        return {"bytes": copies * (PAGE // 2) * token * 2 + 4 * (case["pages"] + 2 * held), "flops": case["pages"]}
    held = sum(-(-n // PAGE) for n in _spread(case["lo"], case["hi"], case["batch"])) - 1
    moved = held * (case["pages"] - held) // case["pages"]
    return {"bytes": moved * PAGE * token * 2 + 8 * held + 4 * case["pages"], "flops": case["pages"]}


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "norm": _exact_norm, "branch": _exact_branch, "compact": _exact_compact}[case["kind"]](s)


def _exact_attend(s: dict):
    heads = s["query"].shape[1]
    q = torch.cat([s["query"], s["query_rope"]], -1).double()
    out = torch.zeros(q.shape[0], heads, LATENT, dtype=torch.float64, device="cuda")
    start = 0
    for b, (end, length) in enumerate(zip(s["ends"].tolist(), s["lengths"].tolist())):
        pages = s["table"][b, : -(-length // PAGE)].long()
        kv = torch.cat([s["kv_cache"][pages].flatten(0, 2), s["k_rope"][pages].flatten(0, 2)], -1)[:length].double()
        for r in range(start, end):
            seen = kv[:length - (end - 1 - r)]
            p = torch.softmax(torch.matmul(q[r], seen.T.contiguous()) * SOFTMAX_SCALE, -1)
            out[r] = torch.matmul(p, seen[:, :LATENT].contiguous())
        start = end
    return out


def _exact_rotation(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    z = torch.view_as_complex(x.unflatten(-1, (-1, 2)).contiguous())
    return torch.view_as_real(z * torch.complex(cos[..., ::2].contiguous(), sin[..., ::2].contiguous())).flatten(-2)


def _exact_norm(s: dict):
    kv, query, cos, sin = (s[k].double() for k in ("kv", "query", "cos", "sin"))
    cache, rope = s["kv_cache"].double(), s["k_rope"].double()
    latent, start = kv[:, :LATENT], 0
    latent = latent / (latent.norm(dim=-1, keepdim=True).square() / LATENT + EPS).sqrt() * s["kv_weight"].double()
    turned = _exact_rotation(kv[:, LATENT:], cos, sin)
    for b, (end, length) in enumerate(zip(s["ends"].tolist(), s["lengths"].tolist())):
        at, slot = start, length - (end - start)
        while at < end:  # page by page
            n = min(end - at, PAGE - slot % PAGE)
            page = int(s["table"][b, slot // PAGE])
            cache[page, slot % PAGE:slot % PAGE + n, 0] = latent[at:at + n]
            rope[page, slot % PAGE:slot % PAGE + n, 0] = turned[at:at + n]
            at, slot = at + n, slot + n
        start = end
    out = {"kv_cache": cache, "k_rope": rope}
    if s["query_weight"] is not None:
        mean = query.norm(dim=-1, keepdim=True).square() / query.shape[-1]
        query = query / (mean + EPS).sqrt() * s["query_weight"].double()
        out["query_nope"] = query[..., :-ROPE]
    return out | {"query_rope": _exact_rotation(query[..., -ROPE:], cos[:, None], sin[:, None])}


def _exact_branch(s: dict):
    cache, rope = s["kv_cache"].double(), s["k_rope"].double()
    refs, old = s["refs"].tolist(), s["table"].tolist()
    lengths, parents, new = (s[k].tolist() for k in ("lengths", "parents", "new"))
    tables, lengths = [list(old[p]) for p in parents], [lengths[p] for p in parents]
    for row, sign in [(r, 1) for r in tables] + [(r, -1) for r in old]:
        for page in row:
            if page >= 0:
                refs[page] += sign
    wanted = []  # (request, column, whether rows of an older page go along)
    for b, (row, length, n) in enumerate(zip(tables, lengths, new)):
        for c in range(length // PAGE, (length + n - 1) // PAGE + 1):
            page = row[c]
            if page < 0:
                wanted.append((b, c, False))
                continue
            part = c == length // PAGE and length % PAGE > 0
            sharers = [o for o in range(len(tables)) if new[o] > 0 and lengths[o] % PAGE > 0 and
                       tables[o][lengths[o] // PAGE] == page]
            if refs[page] > 1 and not (part and refs[page] == len(sharers) and b == sharers[0]):
                wanted.append((b, c, part))
    free = [p for p, r in enumerate(refs) if r == 0]
    if len(wanted) <= len(free):
        for (b, c, part), page in zip(wanted, free):
            if part:
                cache[page, :lengths[b] % PAGE] = cache[tables[b][c], :lengths[b] % PAGE]
                rope[page, :lengths[b] % PAGE] = rope[tables[b][c], :lengths[b] % PAGE]
    whole = ("lengths", "table", "refs", "copy_src", "copy_dst", "copy_tokens", "missing")
    return {k: None for k in whole} | {"kv_cache": cache, "k_rope": rope}


def _exact_compact(s: dict):
    cache, rope = s["kv_cache"].double(), s["k_rope"].double()
    live = [p for p, r in enumerate(s["refs"].tolist()) if r > 0]
    holes = sorted(set(range(len(live))) - set(live))
    for src, dst in zip([p for p in live if p >= len(live)], holes):
        cache[dst], rope[dst] = cache[src], rope[src]
    whole = ("table", "refs", "move_src", "move_dst", "move_count")
    return {k: None for k in whole} | {"kv_cache": cache, "k_rope": rope}
