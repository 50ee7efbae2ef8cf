"""Measurable cases of the 8-bit latent cache's operators: append, attention, eviction.

One case is one call through ``nanovllm_amd.latent_cache`` on a paged latent
KV cache held in e4m3 with one scale per 128-token block and latent head:
quantising new rows into it, attending to it (one row per request, a few, or a
prompt's chunk; over every cached token or over a list), and bringing requests
back under their budget by evicting the tokens that gathered the least
attention weight.  Sizes come from this repository's configurations and tests
(128-token blocks, 512 + 64 dims, 4 to 64 heads, 2048-entry selections, up to
64 requests, prompts to 64K tokens); ``draw`` gives more of the same ranges.

With ``own`` false, ``run`` computes each operator in elementary torch
operations in 32 bits; ``exact`` computes the definitions in 64 bits, request
by request.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

BLOCK, LATENT, ROPE = 128, 512, 64
ROW = LATENT + ROPE
SOFTMAX_SCALE = 1.0 / math.sqrt(ROW)
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _framework():
    path = str(Path(__file__).resolve().parents[1] / "nanovllm-dsa-offload_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from nanovllm_amd import latent_cache

    return latent_cache


# ----------------------------------------------------------------- the cases
def _attend(name: str | None = None, **fields) -> dict:
    case = {"kind": "attend", "batch": 1, "rows": 1, "lo": 1, "hi": 1, "heads": 64, "latent_heads": 1, "list": 0,
            "weights": False, "dtype": "bf16", **fields}
    return case if name is None else {"name": name, **case}


def _append(name: str | None = None, **fields) -> dict:
    case = {"kind": "append", "batch": 1, "rows_lo": 1, "rows_hi": 1, "past_lo": 0, "past_hi": 0, "latent_heads": 1,
            "pool": True, "dtype": "bf16", **fields}
    return case if name is None else {"name": name, **case}


def _evict(name: str | None = None, **fields) -> dict:
    case = {"kind": "evict", "batch": 1, "lo": 1, "hi": 1, "over": 128, "latent_heads": 1, "first": 4, "last": 128,
            **fields}
    return case if name is None else {"name": name, **case}


def listed() -> list[dict]:
    return [
        # One interactive request with a short history, one rank's heads: all latency.
        _attend("attend_b1_short", lo=701, hi=701, heads=16),
        # The benchmark's decode batch: 24 requests of 32K, every token attended.
        _attend("attend_b24_32k", batch=24, lo=32768, hi=32768),
        # A mixed decode batch of one rank's heads under tensor parallelism, ragged odd lengths, fp16.
        _attend("attend_b40_ragged_f16", batch=40, lo=129, hi=40961, heads=8, dtype="f16"),
        # Speculative verify: four query rows per request.
        _attend("attend_mtp_b16", batch=16, rows=4, lo=8192, hi=16387),
        # The indexer's 2048-token selection over a resident history.
        _attend("attend_list_b24", batch=24, lo=20480, hi=65536, list=2048),
        # A prompt's chunk over its prefix, two latent heads.
        _attend("attend_chunk_g2", batch=2, rows=515, lo=4100, hi=8197, heads=32, latent_heads=2),
        # Decode that accumulates each token's attention weight, for the eviction.
        _attend("attend_weights_b24_8k", batch=24, lo=8192, hi=8320, weights=True),
        # One new token for each request of a full batch.
        _append("append_decode_b64", batch=64, past_lo=700, past_hi=32767),
        # A long prompt, and the rest of a batch in chunks: ragged, off the block borders.
        _append("append_prompts_b6_f16", batch=6, rows_lo=301, rows_hi=8200, past_hi=4097, latent_heads=2, dtype="f16"),
        # One request that outgrew its budget by a block.
        _evict("evict_b1_2k", lo=2176, hi=2176),
        # A full batch that outgrew budgets of about 8K by a block.
        _evict("evict_b48_8k", batch=48, lo=8000, hi=8320),
        # After long prompts: 32K of history down to half.
        _evict("evict_b16_32k_half", batch=16, lo=30001, hi=32768, over=15001, first=64, last=512),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(("attend", "attend", "list", "chunk", "weights", "append", "append_long", "evict", "evict"))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    latent_heads = rng.choice((1, 1, 1, 2))
    if kind == "append":
        return _append(batch=_log(rng, 1, 64), rows_hi=rng.choice((1, 1, 2, 4)), past_hi=_log(rng, 1, 32768),
                       latent_heads=latent_heads, pool=rng.random() < 0.5, dtype=dtype)
    if kind == "append_long":
        rows = _log(rng, 33, 8192)
        return _append(batch=_log(rng, 1, max(1, 24000 // rows)), rows_lo=max(1, rows // 3), rows_hi=rows,
                       past_hi=_log(rng, 1, 8192), latent_heads=latent_heads, pool=rng.random() < 0.5, dtype=dtype)
    if kind == "evict":
        hi = _log(rng, 600, 32768)
        return _evict(batch=_log(rng, 1, min(48, 300_000 // hi)), lo=max(500, int(hi * rng.uniform(0.6, 1.0))), hi=hi,
                      over=rng.choice((1, 128, 128, 1 + rng.randrange(400), int(hi * 0.45))), latent_heads=latent_heads,
                      first=rng.choice((0, 4, 64)), last=rng.choice((1, 32, 128)))
    heads = latent_heads * rng.choice((4, 5, 8, 16, 32, 64))
    if kind == "chunk":
        rows = _log(rng, 16, 600)
        hi = _log(rng, rows, 8192)
        heads = min(heads, 32)
        return _attend(batch=_log(rng, 1, max(1, min(4, 150_000_000 // (rows * hi * heads)))), rows=rows,
                       lo=max(1, hi // 2), hi=hi, heads=heads, latent_heads=latent_heads, dtype=dtype)
    if kind == "list":
        return _attend(batch=_log(rng, 1, 32), rows=rng.choice((1, 1, 4)), lo=1024, hi=_log(rng, 2048, 49152),
                       heads=heads, latent_heads=latent_heads, list=rng.choice((512, 1000, 2048, 2048)), dtype=dtype)
    hi = _log(rng, 40, 32768)
    batch = _log(rng, 1, max(1, min(64, 600_000 // (hi * latent_heads))))
    rows = rng.choice((1, 1, 1, 2, 4))
    return _attend(batch=batch, rows=rows, lo=max(1, int(hi * rng.uniform(0.05, 1.0))), hi=hi, heads=heads,
                   latent_heads=latent_heads, weights=kind == "weights", dtype=dtype)


def _spread(lo: int, hi: int, count: int) -> list[int]:
    """``count`` sizes over [lo, hi], the largest first, the others in mixed order."""
    if count == 1:
        return [hi]
    step = next(s for s in (7, 5, 11, 13) if count % s)
    return [hi - (hi - lo) * ((i * step) % count) // (count - 1) for i in range(count)]


def _lengths(case: dict) -> list[int]:
    return _spread(case["lo"], case["hi"], case["batch"])


# -------------------------------------------------------------- the inputs
def _rng(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g: torch.Generator, *shape, dtype=torch.float32) -> torch.Tensor:
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def _ints(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32).cuda()


def _cache(g: torch.Generator, lengths: list[int], latent_heads: int) -> dict:
    """Blocks in shuffled order for requests of these lengths, filled with rows
    of about unit size at scales of 2^-7 and 2^-6, and pool rows for them."""
    batch, cols = len(lengths), -(-max(lengths) // BLOCK)
    counts = [-(-n // BLOCK) for n in lengths]
    blocks = sum(counts) + 3
    order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    first = torch.tensor([0] + counts).cumsum(0)[:-1].cuda()
    col = torch.arange(cols, device="cuda")
    table = order[(first[:, None] + col).clamp(max=blocks - 1)]
    table = torch.where(col < torch.tensor(counts).cuda()[:, None], table, 0).to(torch.int32).contiguous()
    cache = torch.empty(blocks, BLOCK, latent_heads, ROW, dtype=torch.float8_e4m3fn, device="cuda")
    for at in range(0, blocks, 512):
        part = cache[at:at + 512]
        part.copy_((_randn(g, *part.shape, dtype=torch.float16) * 70).clamp(-448, 448))
    scale = torch.exp2(torch.randint(-7, -5, (blocks, latent_heads), generator=g, device="cuda").float())
    entries = torch.randperm(batch + 2, generator=g, device="cuda")[:batch].to(torch.int32)
    return {"table": table, "cache": cache, "scale": scale, "entries": entries, "pool_rows": batch + 2,
            "capacity": cols * BLOCK}


def prepare(case: dict, seed: int) -> dict:
    g = _rng(seed)
    s = {"kind": case["kind"], "latent_heads": case["latent_heads"]}
    if case["kind"] == "append":
        return _prepare_append(case, g, s)
    lengths = _lengths(case)
    s |= _cache(g, lengths, case["latent_heads"])
    s["lengths"], s["longest"] = _ints(lengths), max(lengths)
    shape = (s["pool_rows"], s["capacity"])
    if case["kind"] == "evict":
        # Weights as decode accumulates them: a few heavy tokens, a long tail, and tokens that got none yet.
        weights = torch.exp(2.0 * _randn(g, *shape)) * (torch.rand(shape, generator=g, device="cuda") < 0.97)
        seen = torch.arange(shape[1], device="cuda", dtype=torch.int32).expand(shape)
        s["records"] = torch.stack([weights.view(torch.int32), seen])  # before the eviction, which moves them
        s["live"] = s["records"].clone()
        s["weights"], s["positions"] = s["live"][0].view(torch.float32), s["live"][1]
        s["budgets"] = s["lengths"] - case["over"]
        s["first"], s["last"] = case["first"], case["last"]
        s["move_src"], s["move_dst"] = (torch.full((case["batch"], s["capacity"]), -1, dtype=torch.int32, device="cuda")
                                        for _ in range(2))
        s["move_counts"], s["kept"] = (torch.zeros(case["batch"], dtype=torch.int32, device="cuda") for _ in range(2))
        if own:
            s["api"] = _framework()
        return s
    dtype, batch, heads = DTYPES[case["dtype"]], case["batch"], case["heads"]
    counts = [min(case["rows"], n) for n in lengths]
    total = sum(counts)
    s["rows_most"], s["heads"] = max(counts), heads
    s["ends"] = _ints(counts).cumsum(0).to(torch.int32)
    s["query"] = (2.0 * _randn(g, total, heads, LATENT)).to(dtype)
    s["query_rope"] = (2.0 * _randn(g, total, heads, ROPE)).to(dtype)
    s["out"] = torch.empty(total, heads, LATENT, dtype=dtype, device="cuda")
    s["ids"] = s["weights"] = None
    if case["list"]:
        # Distinct tokens, as a selection gives them, in no order; -1 where a request has fewer.
        seen = s["lengths"].long().repeat_interleave(_ints(counts))
        keys = torch.rand(total, s["capacity"], generator=g, device="cuda")
        keys.masked_fill_(torch.arange(s["capacity"], device="cuda") >= seen[:, None], -1.0)
        top = keys.topk(min(case["list"], s["capacity"]), dim=1)
        ids = torch.where(top.values >= 0, top.indices, -1).to(torch.int32)
        s["ids"] = torch.full((total, case["list"]), -1, dtype=torch.int32, device="cuda")
        s["ids"][:, :ids.shape[1]] = ids
    if case["weights"]:
        s["weights"] = torch.rand(shape, generator=g, device="cuda")
    if own:
        s["api"] = _framework()
    return s


def _prepare_append(case: dict, g: torch.Generator, s: dict) -> dict:
    rows = _spread(case["rows_lo"], case["rows_hi"], case["batch"])
    past = _spread(case["past_lo"], case["past_hi"], case["batch"])[::-1]
    lengths = [r + p for r, p in zip(rows, past)]
    s |= _cache(g, lengths, case["latent_heads"])
    total, dtype = sum(rows), DTYPES[case["dtype"]]
    s["lengths"], s["ends"] = _ints(lengths), _ints(rows).cumsum(0).to(torch.int32)
    size = torch.exp2(torch.rand(total, 1, 1, generator=g, device="cuda") - 0.5)
    s["kv"] = (size * _randn(g, total, case["latent_heads"], LATENT)).to(dtype)
    s["k_rope"] = _randn(g, total, case["latent_heads"], ROPE).to(dtype)
    s["weights"] = s["positions"] = s["row_positions"] = None
    if case["pool"]:
        shape = (s["pool_rows"], s["capacity"])
        s["weights"] = torch.rand(shape, generator=g, device="cuda")
        s["positions"] = torch.zeros(shape, dtype=torch.int32, device="cuda")
        s["row_positions"] = torch.randint(0, 1 << 20, (total,), generator=g, device="cuda", dtype=torch.int32)
    if own:
        s["api"] = _framework()
    return s


# ---------------------------------------------------------------- one pass
def run(s: dict):
    if s["kind"] == "append":
        return _run_append(s)
    if s["kind"] == "evict":
        return _run_evict(s)
    if own:
        s["api"].latent8_attention(s["query_rope"], s["query"], s["ends"], s["lengths"], s["table"], s["cache"],
                                   s["scale"], SOFTMAX_SCALE, s["out"], topk_ids=s["ids"],
                                   req_pool_entries=None if s["weights"] is None else s["entries"],
                                   token_weights=s["weights"])
    elif s["ids"] is None:
        _plain_attention(s)
    else:
        _plain_list_attention(s)
    return {"out": s["out"]} if s["weights"] is None else {"out": s["out"], "weights": s["weights"]}


def _run_append(s: dict):
    if own:
        s["api"].latent8_append(s["kv"], s["k_rope"], s["ends"], s["lengths"], s["table"], s["cache"], s["scale"],
                                positions=s["row_positions"],
                                req_pool_entries=None if s["positions"] is None else s["entries"],
                                token_positions=s["positions"], token_weights=s["weights"])
    else:
        _plain_append(s)
    out = {"cache": s["cache"], "scale": s["scale"]}
    return out if s["positions"] is None else out | {"positions": s["positions"], "weights": s["weights"]}


def _run_evict(s: dict):
    s["live"].copy_(s["records"])  # the records of a request that has grown again
    if own:
        s["api"].latent8_evict(s["lengths"], s["budgets"], s["table"], s["entries"], s["cache"], s["scale"],
                               s["positions"], s["weights"], s["move_src"], s["move_dst"], s["move_counts"], s["kept"],
                               protect_first=s["first"], protect_last=s["last"])
    else:
        _plain_evict(s)
    return {k: s[k] for k in ("cache", "scale", "positions", "weights", "move_src", "move_dst", "move_counts", "kept")}


# ------------------------------------------------------------- plain forms
def _e4m3(x: torch.Tensor) -> torch.Tensor:
    return x.to(torch.float8_e4m3fn)


def _codes(s: dict) -> torch.Tensor:
    return s["cache"].view(torch.uint8)


def _rows_of(s: dict, request: torch.Tensor, slots: torch.Tensor) -> torch.Tensor:
    """Dequantised rows [..., latent_heads, 576] in fp32 of the requests' slots."""
    block = s["table"][request, slots // BLOCK].long()
    rows = _codes(s)[block, slots % BLOCK].view(torch.float8_e4m3fn).float()
    return rows * s["scale"][block][..., None]


def _queries(s: dict) -> torch.Tensor:
    return torch.cat([s["query"], s["query_rope"]], dim=-1).float()


def _softmax(scores: torch.Tensor, seen: torch.Tensor) -> torch.Tensor:
    """Softmax over the last axis of what is seen; rows that see nothing are 0."""
    scores = torch.where(seen, scores, -math.inf)
    most = scores.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(scores - torch.where(seen.any(-1, keepdim=True), most, 0.0)), 0.0)
    return p / torch.where(seen.any(-1, keepdim=True), p.sum(-1, keepdim=True), 1.0)


def _plain_attention(s: dict) -> None:
    g, batch, most = s["latent_heads"], s["lengths"].shape[0], s["rows_most"]
    ends, lengths = s["ends"].long(), s["lengths"].long()
    counts = torch.diff(ends, prepend=ends.new_zeros(1))
    turn = torch.arange(most, device="cuda")
    row = ((ends - counts)[:, None] + turn).clamp(max=s["query"].shape[0] - 1)
    slots = torch.arange(s["longest"], device="cuda")
    kv = _rows_of(s, torch.arange(batch, device="cuda")[:, None], slots[None]).transpose(1, 2).contiguous()
    q = _queries(s)[row]                                                       # [batch, most, heads, 576]
    q = q.view(batch, most, g, -1, ROW).transpose(1, 2).reshape(batch, g, -1, ROW)
    visible = lengths[:, None] - (counts[:, None] - 1 - turn)
    seen = (slots < visible[..., None]) & (turn < counts[:, None])[..., None]  # [batch, most, slots]
    per = s["heads"] // g
    seen_rows = seen[:, None, :, None].expand(-1, -1, -1, per, -1).reshape(batch, 1, most * per, -1)
    p = _softmax(torch.matmul(q, kv.transpose(2, 3)) * SOFTMAX_SCALE, seen_rows)
    out = torch.matmul(p, kv[..., :LATENT]).view(batch, g, most, per, LATENT).transpose(1, 2)
    real = turn < counts[:, None]
    s["out"][row[real]] = out.reshape(batch, most, -1, LATENT)[real].to(s["out"].dtype)
    if s["weights"] is not None:
        s["weights"][s["entries"].long(), :s["longest"]] += p.sum((1, 2))


def _plain_list_attention(s: dict) -> None:
    g, total = s["latent_heads"], s["query"].shape[0]
    ends, lengths = s["ends"].long(), s["lengths"].long()
    t = torch.arange(total, device="cuda")
    request = torch.searchsorted(ends, t, right=True)
    visible = lengths[request] - (ends[request] - 1 - t)
    ids = s["ids"].long()
    seen = (ids >= 0) & (ids < visible[:, None])
    kv = _rows_of(s, request[:, None], torch.where(seen, ids, 0)).transpose(1, 2).contiguous()  # [rows, g, list, 576]
    q = _queries(s).view(total, g, -1, ROW)
    p = _softmax(torch.matmul(q, kv.transpose(2, 3)) * SOFTMAX_SCALE, seen[:, None, None])
    s["out"].copy_(torch.matmul(p, kv[..., :LATENT]).reshape(s["out"].shape))


def _needed_scale(amax: torch.Tensor) -> torch.Tensor:
    """The least power of two s (2^-126 to 2^120) with amax / s <= 448 = 0.875 * 2^9."""
    part, power = torch.frexp(amax)
    power = torch.where(part > 0.875, power - 8, power - 9)
    return torch.exp2(torch.where(amax > 0, power, -126).clamp(-126, 120).float())


def _plain_append(s: dict) -> None:
    ends, lengths, table = s["ends"].long(), s["lengths"].long(), s["table"].long()
    counts = torch.diff(ends, prepend=ends.new_zeros(1))
    t = torch.arange(s["kv"].shape[0], device="cuda")
    request = torch.searchsorted(ends, t, right=True)
    slot = lengths[request] - ends[request] + t
    block = table[request, slot // BLOCK]
    x = torch.cat([s["kv"], s["k_rope"]], dim=-1).float()
    amax = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)                     # [rows, latent_heads]
    scale = s["scale"]
    need = torch.zeros_like(scale).scatter_reduce_(0, block[:, None].expand_as(amax), amax, "amax")
    need = _needed_scale(need)
    # The block that a request's rows begin in keeps its older rows, under a scale that holds both.
    base = lengths - counts
    edge, older = table[torch.arange(len(base), device="cuda"), base // BLOCK], base % BLOCK
    grown = torch.where((older > 0)[:, None], torch.maximum(scale[edge], need[edge]), need[edge])
    ratio = scale[edge] / grown
    before = _codes(s)[edge].view(torch.float8_e4m3fn).float()
    kept = (torch.arange(BLOCK, device="cuda") < older[:, None])[..., None, None]
    after = _e4m3(torch.where(kept, before * ratio[:, None, :, None], before))
    _codes(s)[edge] = after.view(torch.uint8)
    scale[block] = need[block]
    scale[edge] = grown
    _codes(s)[block, slot % BLOCK] = _e4m3(x / scale[block][..., None]).view(torch.uint8)
    if s["positions"] is not None:
        entry = s["entries"].long()[request]
        s["positions"][entry, slot] = s["row_positions"]
        s["weights"][entry, slot] = 0.0


def _plain_evict(s: dict) -> None:
    lengths, budgets, table = s["lengths"].long(), s["budgets"].long(), s["table"].long()
    entry, capacity = s["entries"].long(), s["capacity"]
    slots = torch.arange(capacity, device="cuda")
    inside = slots < lengths[:, None]
    weights, positions = s["weights"][entry], s["positions"][entry].long()
    latest = torch.where(inside, positions, -1).amax(1, keepdim=True)
    protected = (positions < s["first"]) | (positions > latest - s["last"])
    rank = torch.where(protected, math.inf, weights).masked_fill(~inside, -math.inf)
    order = rank.argsort(dim=1, descending=True, stable=True)                   # ties: the lower slot first
    keep = torch.minimum(lengths, budgets)
    kept = torch.zeros_like(inside).scatter_(1, order, slots < keep[:, None])
    hole, source = ~kept & (slots < keep[:, None]), kept & (slots >= keep[:, None])
    request, dst = hole.nonzero(as_tuple=True)
    _, src = source.nonzero(as_tuple=True)                                      # as many of each in every request
    counts = hole.sum(1)
    nth = hole.cumsum(1)[request, dst] - 1
    s["move_src"][request, nth], s["move_dst"][request, nth] = src.to(torch.int32), dst.to(torch.int32)
    s["move_counts"].copy_(counts)
    s["kept"].copy_(keep)
    # A block that receives rows takes the largest scale among them and its own.
    scale, codes = s["scale"], _codes(s)
    from_block, to_block = table[request, src // BLOCK], table[request, dst // BLOCK]
    offered = scale[from_block]
    grown = scale.scatter_reduce(0, to_block[:, None].expand_as(offered), offered, "amax")
    moved = codes[from_block, src % BLOCK].view(torch.float8_e4m3fn).float()
    moved = _e4m3(moved * (scale[from_block] / grown[to_block])[..., None])
    wider = torch.unique(to_block)
    last = torch.full((scale.shape[0],), BLOCK, device="cuda")                  # rows of a block that stay
    last[table[torch.arange(len(keep), device="cuda"), (keep - 1) // BLOCK]] = (keep - 1) % BLOCK + 1
    before = codes[wider].view(torch.float8_e4m3fn).float()
    stays = (torch.arange(BLOCK, device="cuda") < last[wider][:, None])[..., None, None]
    again = _e4m3(torch.where(stays, before * (scale / grown)[wider][:, None, :, None], before))
    codes[wider] = again.view(torch.uint8)
    codes[to_block, dst % BLOCK] = moved.view(torch.uint8)
    scale.copy_(grown)
    owner = entry[request]
    s["weights"][owner, dst] = s["weights"][owner, src]
    s["positions"][owner, dst] = s["positions"][owner, src]


# --------------------------------------------------------- work and 64 bits
def work(case: dict) -> dict:
    g = case["latent_heads"]
    if case["kind"] == "append":
        rows = sum(_spread(case["rows_lo"], case["rows_hi"], case["batch"]))
        return {"bytes": rows * (g * ROW * 3 + (12 if case["pool"] else 0)), "flops": 2 * rows * g * ROW}
    lengths = _lengths(case)
    if case["kind"] == "evict":
        # Which tokens move depends on the weights: those kept beyond the budget, in proportion.
        kept = [n - case["over"] for n in lengths]
        moved = sum(min(case["over"], k * case["over"] // n + case["last"]) for n, k in zip(lengths, kept))
        return {"bytes": 8 * sum(lengths) + moved * (2 * g * ROW + 24), "flops": sum(lengths)}
    heads, counts = case["heads"], [min(case["rows"], n) for n in lengths]
    rows = sum(counts)
    if case["list"]:
        seen = [min(case["list"], n - (c - 1 - i)) for n, c in zip(lengths, counts) for i in range(c)]
        read, pairs = sum(seen) * (g * ROW + 4), sum(seen) * heads
    else:
        read = sum(lengths) * g * ROW + (8 * sum(lengths) if case["weights"] else 0)
        pairs = heads * sum(c * n - c * (c - 1) // 2 for n, c in zip(lengths, counts))
    return {"bytes": read + rows * heads * 2 * (ROW + LATENT), "flops": 2 * pairs * (ROW + LATENT)}


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(s)
    if case["kind"] == "evict":
        return _exact_evict(s)
    g, per = case["latent_heads"], case["heads"] // case["latent_heads"]
    q = torch.cat([s["query"], s["query_rope"]], -1).double()
    out = torch.zeros(q.shape[0], case["heads"], LATENT, dtype=torch.float64, device="cuda")
    weights = None if s["weights"] is None else s["weights"].double()
    start = 0
    for b, (end, length) in enumerate(zip(s["ends"].tolist(), s["lengths"].tolist())):
        blocks = s["table"][b, : -(-length // BLOCK)].long()
        kv = (s["cache"][blocks].double() * s["scale"][blocks].double()[:, None, :, None]).flatten(0, 1)[:length]
        for lo in range(start, end, 32):
            r = torch.arange(lo, min(end, lo + 32), device="cuda")
            visible = length - (end - 1 - r)
            for h in range(g):
                if s["ids"] is None:
                    keys = kv[:, h].expand(len(r), -1, -1)
                    seen = torch.arange(length, device="cuda") < visible[:, None]
                else:
                    ids = s["ids"][r].long()
                    seen = (ids >= 0) & (ids < visible[:, None])
                    keys = kv[ids.clamp(0, length - 1), h]
                mine = q[r, h * per:(h + 1) * per]
                score = (torch.matmul(mine.reshape(-1, ROW), kv[:, h].T).view(len(r), per, -1) if s["ids"] is None
                         else torch.matmul(mine, keys.transpose(1, 2))) * SOFTMAX_SCALE
                score.masked_fill_(~seen[:, None], -math.inf)
                p = torch.softmax(score, -1).nan_to_num(0.0)
                out[r, h * per:(h + 1) * per] = (torch.matmul(p.flatten(0, 1), kv[:, h, :LATENT]).view(len(r), per, -1)
                                                 if s["ids"] is None else torch.matmul(p, keys[..., :LATENT]))
                if weights is not None:
                    weights[int(s["entries"][b]), :length] += p.sum((0, 1))
        start = end
    return {"out": out} if weights is None else {"out": out, "weights": weights}


def _least_scale(amax: float) -> float:
    return 2.0 ** min(120, max(-126, math.ceil(math.log2(amax / 448.0)))) if amax > 0 else 2.0 ** -126


def _exact_append(s: dict):
    cache, scale = s["cache"].double(), s["scale"].double()
    start = 0
    for b, (end, length) in enumerate(zip(s["ends"].tolist(), s["lengths"].tolist())):
        x = torch.cat([s["kv"][start:end], s["k_rope"][start:end]], -1).double()
        base, done = length - (end - start), 0
        while done < end - start:
            slot = base + done
            block, row = int(s["table"][b, slot // BLOCK]), slot % BLOCK
            n = min(BLOCK - row, end - start - done)
            part = x[done:done + n]
            need = torch.tensor([_least_scale(v) for v in part.abs().amax((0, 2)).tolist()], device="cuda").double()
            new = torch.maximum(scale[block], need) if row else need
            cache[block, :row] *= (scale[block] / new)[:, None]
            cache[block, row:row + n] = part / new[:, None]
            scale[block] = new
            done += n
        start = end
    out = {"cache": cache, "scale": scale}
    if s["positions"] is None:
        return out
    weights, start = s["weights"].double(), 0
    for b, (end, length) in enumerate(zip(s["ends"].tolist(), s["lengths"].tolist())):
        weights[int(s["entries"][b]), length - (end - start):length] = 0.0
        start = end
    return out | {"positions": None, "weights": weights}


def _exact_evict(s: dict):
    cache, scale = s["cache"].double(), s["scale"].double()
    weights, rows = s["weights"].double(), s["cache"].double() * s["scale"].double()[:, None, :, None]
    before = s["scale"].double()
    for b, (length, budget) in enumerate(zip(s["lengths"].tolist(), s["budgets"].tolist())):
        e, keep = int(s["entries"][b]), min(length, budget)
        w, pos = weights[e, :length].tolist(), s["positions"][e, :length].tolist()
        top = max(pos)
        free = sorted((t for t in range(length) if s["first"] <= pos[t] <= top - s["last"]), key=lambda t: (-w[t], t))
        held = [t for t in range(length) if not s["first"] <= pos[t] <= top - s["last"]]
        kept = set((held + free)[:keep])
        holes = [t for t in range(keep) if t not in kept]
        sources = [t for t in range(keep, length) if t in kept]
        table = s["table"][b].long()
        src, dst = (torch.tensor(v, dtype=torch.long, device="cuda") for v in (sources, holes))
        for i, j in zip(sources, holes):
            to = int(table[j // BLOCK])
            scale[to] = torch.maximum(scale[to], before[table[i // BLOCK]])
        for block, cut in ((int(table[j]), min(BLOCK, keep - j * BLOCK)) for j in range(-(-keep // BLOCK))):
            cache[block, :cut] *= (before[block] / scale[block])[:, None]
        cache[table[dst // BLOCK], dst % BLOCK] = (rows[table[src // BLOCK], src % BLOCK]
                                                   / scale[table[dst // BLOCK]][..., None])
        weights[e, dst] = weights[e, src]
    return {"cache": cache, "scale": scale, "positions": None, "weights": weights, "move_src": None, "move_dst": None,
            "move_counts": None, "kept": None}
