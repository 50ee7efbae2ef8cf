"""The attention's weights, held in 16 bits, sum to one: what their rounding does
to a row is bounded by how far the values lie from the row's output, and not by
their size."""

from __future__ import annotations

import math

import pytest
import torch

from _prefix import DTYPES, HALF_STEP, PAGE, call_attention, make_cache, make_queries
from oracle import prefix_oracle as O

pytestmark = pytest.mark.gpu

# A tile's largest P is 256; the other keys' lies between two of the type's values there.
BETWEEN = {"bf16": 255.4, "f16": 255.92}


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("requests,heads,tokens", [(1, 16, 1000), (3, 64, 700), (2, 100, 260), (46, 128, 900)])
def test_weights_between_two_steps(requests, heads, tokens, dtype):
    """Every 32nd key scores a little above the others, whose weights are all
    rounded the same way: by up to half a step, which the normaliser shares.

    The bound: the store's half step; half a step of each weight times the distance
    of its value from the output, twice (the values' own distances are summed with
    weights that are off by as much); sums of n fp32 terms, n 2^-24 each, of P and P V."""
    t = DTYPES[dtype]
    print(f"WEIGHTS {requests} {heads} {tokens} {dtype}", flush=True)
    c = make_queries(make_cache([], [], [tokens] * requests, 50, t), [1] * requests, heads, 51)
    g = torch.Generator().manual_seed(52)
    step = torch.finfo(t).eps
    c["kv_cache"] = (1.0 + step * torch.randint(0, 16, c["kv_cache"].shape, generator=g)).to(t)
    c["k_rope"].zero_()
    c["k_rope"][:, ::32, 0, 63] = 1.0
    c["query"].zero_()
    c["query_rope"].zero_()
    c["query_rope"][..., 63] = 1.0
    scale = math.log(256.0 / BETWEEN[dtype])
    d = {k: v.cuda() for k, v in c.items()}
    call_attention(d, scale, groups=False)
    torch.cuda.synchronize()
    want, _, _ = O.attention(c["query_rope"], c["query"], c["ends"], c["lengths"], c["table"], c["k_rope"], c["kv_cache"], scale)
    spread = torch.empty_like(want)   # sum of p |v - o|
    for b, n in enumerate(c["lengths"].tolist()):
        rows = c["kv_cache"][c["table"][b, : -(-n // PAGE)].long()].flatten(0, 2)[:n].double()
        p = torch.where(torch.arange(n) % 32 == 0, 256.0, BETWEEN[dtype]).double()
        spread[b] = ((p / p.sum())[:, None] * (rows - want[b, 0]).abs()).sum(0)
    bound = want.abs() * HALF_STEP[t] + 2 * HALF_STEP[t] * spread + want.abs() * (2 * tokens * 2.0 ** -24)
    worst = float(((d["out"].cpu().double() - want).abs() / bound).max())
    print("  of the bound:", round(worst, 3), flush=True)
    assert worst <= 1.0, worst
