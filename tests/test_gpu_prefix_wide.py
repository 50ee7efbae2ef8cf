"""Calls with work enough for items of 128 pairs, and those just below, whose
items hold 64."""

from __future__ import annotations

import pytest
import torch

from _prefix import DTYPES, call_attention, check_attention, make_cache, make_queries

pytestmark = pytest.mark.gpu

WIDE = 5 * 256  # tiles of 32 keys, of items of 128 pairs, above which items hold as many


def _tiles(c, counts, heads):
    return sum(-(-n * heads // 128) * -(-int(length) // 32) for n, length in zip(counts, c["lengths"]) if n > 0)


def _run(c, counts, heads, wide=True):
    assert (_tiles(c, counts, heads) > WIDE) == wide
    d = {k: v.cuda() for k, v in c.items()}
    call_attention(d)
    torch.cuda.synchronize()
    check_attention(d["out"].cpu(), c)
    return d


def _lengths(n, low, spread):
    return [low + (i * 53) % spread for i in range(n)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads", [65, 96, 127, 128])
def test_single_rows(heads, dtype):
    print(f"WIDE {heads} {dtype}", flush=True)
    counts = [1] * 48
    c = make_queries(make_cache([], [], _lengths(48, 800, 300), heads, DTYPES[dtype]), counts, heads, 1, pad=1)
    _run(c, counts, heads)


@pytest.mark.parametrize("low,wide", [(830, False), (900, True)])
def test_either_side_of_the_rule(low, wide):
    counts = [1] * 46
    c = make_queries(make_cache([], [], [low] * 46, 2, torch.bfloat16), counts, 100, 2)
    _run(c, counts, 100, wide)


def test_drafted_rows_and_rests_of_items():
    """Rows of several items, the last of them of one to 128 pairs; rows that see
    a tile less than others of their item; rows without keys."""
    counts = [3, 5, 7, 1, 12, 2, 0, 9, 4, 33]
    c = make_queries(make_cache([], [], _lengths(10, 1700, 600), 3, torch.bfloat16), counts, 40, 3, pad=2)
    c["lengths"][3] = 0
    c["lengths"][4] = 6       # the first six rows of twelve see nothing
    c["lengths"][5] = 65
    _run(c, counts, 40)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_values_in_masked_places(dtype):
    counts = [1 + i % 3 for i in range(20)]
    c = make_queries(make_cache([], [], _lengths(20, 1100, 290), 4, DTYPES[dtype]), counts, 80, 4)
    for b in range(20):
        n = int(c["lengths"][b])
        page, row = int(c["table"][b, (n - 1) // 128]), (n - 1) % 128
        c["kv_cache"][page, row + 1:] = float("nan") if b % 2 else float("inf")
        c["k_rope"][page, row + 1:] = float("-inf")
    c["table"][3, 2] = -1
    c["table"][4, -1] = 1 << 29
    for page in set(range(c["kv_cache"].shape[0])) - set(c["table"].flatten().tolist()):
        c["kv_cache"][page] = float("nan")
    _run(c, counts, 80)


def test_growing_and_extreme_scores():
    counts = [1] * 40
    c = make_queries(make_cache([], [], _lengths(40, 1100, 200), 5, torch.bfloat16), counts, 128, 5)
    for b in range(0, 40, 3):
        length = int(c["lengths"][b])
        for s in range(0, length, 40):
            page, row = int(c["table"][b, s // 128]), s % 128
            c["kv_cache"][page, row, 0] = (c["query"][b, 77].float() * (s / length)).to(torch.bfloat16)
    c["query"][1], c["query_rope"][1] = 0, 0
    c["query"][2] *= 30
    _run(c, counts, 128)


def test_replays_of_both_widths():
    """A graph whose replays take either width."""
    counts = [1] * 48
    c = make_queries(make_cache([], [], _lengths(48, 900, 200), 6, torch.bfloat16), counts, 96, 6)
    d = {k: v.cuda() for k, v in c.items()}
    call_attention(d)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call_attention(d)
    seen = set()
    for less in (0, 300, 7, 860):
        lengths = c["lengths"] - less
        seen.add(_tiles({"lengths": lengths}, counts, 96) > WIDE)
        d["lengths"].copy_(lengths)
        d["out"].fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        (d["query"].float().sum() + 1).item()
        torch.cuda.synchronize()
        check_attention(d["out"].cpu(), {**c, "lengths": lengths})
    assert seen == {True, False}
