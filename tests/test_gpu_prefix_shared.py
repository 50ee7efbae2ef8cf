"""Prefixes that are read once: calls that save enough by it, where a group's
items and its requests' own meet in the join."""

from __future__ import annotations

import pytest
import torch

from _prefix import (DTYPES, READ_ONCE, SCALE, api, call_attention, check_attention, i32, make_cache, make_queries,
                     shared_units)

pytestmark = pytest.mark.gpu


def _run(c, counts, heads, once=True):
    assert (shared_units(c, counts, heads) >= READ_ONCE) == once
    d = {k: v.cuda() for k, v in c.items()}
    call_attention(d)
    torch.cuda.synchronize()
    check_attention(d["out"].cpu(), c)
    return d


def _own(n, most, seed=3):
    return [(i * 37 + seed) % (most + 1) for i in range(n)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("requests,prefix,heads", [
    (120, 2048, 1), (60, 1024, 5), (48, 1536, 16), (33, 2048, 33), (48, 2560, 64), (20, 6144, 96),
])
def test_one_group(requests, prefix, heads, dtype):
    print(f"SHARED {requests} {prefix} {heads} {dtype}", flush=True)
    counts = [1] * requests
    c = make_cache([prefix], [requests], _own(requests, 70), requests, DTYPES[dtype])
    _run(make_queries(c, counts, heads, 5, pad=1), counts, heads)


def test_either_side_of_the_rule():
    """The same requests a page below and above what makes their prefix be read once."""
    counts = [1] * 64
    seen = []
    for pages in (6, 7, 8, 9):
        c = make_queries(make_cache([pages * 128], [64], _own(64, 40), pages, torch.bfloat16), counts, 16, 6)
        once = shared_units(c, counts, 16) >= READ_ONCE
        seen.append(once)
        _run(c, counts, 16, once)
    assert True in seen and False in seen


def test_groups_rows_and_loose_requests():
    """Groups of several sizes and prefixes, drafted rows, requests without rows,
    requests that share nothing, rows behind the last."""
    groups, prefixes = [30, 1, 50, 2, 60], [1280, 900, 770, 300, 1024]
    own = _own(sum(groups) + 9, 150)
    counts = [(i % 4 != 3) + (i % 11 == 0) * 2 for i in range(len(own))]
    c = make_queries(make_cache(prefixes, groups, own, 8, torch.bfloat16), counts, 8, 9, pad=3)
    _run(c, counts, 8)


def test_more_requests_than_a_workgroup_plans():
    groups, prefixes = [200, 150], [768, 512]
    own = _own(400, 30)
    counts = [1] * 400
    c = make_queries(make_cache(prefixes, groups, own, 10, torch.float16), counts, 4, 11)
    _run(c, counts, 4)


def test_requests_shorter_than_their_prefix():
    """Rows that end within the prefix, and lengths of zero."""
    counts = [1 + i % 2 for i in range(64)]
    c = make_queries(make_cache([1536], [64], _own(64, 20), 12, torch.bfloat16), counts, 8, 13)
    for i in range(0, 64, 3):
        c["lengths"][i] = (i * 61) % 1536
    c["lengths"][5] = 0
    c["lengths"][7] = -4
    _run(c, counts, 8)


def test_pages_that_name_nothing():
    counts = [1] * 64
    c = make_queries(make_cache([1536], [64], _own(64, 140), 14, torch.bfloat16), counts, 8, 15)
    c["table"][:, 3] = -1
    c["table"][:, 7] = 1 << 30
    c["table"][9, -1] = -1
    _run(c, counts, 8)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_values_in_masked_places(dtype):
    """Infinities and NaN behind what a short request sees, in pages that the
    others see nothing of."""
    counts = [1] * 64
    c = make_queries(make_cache([1536], [64], _own(64, 100), 16, DTYPES[dtype]), counts, 8, 17)
    for b in range(0, 64, 7):
        n = int(c["lengths"][b])
        page, row = int(c["table"][b, (n - 1) // 128]), (n - 1) % 128
        c["kv_cache"][page, row + 1:] = float("nan")
        c["k_rope"][page, row + 1:] = float("inf")
    _run(c, counts, 8)


def test_growing_scores():
    """References that move within the prefix and behind it."""
    counts = [1] * 64
    c = make_queries(make_cache([1536], [64], _own(64, 100), 18, torch.bfloat16), counts, 8, 19)
    for b in (0, 9, 31):
        length = int(c["lengths"][b])
        for s in range(0, length, 50):
            page, row = int(c["table"][b, s // 128]), s % 128
            c["kv_cache"][page, row, 0] = c["query"][b, 3].float().mul(s / length).to(torch.bfloat16)
    _run(c, counts, 8)


def test_replays_on_other_lengths():
    """A graph whose replays share, share other prefixes, and do not share."""
    counts = [1] * 64
    c = make_queries(make_cache([1536], [64], [60 + i for i in range(64)], 20, torch.bfloat16), counts, 8, 21)
    d = {k: v.cuda() for k, v in c.items()}
    call_attention(d)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call_attention(d)
    for prefix, end, less in ((1536, 64, 0), (1024, 64, 30), (1536, 50, 7), (128, 64, 1), (0, 0, 2), (1536, 64, 40)):
        lengths = c["lengths"] - less
        d["prefix"].fill_(prefix)
        d["group_ends"].fill_(end)
        d["lengths"].copy_(lengths)
        d["out"].fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        (d["query"].float().sum() + 1).item()
        torch.cuda.synchronize()
        check_attention(d["out"].cpu(), {**c, "lengths": lengths})


def test_overlapping_groups():
    """Group ends in any order: a request counts with one group at most."""
    counts = [1] * 64
    c = make_queries(make_cache([1536], [64], _own(64, 50), 22, torch.bfloat16), counts, 8, 23)
    for ends in ([64, 0, 64], [64, 10, 64, 5, 64], [70, -9, 64, 64]):
        d = {k: v.cuda() for k, v in c.items()}
        d["group_ends"], d["prefix"] = i32(ends).cuda(), i32([1536] * len(ends)).cuda()
        call_attention(d)
        check_attention(d["out"].cpu(), c)


def test_same_call_twice_is_the_same():
    counts = [1] * 64
    c = make_queries(make_cache([1536], [64], _own(64, 90), 24, torch.bfloat16), counts, 16, 25)
    d = _run(c, counts, 16)
    first = d["out"].clone()
    for _ in range(3):
        d["out"].fill_(7.0)
        call_attention(d)
        assert torch.equal(d["out"], first)
    api().shared_prefix_attention(d["query_rope"], d["query"], d["ends"], d["lengths"], d["table"], d["k_rope"], d["kv_cache"],
                                  SCALE, d["out"])
    check_attention(d["out"].cpu(), c)
