"""Prompts behind a shared prefix, and from their first token: hundreds of rows a
request, whose items see different numbers of keys."""

from __future__ import annotations

import pytest
import torch

from _prefix import DTYPES, call_attention, make_cache, make_queries
from _prefix_long import Check

pytestmark = pytest.mark.gpu


def _run(c):
    d = {k: v.cuda() for k, v in c.items()}
    call_attention(d)
    torch.cuda.synchronize()
    worst = Check(d).worst(d["out"])
    print("  of the tolerance:", round(worst, 3), flush=True)
    assert worst <= 1.0, worst
    rows = int(c["ends"][-1])
    assert bool((d["out"][rows:] == 7.0).all())
    return d["out"]


@pytest.mark.parametrize("prefix,own,heads,dtype", [
    (2048, [700, 300, 1, 129], 16, "bf16"),
    (2048, [128, 256, 3], 64, "f16"),
    (384, [900, 33], 5, "bf16"),
    (1000, [400, 500], 128, "bf16"),
    (0, [1500, 2, 31], 16, "bf16"),
    (0, [700], 65, "f16"),
])
def test_prompts(prefix, own, heads, dtype):
    print(f"PROMPTS {prefix} {own} {heads} {dtype}", flush=True)
    c = make_cache([prefix], [len(own)], own, 100 + heads, DTYPES[dtype])
    _run(make_queries(c, own, heads, 101, pad=5))


def test_chunks_of_a_prompt_are_the_prompt():
    """The rows of a prompt, attended at once and in three chunks behind each other."""
    own, heads = 900, 16
    c = make_queries(make_cache([], [], [own], 102, torch.bfloat16), [own], heads, 103)
    whole = _run(c)
    for first, stop in ((0, 130), (130, 700), (700, 900)):
        part = {**c, "query": c["query"][first:stop].contiguous(), "query_rope": c["query_rope"][first:stop].contiguous(),
                "out": c["out"][first:stop].contiguous(), "ends": c["ends"] * 0 + (stop - first), "lengths": c["lengths"] * 0 + stop}
        got = _run(part)
        # (Two outputs within the check's tolerance of the same value.)
        off = (got.double() - whole[first:stop].double()).square().mean(-1).sqrt()
        assert bool((off <= 2 * Check({k: v.cuda() for k, v in part.items()}).tolerance).all())


def test_more_rows_and_requests_than_a_workgroup_plans():
    counts = [(i * 37) % 12 for i in range(400)]
    c = make_queries(make_cache([256, 640], [150, 100], [12 + i % 30 for i in range(400)], 104, torch.bfloat16), counts, 4, 105, pad=2)
    assert sum(counts) > 1024
    _run(c)
