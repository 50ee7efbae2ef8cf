"""Lengths past the table: its tokens behind the last slot are nowhere, and a row
sees the slots that its own length names, as norm_rope_append writes them."""

from __future__ import annotations

import pytest
import torch

from _prefix import DTYPES, PAGE, READ_ONCE, call_attention, check_attention, make_cache, make_queries, shared_units

pytestmark = pytest.mark.gpu


def _run(c, groups=False):
    d = {k: v.cuda() for k, v in c.items()}
    call_attention(d, groups=groups)
    torch.cuda.synchronize()
    check_attention(d["out"].cpu(), c)
    return d["out"].cpu()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("requests,heads", [(2, 8), (2, 64), (40, 100), (300, 2)])
def test_rows_past_the_table(requests, heads, dtype):
    """Rows of which some have slots and some have not, and all have not; by the plan of
    every workgroup and by the one before."""
    print(f"PAST {requests} {heads} {dtype}", flush=True)
    counts = [1 + i % 4 for i in range(requests)]
    tokens = 8 * PAGE if heads == 100 else 2 * PAGE
    c = make_queries(make_cache([], [], [tokens] * requests, 90, DTYPES[dtype]), counts, heads, 91, pad=1)
    for i in range(requests):
        c["lengths"][i] += (2, 1, 0, 3, 4, 700)[i % 6]
    got = _run(c)
    c["lengths"][c["lengths"] == tokens + 700] = 2 ** 31 - 1   # (the largest: as many slots)
    d = {k: v.cuda() for k, v in c.items()}
    call_attention(d, groups=False)
    assert torch.equal(d["out"].cpu(), got)


def test_a_row_sees_no_less_than_the_one_before_it_wrote():
    """Two rows: the first has the last slot, the second none.  Both see every slot."""
    c = make_queries(make_cache([], [], [PAGE], 92, torch.bfloat16), [2], 4, 93)
    c["lengths"][0] = PAGE + 1
    c["kv_cache"][int(c["table"][0, 0]), -1] = 30.0 * c["query"][0, 0].sign()   # what the first row's first head looks for
    c["query"][1], c["query_rope"][1] = c["query"][0], c["query_rope"][0]
    got = _run(c)
    assert torch.equal(got[0], got[1]) and bool((got[0, 0].abs() > 25).all())


def test_groups_past_the_table():
    counts = [1 + i % 3 for i in range(64)]
    c = make_queries(make_cache([1536], [64], [128] * 64, 94, torch.bfloat16), counts, 8, 95)
    c["lengths"] += torch.arange(64, dtype=torch.int32) % 5
    assert shared_units(c, counts, 8) >= READ_ONCE
    _run(c, groups=True)
