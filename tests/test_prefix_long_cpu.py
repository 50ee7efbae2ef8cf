"""The check of the attention over many keys, on outputs that are wrong by a page, a
window of pages or a part, and on those that are not."""

from __future__ import annotations

import functools

import pytest
import torch

from _prefix import DTYPES, SCALE, make_cache, make_queries
from _prefix_long import Check, batch_on_a_prefix, many_keys, two_on_a_prefix, with_table
from oracle import prefix_oracle as O

LOG2E = 1.4426950408889634


def _drop(first, stop, step=1):
    return lambda table: [row.__setitem__(i, -1) for row in table for i in range(first, min(stop, len(row)), step)]


def _instead(first, stop, other):
    """Pages [first, stop) are read from `other` on."""
    return lambda table: [row.__setitem__(i, row[other + i - first]) for row in table for i in range(first, min(stop, len(row)))]


def _of_the_other(first, stop):
    def change(table):
        table[0][first:stop], table[1][first:stop] = table[1][first:stop], table[0][first:stop]
    return change


@functools.cache
def _check(make, dtype):
    return Check(make(2, DTYPES[dtype]))


def test_the_checks_output_is_the_oracles():
    c = make_queries(make_cache([384], [2], [30, 200], 83, torch.bfloat16), [3, 2], 5, 84)
    want, _, _ = O.attention(c["query_rope"], c["query"], c["ends"], c["lengths"], c["table"], c["k_rope"], c["kv_cache"], SCALE)
    assert torch.allclose(Check(c).want, want, rtol=1e-12, atol=1e-14)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("make", [many_keys, two_on_a_prefix])
@pytest.mark.parametrize("change", [
    _drop(0, 4096, 2), _drop(64, 128), _instead(64, 128, 0), _drop(700, 701), _instead(700, 701, 699), _instead(1000, 1004, 0),
    _drop(1024, 4096),
], ids=["half", "window", "window-again", "page", "page-again", "pages-again", "end"])
def test_wrong_pages_are_noticed(change, make, dtype):
    check = _check(make, dtype)
    got = with_table(check.c, change)
    assert got is None or check.worst(got) > 1.0
    assert got is not None or make is many_keys


def test_another_requests_page_is_noticed():
    check = Check(batch_on_a_prefix(4, torch.bfloat16, requests=4))
    last = int(check.c["lengths"].min()) // 128
    assert check.worst(with_table(check.c, _of_the_other(130, 131))) > 1.0
    assert check.worst(with_table(check.c, _drop(last - 1, last))) > 1.0


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("part", ["lost", "twice"])
def test_a_part_lost_or_counted_twice_is_noticed(part, dtype):
    check = _check(many_keys, dtype)
    c = check.c
    keys = c["kv_cache"][c["table"][0].long()].flatten(0, 2).double()
    rope = c["k_rope"][c["table"][0].long()].flatten(0, 2).double()
    p = torch.softmax((c["query"][0].double() @ keys.T + c["query_rope"][0].double() @ rope.T) * SCALE, -1)
    p[:, 512 * 77:512 * 78] *= 0.0 if part == "lost" else 2.0
    assert check.worst((p @ keys / p.sum(-1, keepdim=True))[None].to(DTYPES[dtype])) > 1.0


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_rounded_weights_and_sums_pass(dtype):
    """The operator's own arithmetic: weights in 16 bits, sums in fp32."""
    t = DTYPES[dtype]
    for make in (many_keys, two_on_a_prefix):
        check = _check(make, dtype)
        c = check.c
        out = torch.zeros(c["query"].shape, dtype=t)
        for b, n in enumerate(c["lengths"].tolist()):
            at = c["table"][b, : -(-n // 128)].long()
            keys, rope = (c[k][at].flatten(0, 2)[:n].float() for k in ("kv_cache", "k_rope"))
            x = (c["query"][b].float() @ keys.T + c["query_rope"][b].float() @ rope.T) * (SCALE * LOG2E)
            p = torch.exp2(x - x.amax(-1, keepdim=True) + 8.0).to(t).float()
            out[b] = (p @ keys / p.sum(-1, keepdim=True)).to(t)
        assert check.worst(out) <= 1.0
