"""Groups in which requests have ended: they have no rows and hold no pages, the
first of the group among them."""

from __future__ import annotations

import pytest
import torch

from _prefix import READ_ONCE, call_attention, check_attention, make_cache, make_queries, shared_units

pytestmark = pytest.mark.gpu


def _run(groups, prefixes, own, heads, ended, dtype=torch.bfloat16):
    counts = [0 if b in ended else 1 for b in range(len(own))]
    c = make_queries(make_cache(prefixes, groups, own, 110 + len(ended), dtype), counts, heads, 111, pad=2)
    for b in ended:
        c["lengths"][b] = 0
        c["table"][b] = -1
    assert shared_units(c, counts, heads) >= READ_ONCE
    d = {k: v.cuda() for k, v in c.items()}
    call_attention(d)
    torch.cuda.synchronize()
    check_attention(d["out"].cpu(), c)


@pytest.mark.parametrize("ended", [{0}, {0, 1, 2}, {5, 63}, set(range(20)), {0} | set(range(9, 64, 5))])
def test_one_group(ended):
    print(f"ENDED {sorted(ended)[:5]}", flush=True)
    _run([64], [2560], [(i * 37) % 70 for i in range(64)], 8, ended)


def test_all_of_a_group_have_ended():
    _run([40, 3, 60], [1280, 640, 1536], [(i * 41) % 90 for i in range(110)], 8, {40, 41, 42, 43, 44, 103})


def test_more_requests_than_a_workgroup_plans():
    _run([200, 150], [1280, 768], [(i * 29) % 40 for i in range(400)], 4, {0, 1, 200, 201, 202, 333}, torch.float16)
