"""shared_prefix_attention over many keys, on every way through the kernels, with a
check that notices a page: windows of page ids, parts and their join."""

from __future__ import annotations

import pytest
import torch

from _prefix import DTYPES, READ_ONCE, call_attention, make_cache, make_queries, shared_units
from _prefix_long import Check, batch_on_a_prefix, many_keys, two_on_a_prefix

pytestmark = pytest.mark.gpu


def _run(c, groups=True):
    d = {k: v.cuda() for k, v in c.items()}
    call_attention(d, groups=groups)
    torch.cuda.synchronize()
    worst = Check(d).worst(d["out"])
    print("  of the tolerance:", round(worst, 3), flush=True)
    assert worst <= 1.0, worst


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads", [2, 33, 64, 65, 128])
def test_many_keys(heads, dtype):
    """One row in as many parts as there are."""
    print(f"LONG {heads} {dtype}", flush=True)
    _run(many_keys(heads, DTYPES[dtype], tokens=131072 if heads < 64 else 40000), groups=False)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads", [2, 17, 64])
def test_two_on_a_prefix(heads, dtype):
    print(f"LONG prefix {heads} {dtype}", flush=True)
    _run(two_on_a_prefix(heads, DTYPES[dtype], pages=1100 if heads < 64 else 300))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("requests,heads", [(33, 4), (20, 16), (40, 2)])
def test_read_once(requests, heads, dtype):
    print(f"LONG once {requests} {heads} {dtype}", flush=True)
    c = batch_on_a_prefix(heads, DTYPES[dtype], requests)
    assert shared_units(c, [1] * requests, heads) >= READ_ONCE
    _run(c)


@pytest.mark.parametrize("heads,requests,tokens", [(16, 40, 70000), (64, 30, 90000), (128, 24, 100000)])
def test_several_windows_in_a_part(heads, requests, tokens):
    """Work enough that a part holds more pages than a wave has lanes: a window ends
    within it.  Two requests' pages, under the tables of many."""
    print(f"LONG windows {heads}", flush=True)
    c = make_cache([], [], [tokens, tokens + 11], 76, torch.bfloat16, size=0.5)
    for k in ("table", "lengths"):
        c[k] = torch.cat([c[k]] * (requests // 2))
    assert sum(-(-int(n) // 32) for n in c["lengths"]) > 256 * 64 * 4
    _run(make_queries(c, [1] * requests, heads, 77, size=0.5), groups=False)


def test_more_requests_than_a_workgroup_plans():
    c = make_queries(make_cache([], [], [900 + 7 * i for i in range(300)], 79, torch.bfloat16), [1] * 300, 2, 80)
    _run(c, groups=False)


def test_drafted_rows():
    c = make_queries(make_cache([20000], [6], [40 + 100 * i for i in range(6)], 81, torch.float16), [4, 1, 3, 4, 2, 4], 16, 82)
    _run(c)
