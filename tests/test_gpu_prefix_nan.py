"""A row that sees a NaN is NaN, wherever the work is cut: also where another part
of its keys has scores so large that nothing else counts."""

from __future__ import annotations

import pytest
import torch

from _prefix import DTYPES, PAGE, call_attention, check_attention, make_cache, make_queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads", [4, 64, 128])
def test_a_part_without_weight_keeps_its_nan(heads, dtype):
    """Scores of the last page lie 288 powers of two above the others': exp2 of the
    distance is zero in fp32."""
    print(f"NAN {heads} {dtype}", flush=True)
    c = make_queries(make_cache([], [], [4000, 3000], 60, DTYPES[dtype]), [1, 1], heads, 61)
    c["kv_cache"][..., 0] = 0.0
    c["query"][..., 0] = 240.0
    for b in range(2):
        c["kv_cache"][int(c["table"][b, int(c["lengths"][b] - 1) // PAGE]), ..., 0] = 20.0
    d = {k: v.cuda() for k, v in c.items()}
    call_attention(d, groups=False)
    check_attention(d["out"].cpu(), c)
    d["kv_cache"][int(c["table"][0, 1]), 5, 0, 9] = float("nan")
    call_attention(d, groups=False)
    got = d["out"].cpu()
    assert bool(got[0].isnan().all()) and bool(got[1].isfinite().all())


def test_a_shared_part_without_weight_keeps_its_nan():
    """The same between a prefix that is read once and the requests' own tokens."""
    n = 64
    c = make_queries(make_cache([1536], [n], [40 + i for i in range(n)], 62, torch.bfloat16), [1] * n, 8, 63)
    c["kv_cache"][..., 0] = 0.0
    c["query"][..., 0] = 240.0
    for b in range(n):
        c["kv_cache"][int(c["table"][b, 12]), ..., 0] = 20.0   # (the first page of their own)
    d = {k: v.cuda() for k, v in c.items()}
    call_attention(d)
    check_attention(d["out"].cpu(), c)
    d["kv_cache"][int(c["table"][0, 3]), 77, 0, 9] = float("nan")
    call_attention(d)
    assert bool(d["out"].isnan().all())
