"""A row that sees a NaN is NaN, wherever the work is cut: also where another part
of its keys has scores so large that nothing else counts."""

from __future__ import annotations

import pytest
import torch

from _prefix import DTYPES, PAGE, SCALE, attention_bound, call_attention, check_attention, make_cache, make_queries
from oracle import prefix_oracle as O

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


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,at", [(4, 40), (4, 399), (64, 40), (64, 399), (128, 40), (128, 399)])
def test_infinite_values(heads, at, dtype):
    """In a tile that every row sees whole, and in the last one: under a score of
    +inf the row is NaN; under one of -inf the key has no weight, and only its
    infinite dim may be NaN."""
    t = DTYPES[dtype]
    print(f"INF {heads} {at} {dtype}", flush=True)
    c = make_queries(make_cache([], [], [400] * 8, 64, t), [2] * 8, heads, 65)   # (the first of two rows sees a key less)
    c["query"][..., 5] = c["query"][..., 5].abs() + 0.5
    for b in range(8):
        c["kv_cache"][int(c["table"][b, at // PAGE]), at % PAGE, 0, 5] = float("inf") if b % 2 else float("-inf")
    without = {k: v.clone() for k, v in c.items()}   # that key far below all others: no weight either
    for b in range(0, 8, 2):
        page = int(c["table"][b, at // PAGE])
        without["kv_cache"][page, at % PAGE] = 0.0
        without["kv_cache"][page, at % PAGE, 0, 5] = torch.finfo(t).min / 2
    d = {k: v.cuda() for k, v in c.items()}
    call_attention(d, groups=False)
    got = d["out"].cpu()
    sees = [at < 400 - (1 - row % 2) for row in range(16)]
    for row in range(16):
        if row // 2 % 2 and sees[row]:
            assert bool(got[row].isnan().all()), row
            got[row] = 0
        else:   # (the dim of the infinite value: NaN, or without the key)
            assert bool(got[row][:, [i for i in range(512) if i != 5]].isfinite().all()), row
            assert not bool(got[row, :, 5].isinf().any()), row
    args = [c[k] for k in ("query_rope", "query", "ends", "lengths", "table")]
    want, size, _ = O.attention(*args, without["k_rope"], without["kv_cache"], SCALE)
    clean = {**c, "kv_cache": c["kv_cache"].nan_to_num(0, 0, 0)}   # (the scores' sizes without the key)
    bound = attention_bound(clean, want, size, O.attention(*args, clean["k_rope"], clean["kv_cache"], SCALE)[2])
    for row in range(16):
        if not (row // 2 % 2 and sees[row]):
            off = (got[row].double() - want[row]).abs()
            assert bool(((off <= bound[row]) | got[row].isnan()).all()), row
