"""norm_rope_append on the GPU vs the 64-bit oracle, within bounds that follow
from the roundings; rows that nobody names stay bit for bit."""

from __future__ import annotations

import pytest
import torch

from _prefix import DTYPES, api, call_norm, check_norm, i32, norm_inputs

pytestmark = pytest.mark.gpu


def _run(d, eps=1e-6):
    got = {k: None if v is None else v.cuda() for k, v in d.items()}
    call_norm(got, eps)
    torch.cuda.synchronize()
    got = {k: None if v is None else v.cpu() for k, v in got.items()}
    check_norm(got, d, eps)
    return got


@pytest.mark.parametrize("counts,past,heads,nope,dtype", [
    ([1], [0], 1, 0, "bf16"),
    ([1, 1, 1, 1], [127, 128, 5, 300], 64, 0, "bf16"),
    ([1, 1, 1], [0, 255, 12], 4, 192, "f16"),
    ([3, 0, 5, 130], [126, 9, 0, 64], 5, 8, "bf16"),
    ([129, 256], [0, 90], 3, 64, "f16"),
    ([17], [1000], 7, 120, "bf16"),
    ([9], [1], 2, 448, "f16"),
    ([9, 4], [1, 130], 2, 456, "bf16"),
    ([5], [1], 3, 512, "f16"),
    ([2] * 70, [i for i in range(70)], 2, 128, "bf16"),
])
def test_rows(counts, past, heads, nope, dtype):
    print(f"NORM {counts[:4]} {past[:4]} N={heads} nope={nope} {dtype}", flush=True)
    _run(norm_inputs(counts, past, heads, nope, DTYPES[dtype], seed=len(counts) + heads, pad=3))


def test_nope_dims_without_norms_are_not_read():
    d = norm_inputs([4, 1], [3, 128], 3, 64, torch.bfloat16, 5, norm=False)
    d["query"][..., :64] = float("nan")
    _run(d)


def test_norm_of_a_query_without_nope_dims():
    _run(norm_inputs([4, 1], [3, 128], 6, 0, torch.bfloat16, 6, norm=True))


def test_wider_tables_of_angles():
    _run(norm_inputs([4, 7], [3, 128], 2, 64, torch.float16, 7, stride=128))


def test_many_requests():
    """More requests than a wave has lanes, and than 64 times as many; empty ones among them."""
    for batch in (300, 5000):
        counts = [(i * 7) % 3 for i in range(batch)]
        _run(norm_inputs(counts, [(i * 13) % 140 for i in range(batch)], 1, 0, torch.bfloat16, batch, pad=2))


@pytest.mark.parametrize("eps", [0.0, 1e-6, 0.5])
def test_values(eps):
    """Zero rows, the types' extremes, infinities and NaN stay in their rows."""
    d = norm_inputs([1] * 7, [0] * 7, 2, 64, torch.bfloat16, 8)
    for k in ("kv", "query"):
        x = d[k]
        x[0] = 2.0 ** -100 if eps else 1.0
        x[1] = 2.0 ** 50
        x[2, ..., 3] = 2.0 ** 60
        x[3, ..., 5] = float("nan")
        x[4] = 2.0 ** -60 if eps else 2.0 ** -30
        if eps:
            x[5] = 0.0
    _run(d, eps)


def test_infinite_values_stay_in_their_rows():
    d = norm_inputs([1] * 3, [0] * 3, 2, 64, torch.float16, 9)
    clean = _run({k: None if v is None else v.clone() for k, v in d.items()})
    for k in ("kv", "query"):
        d[k][1, ..., 4] = float("inf")
    got = {k: None if v is None else v.cuda() for k, v in d.items()}
    call_norm(got)
    for k in ("query_rope", "query_nope"):
        for t in (0, 2):
            assert torch.equal(got[k][t].cpu(), clean[k][t])
    page = d["table"][:, 0].long()
    for t in (0, 2):
        assert torch.equal(got["kv_cache"][page[t], 0].cpu(), clean["kv_cache"][page[t], 0])
    # inf / inf: NaN; every other value of the row over an infinite root: 0
    row = got["kv_cache"][page[1], 0, 0].cpu()
    assert row[4].isnan() and bool((row[:4] == 0).all()) and bool((row[5:] == 0).all())


def test_skips_what_names_nothing():
    d = norm_inputs([80, 20, 95, 10, 4], [120, 280, 0, 50, 0], 2, 0, torch.bfloat16, 10, pad=4)
    blocks = d["kv_cache"].shape[0]
    d["table"][0, 1], d["table"][1, 2] = -1, blocks
    d["lengths"][2] = 90      # begins before slot 0
    d["lengths"][3] = 70000   # behind the table
    d["lengths"][4] = -5
    _run(d)


def test_ends_past_the_rows():
    d = norm_inputs([6, 6], [0, 130], 2, 8, torch.bfloat16, 11)
    d["ends"][1] = 99
    got = {k: None if v is None else v.cuda() for k, v in d.items()}
    call_norm(got)  # the second request's rows lie at other slots than it says: only what is in range is touched
    torch.cuda.synchronize()


def test_replays_and_streams():
    d = {k: None if v is None else v.cuda() for k, v in norm_inputs([3, 2], [126, 0], 4, 64, torch.bfloat16, 12).items()}
    eager = {k: None if v is None else v.clone() for k, v in d.items()}
    call_norm(eager)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call_norm(d)
    for _ in range(3):
        for k in ("kv_cache", "k_rope", "query_rope", "query_nope"):
            d[k].zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for k in ("query_rope", "query_nope"):
            assert torch.equal(d[k], eager[k])
        page = d["table"][:, 0].long()
        assert torch.equal(d["kv_cache"][page[0], 126], eager["kv_cache"][page[0], 126])
        assert torch.equal(d["k_rope"][page[1], :2], eager["k_rope"][page[1], :2])


def test_a_call_without_rows():
    d = norm_inputs([0, 0], [5, 6], 2, 0, torch.bfloat16, 13)
    _run(d)
    e = norm_inputs([1], [0], 2, 0, torch.bfloat16, 14)
    e["ends"], e["lengths"], e["table"] = i32([]), i32([]), torch.zeros(0, 1, dtype=torch.int32)
    with pytest.raises(RuntimeError):  # (requests there have to be, or none at all: a table of no rows is fine)
        api().norm_rope_append(*[e[k].cuda() for k in ("query", "kv", "cos", "sin", "kv_weight", "ends", "lengths")],
                               torch.zeros(1, 0, dtype=torch.int32, device="cuda"), e["k_rope"].cuda(), e["kv_cache"].cuda(),
                               e["query_rope"].cuda())
    call_norm({k: None if v is None else v.cuda() for k, v in e.items()})
