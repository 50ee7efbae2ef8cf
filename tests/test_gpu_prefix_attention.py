"""shared_prefix_attention on the GPU vs the 64-bit oracle, within bounds that
follow from the roundings."""

from __future__ import annotations

import pytest
import torch

from _prefix import DTYPES, PAGE, SCALE, call_attention, check_attention, i32, make_cache, make_queries

pytestmark = pytest.mark.gpu


def _run(c, scale=SCALE, groups=True):
    d = {k: v.cuda() for k, v in c.items()}
    call_attention(d, scale, groups)
    torch.cuda.synchronize()
    got = d["out"].cpu()
    print("  of the bound:", round(check_attention(got, c, scale), 3), flush=True)
    return got


@pytest.mark.parametrize("heads", [1, 4, 5, 16, 32, 33, 64, 96, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_one_request(heads, dtype):
    print(f"ATTEND 1 x {heads} {dtype}", flush=True)
    for own in (1, 31, 32, 33, 128, 700):
        _run(make_queries(make_cache([], [], [own], 3, DTYPES[dtype]), [1], heads, 4), groups=False)


@pytest.mark.parametrize("prefixes,groups,own,rows,heads,dtype", [
    ([256], [2], [1, 1], 1, 4, "bf16"),
    ([389], [2], [20, 37], 1, 16, "bf16"),
    ([1024], [5], [1, 128, 3, 300, 127], 1, 64, "f16"),
    ([512, 1300], [3, 4], [5, 1, 40, 130, 129, 128, 2], 1, 8, "bf16"),
    ([640, 256], [4, 2], [10, 20, 30, 40, 4, 5, 700, 3], 4, 5, "f16"),
    ([256], [40], [1 + i * 7 % 50 for i in range(40)], 1, 33, "bf16"),
    ([2048], [9], [1 + i for i in range(9)], 2, 16, "bf16"),
    ([128, 127, 0, 5, 384], [2, 2, 2, 1, 2], [3] * 11, 1, 4, "bf16"),
    ([4096], [70], [1 + i % 3 for i in range(70)], 1, 1, "f16"),
    ([300], [3], [200, 150, 90], 40, 16, "bf16"),
    ([300], [2], [300, 150], 130, 3, "f16"),
])
def test_groups(prefixes, groups, own, rows, heads, dtype):
    print(f"ATTEND {prefixes} {groups} rows={rows} N={heads} {dtype}", flush=True)
    c = make_cache(prefixes, groups, own, seed=len(own) + heads, dtype=DTYPES[dtype])
    counts = [min(rows, n) for n in c["lengths"].tolist()]
    got = _run(make_queries(c, counts, heads, 5, pad=3))
    plain = _run(c, groups=False)
    assert got.shape == plain.shape


def test_many_requests():
    """More requests and groups than the plan has threads."""
    groups = [2 + i % 2 for i in range(500)]
    prefixes = [256 if i % 3 else 130 for i in range(500)]
    own = [(i * 7) % 40 for i in range(sum(groups) + 30)]
    c = make_cache(prefixes, groups, own, 6, torch.bfloat16)
    print("ATTEND many", flush=True)
    _run(make_queries(c, [i % 2 for i in range(len(own))], 2, 7, pad=2))


def test_windows_of_pages():
    """A prefix of more pages than are held at a time."""
    pages = 1100
    c = make_cache([pages * PAGE], [2], [3, 150], 8, torch.bfloat16)
    print("ATTEND long", flush=True)
    _run(make_queries(c, [1, 1], 2, 9))
    c = make_cache([], [], [pages * PAGE + 5], 8, torch.bfloat16)
    _run(make_queries(c, [1], 128, 9))


def test_lengths_of_zero_and_rows_that_see_nothing():
    c = make_cache([256], [4], [0, 3, 0, 5], 10, torch.bfloat16)
    c["lengths"][2] = 0
    c = make_queries(c, [1, 2, 3, 1], 8, 11)
    got = _run(c)
    assert bool((got[3:6] == 0).all())
    c = make_cache([], [], [2, 0, 1], 12, torch.float16)
    got = _run(make_queries(c, [5, 2, 1], 8, 13))  # more rows than tokens
    assert bool((got[:3] == 0).all()) and bool((got[5:7] == 0).all())


def test_requests_shorter_than_their_prefix():
    c = make_cache([640], [5], [4, 4, 4, 4, 4], 14, torch.bfloat16)
    c["lengths"][1], c["lengths"][3] = 200, 1
    _run(make_queries(c, [1, 3, 1, 1, 2], 16, 15))


def test_empty_groups_and_ends_past_the_batch():
    c = make_cache([512], [3], [4, 5, 6], 16, torch.bfloat16)
    c = make_queries(c, [1, 1, 1], 16, 17)
    c["group_ends"], c["prefix"] = i32([0, 0, 3, 3, 90]), i32([512, 99, 512, 7, 10 ** 9])
    _run(c)
    c["prefix"] = i32([1, 1, -5, 7, 2 ** 31 - 1])
    _run(c)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_values_in_masked_places(dtype):
    """NaN and infinities behind the last token, on pages that nobody names, and
    where only later rows of the request see them."""
    t = DTYPES[dtype]
    c = make_cache([256], [3], [40, 100, 7], 18, t)
    c = make_queries(c, [1, 2, 1], 16, 19)
    used = torch.zeros(c["kv_cache"].shape[0], PAGE, dtype=torch.bool)
    for row, n in zip(c["table"].tolist(), c["lengths"].tolist()):
        for slot in range(n):
            used[row[slot // PAGE], slot % PAGE] = True
    for k in ("kv_cache", "k_rope"):
        x = c[k]
        bad = torch.tensor([float("nan"), float("inf"), float("-inf"), torch.finfo(t).min])
        fill = bad[torch.arange(x[~used].numel()) % 4].view(x[~used].shape).to(t)
        x[~used] = fill
    print(f"ATTEND masked {dtype}", flush=True)
    _run(c)
    # The newest token of request 1 holds NaN: its last row does not stay finite, the others do.
    page, slot = int(c["table"][1, 2]), int(c["lengths"][1]) - 1 - 2 * PAGE
    c["kv_cache"][page, slot, 0, 9] = float("nan")
    d = {k: v.cuda() for k, v in c.items()}
    call_attention(d)
    got = d["out"].cpu()
    assert bool(got[2].isnan().all()) and bool(got[[0, 1, 3]].isfinite().all())


def test_pages_that_name_nothing():
    c = make_cache([512], [3], [200, 300, 40], 20, torch.bfloat16)
    blocks = c["kv_cache"].shape[0]
    c["table"][:, 1] = blocks          # of the prefix, in every table
    c["table"][0, 4], c["table"][1, 5] = -1, blocks + 7
    c["lengths"][2] = c["table"].shape[1] * PAGE + 900  # behind the table
    c["table"][2] = c["table"][1]
    _run(make_queries(c, [1, 2, 1], 16, 21))


def test_all_pages_unnamed():
    c = make_cache([256], [2], [3, 4], 22, torch.bfloat16)
    c["table"][:] = -1
    got = _run(make_queries(c, [1, 1], 8, 23))
    assert bool((got == 0).all())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_growing_and_extreme_scores(dtype):
    """Scores that grow along the tokens, so that references move; large ones,
    where one key has everything; tiny ones; a negative scale."""
    t = DTYPES[dtype]
    c = make_cache([1024], [3], [300, 200, 100], 24, t)
    c = make_queries(c, [1, 1, 1], 32, 25)
    for b, n in enumerate(c["lengths"].tolist()):
        for col in range(-(-n // PAGE)):
            c["kv_cache"][int(c["table"][b, col])] = (0.05 + 0.2 * col) * torch.randn(PAGE, 1, 512, generator=torch.Generator().manual_seed(int(c["table"][b, col]))).to(t)
    print(f"ATTEND growing {dtype}", flush=True)
    _run(c)
    for scale in (-SCALE, SCALE * 8, SCALE * 1e-3, 0.0):
        _run(c, scale)


def test_scores_far_below_zero():
    """All scores of a row near -1000: its weights are still those of its largest."""
    c = make_cache([256], [2], [10, 20], 26, torch.float16)
    c = make_queries(c, [1, 1], 8, 27)
    c["kv_cache"][..., 0] = 20.0
    c["query"][..., 0] = -1200.0
    _run(c)


def test_chunk_of_a_prompt():
    c = make_cache([], [], [515, 700], 28, torch.bfloat16)
    _run(make_queries(c, [515, 300], 5, 29), groups=False)


def test_other_tables_and_streams():
    """Wider tables, and two calls at once on streams of their own."""
    cases = [make_queries(make_cache([384], [3], [9, 200, 40], 30 + i, torch.bfloat16, cols=40), [1, 1, 2], 16, 31 + i)
             for i in range(2)]
    ds = [{k: v.cuda() for k, v in c.items()} for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ds]
    for _ in range(4):
        for d, s in zip(ds, streams):
            with torch.cuda.stream(s):
                call_attention(d)
    torch.cuda.synchronize()
    for c, d in zip(cases, ds):
        check_attention(d["out"].cpu(), c)


def test_replays():
    """Two captured calls, replayed in turn on other lengths and groups, with
    eager work between them."""
    c = make_queries(make_cache([512], [4], [100, 90, 80, 70], 32, torch.bfloat16), [1, 1, 1, 1], 16, 33)
    d = {k: v.cuda() for k, v in c.items()}
    e = {k: v.clone() for k, v in d.items()}
    call_attention(d)
    torch.cuda.synchronize()
    graphs = []
    for s in (d, e):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call_attention(s)
        graphs.append(graph)
    for i in range(4):
        lengths = i32([512 + 100 - 9 * i, 512 + i, 600, 512])
        prefix = i32([512 if i % 2 else 0])
        for s, graph in zip((d, e), graphs):
            s["lengths"].copy_(lengths)
            s["prefix"].copy_(prefix)
            s["out"].fill_(7.0)
            torch.cuda.synchronize()
            graph.replay()
            (s["query"].float().sum() + 1).item()
            torch.cuda.synchronize()
            check_attention(s["out"].cpu(), {**c, "lengths": lengths})


def test_same_call_twice_is_the_same():
    c = make_queries(make_cache([2048], [12], [30 * i + 1 for i in range(12)], 34, torch.bfloat16), [1] * 12, 64, 35)
    d = {k: v.cuda() for k, v in c.items()}
    call_attention(d)
    first = d["out"].clone()
    for _ in range(3):
        d["out"].fill_(7.0)
        call_attention(d)
        assert torch.equal(d["out"], first)
