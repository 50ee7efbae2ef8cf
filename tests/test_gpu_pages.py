"""Branching, compacting and copying of pages on the GPU vs the oracle's lists,
every integer and every byte."""

from __future__ import annotations

import random

import pytest
import torch

from _prefix import PAGE, api, i32, make_pages
from oracle import prefix_oracle as O

pytestmark = pytest.mark.gpu


def _branch(lengths, new, table, refs, parents=None):
    d = {"lens": i32(lengths), "new": i32(new), "table": i32(table), "refs": i32(refs)}
    d = {k: v.cuda() for k, v in d.items()}
    out = [torch.full((len(lengths),), 99, dtype=torch.int32, device="cuda") for _ in range(3)]
    missing = torch.full((1,), 99, dtype=torch.int32, device="cuda")
    api().pages_branch(d["lens"], d["new"], d["table"], d["refs"], *out, missing,
                       parents=None if parents is None else i32(parents).cuda())
    torch.cuda.synchronize()
    w_len, w_table, w_refs, copies, lack = O.branch(lengths, new, table, refs, parents)
    assert d["lens"].tolist() == w_len
    assert d["table"].tolist() == w_table
    assert d["refs"].tolist() == w_refs
    assert list(zip(*[o.tolist() for o in out])) == copies
    assert missing.item() == lack
    return d, out, missing


@pytest.mark.parametrize("parents", [None, [0, 0], [1, 0], [-1, 0], [1, 1], [-1, -1], [5, 0]])
@pytest.mark.parametrize("lengths", [[130, 260], [128, 0], [1, 127]])
def test_two_rows(lengths, parents):
    table, refs = make_pages(lengths, 9, 4, 1)
    print(f"BRANCH {lengths} {parents}", flush=True)
    _branch(lengths, [1, 1], table, refs, parents)
    _branch(lengths, [0, 300], table, refs, parents)


def test_shared_pages():
    """Shared full pages, a shared page of older rows with and without other
    holders, different lengths on one page, reserved pages ahead."""
    lengths = [300, 300, 290, 256, 300, 384]
    table, refs = make_pages(lengths, 24, 6, 2, shared=[(1, 0, 3), (2, 0, 3), (3, 0, 2), (4, 0, 3)])
    _branch(lengths, [1, 1, 1, 1, 1, 1], table, refs)
    _branch(lengths, [1, 1, 0, 1, 1, 1], table, refs)       # row 2 does not write: nobody keeps the page
    held = list(refs)
    held[table[0][2]] += 1                                  # somebody outside the table holds it
    _branch(lengths, [1] * 6, table, held)
    ahead = [list(r) for r in table]
    counts = list(refs)
    spare = [p for p, r in enumerate(refs) if r == 0]
    ahead[0][3] = ahead[1][3] = spare[0]                    # a page ahead of both rows
    counts[spare[0]] = 2
    _branch(lengths, [200, 200, 200, 1, 1, 300], ahead, counts)


def test_too_few_pages():
    lengths = [130, 260, 5]
    table, refs = make_pages(lengths, 7, 4, 3)
    _branch(lengths, [200, 200, 100], table, refs)          # takes the last one
    _branch(lengths, [200, 300, 200], table, refs)          # one short: nothing changes
    _branch(lengths, [200, 300, 200], table, refs, [0, 0, 0])


def test_lengths_that_name_nothing():
    table, refs = make_pages([130, 260, 5, 0], 16, 4, 4)
    table[0][1], table[1][0] = 99, -7
    _branch([-3, 4 * PAGE, 4 * PAGE - 1, 600], [4, 9, 9, 9], table, refs)
    _branch([130, 260, 5, 0], [-4, 2 ** 31 - 1, 0, 2 ** 31 - 1], table, refs, [0, 3, 3, 2 ** 31 - 1])


@pytest.mark.parametrize("seed", range(8))
def test_random(seed):
    rng = random.Random(seed)
    batch, cols = rng.choice([1, 3, 40, 300, 1500]), rng.choice([1, 5, 33])
    lengths = [rng.randrange(0, cols * PAGE + 1) for _ in range(batch)]
    shared = []
    for _ in range(batch // 2):
        b, o = rng.randrange(batch), rng.randrange(batch)
        n = min(lengths[b], lengths[o])
        if n > 0 and b != o:
            shared.append((b, o, -(-n // PAGE)))
    held = sum(-(-n // PAGE) for n in lengths)
    table, refs = make_pages(lengths, held + rng.choice([0, batch, 9000]), cols, seed, shared)
    for p in rng.sample(range(len(refs)), min(5, len(refs))):
        refs[p] += rng.randrange(2)
    print(f"BRANCH random {seed} {batch} {cols} {len(refs)}", flush=True)
    parents = rng.choice([None, [rng.randrange(-1, batch) for _ in range(batch)], list(range(batch))[::-1]])
    _branch(lengths, [rng.choice([0, 1, 1, 4, 150]) for _ in range(batch)], table, refs, parents)


def test_most_rows_and_many_pages():
    """16384 rows, and free pages that lie behind a million held ones."""
    batch = 16384
    table, refs = make_pages([i % 128 for i in range(batch)], batch + 4000, 1, 5)
    _branch([i % 128 for i in range(batch)], [1] * batch, table, refs, [i ^ 1 for i in range(batch)])
    refs = [1] * 1_000_003
    refs[1_000_001] = 0
    refs[999_999] = 0
    table = [[5, -1], [6, -1]]
    _branch([128, 128], [1, 1], table, refs)
    _branch([128, 128], [1, 129], table, refs)


def _compact(table, refs):
    t, r = i32(table).cuda(), i32(refs).cuda()
    src, dst = (torch.full((len(refs),), -5, dtype=torch.int32, device="cuda") for _ in range(2))
    count = torch.full((1,), 99, dtype=torch.int32, device="cuda")
    api().pages_compact(t, r, src, dst, count)
    torch.cuda.synchronize()
    w_table, w_refs, moves = O.compact(table, refs)
    assert t.tolist() == w_table
    assert r.tolist() == w_refs
    n = len(moves)
    assert count.item() == n
    assert list(zip(src.tolist(), dst.tolist())) == moves + [(-5, -5)] * (len(refs) - n)
    return t, r, src, dst, count


@pytest.mark.parametrize("pages,lengths", [(1, [0]), (1, [5]), (7, [130, 260]), (300, [1000] * 8), (4096, [5000] * 40),
                                           (4097, [128 * 2048, 128 * 2049]), (9000, [30000] * 20), (70000, [100] * 3000)])
def test_compact(pages, lengths):
    cols = max(1, -(-max(lengths) // PAGE))
    table, refs = make_pages(lengths, pages, cols, pages)
    print(f"COMPACT {pages}", flush=True)
    _compact(table, refs)
    if len(lengths) > 1 and lengths[0]:
        table[1][0] = table[0][0]
        refs = [0] * len(refs)
        for row in table:
            for p in row:
                if p >= 0:
                    refs[p] += 1
        refs[-1] += 3      # a holder outside the table
        table[0][-1] = pages + 4
        _compact(table, refs)


def test_compact_without_rows():
    _compact([[-1]], [0, 2, 0, 1, 0, 0, 1])


def _caches(pages, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return [r(pages, PAGE, 1, 512).bfloat16(), r(pages, PAGE, 1, 64).bfloat16(), r(pages, PAGE, 1, 128).half(),
            r(pages, PAGE, 2, 576).to(torch.float8_e4m3fn), r(pages, 2), r(pages, 3), r(pages, PAGE, 2).bfloat16(),
            torch.arange(pages * 5, dtype=torch.int32).view(pages, 5), r(pages, 256)]


@pytest.mark.parametrize("tokens", [None, [0, 1, 127, 128, 500, -3, 64]])
@pytest.mark.parametrize("count", [None, 0, 3, 7, 99, -1])
def test_copy(tokens, count):
    caches = _caches(20, 3)
    pairs = [(0, 11), (1, 12), (2, 13), (3, 14), (0, 15), (4, 16), (19, 17)]
    print(f"COPY {tokens} {count}", flush=True)
    d = [c.cuda() for c in caches]
    api().pages_copy(i32([p[0] for p in pairs]).cuda(), i32([p[1] for p in pairs]).cuda(), d,
                     tokens=None if tokens is None else i32(tokens).cuda(), count=None if count is None else i32([count]).cuda())
    n = len(pairs) if count is None else min(max(count, 0), len(pairs))
    for c, got in zip(caches, d):
        O.copy(c, pairs[:n], tokens)
        assert torch.equal(got.cpu().view(torch.uint8), c.view(torch.uint8)), c.shape


def test_copy_skips_what_names_nothing():
    caches = _caches(9, 4)[:5]
    pairs = [(-1, 3), (2, -1), (9, 4), (1, 9), (5, 5), (0, 8)]
    d = [c.cuda() for c in caches]
    api().pages_copy(i32([p[0] for p in pairs]).cuda(), i32([p[1] for p in pairs]).cuda(), d)
    for c, got in zip(caches, d):
        O.copy(c, pairs)
        assert torch.equal(got.cpu().view(torch.uint8), c.view(torch.uint8))


def test_copy_of_many_pages():
    pages = 1500
    caches = [torch.randn(pages, PAGE, 1, 512, device="cuda").bfloat16(), torch.randn(pages, PAGE, 1, 64, device="cuda").bfloat16()]
    order = torch.randperm(pages).to(torch.int32)
    src, dst = order[:700].cuda(), order[700:1400].cuda()
    want = [c.clone() for c in caches]
    for w in want:
        w[dst.long()] = w[src.long()]
    api().pages_copy(src, dst, caches)
    for c, w in zip(caches, want):
        assert torch.equal(c, w)


def test_copy_on_unaligned_memory():
    """Views that begin 4 bytes into a 16-byte line take the narrow copy."""
    flat = torch.randn(9 * 64 + 1, device="cuda")
    cache = flat[1:].view(9, 64)
    want = cache.clone()
    want[7] = want[2]
    api().pages_copy(i32([2]).cuda(), i32([7]).cuda(), [cache])
    assert torch.equal(cache, want)


def test_replays():
    """A captured step (branch and copy), replayed on other tables."""
    lengths = [300, 300, 290]
    table, refs = make_pages(lengths, 24, 6, 2, shared=[(1, 0, 3)])
    t, r, lens, new, parents = (i32(v).cuda() for v in (table, refs, lengths, [1] * 3, [0, 0, 0]))
    src, dst, tokens = (torch.zeros(3, dtype=torch.int32, device="cuda") for _ in range(3))
    missing = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache = torch.randn(24, PAGE, 1, 64, device="cuda").bfloat16()

    def step():
        api().pages_branch(lens, new, t, r, src, dst, tokens, missing, parents=parents)
        api().pages_copy(src, dst, [cache], tokens=tokens)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for case in ([0, 0, 0], [2, 1, 0], [-1, 2, 2]):
        state = lengths, table, refs
        for x, v in zip((lens, t, r, parents), (*state, case)):
            x.copy_(i32(v).cuda())
        before = cache.cpu()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        w_len, w_table, w_refs, copies, lack = O.branch(lengths, [1] * 3, table, refs, case)
        assert (lens.tolist(), t.tolist(), r.tolist(), missing.item()) == (w_len, w_table, w_refs, lack)
        O.copy(before, [c[:2] for c in copies], [c[2] for c in copies])
        assert torch.equal(cache.cpu(), before)
