"""The prefix-sharing operators as a decode step uses them: requests branch,
pages are copied, rows appended and attended, and the cache is compacted, on the
GPU beside the oracle on the CPU."""

from __future__ import annotations

import random

import pytest
import torch

from _prefix import HALF_STEP, PAGE, SCALE, api, call_attention, check_attention, i32, make_cache, make_queries
from oracle import prefix_oracle as O

pytestmark = pytest.mark.gpu

HEADS, LAYERS, NOPE = 16, 2, 128


class Serving:
    """Buffers of a batch whose requests continue a prompt of ``prompt`` tokens,
    request 0's; the others are empty until they branch."""

    def __init__(self, batch, prompt, pages, cols, dtype, seed):
        g = torch.Generator().manual_seed(seed)
        self.g, self.dtype, self.batch = g, dtype, batch
        rand = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
        held = -(-prompt // PAGE)
        order = torch.randperm(pages, generator=g).tolist()
        self.table = [order[:held] + [-1] * (cols - held)] + [[-1] * cols for _ in range(batch - 1)]
        self.refs = [0] * pages
        for p in order[:held]:
            self.refs[p] = 1
        self.lens = [prompt] + [0] * (batch - 1)
        self.caches = [(rand(pages, PAGE, 1, 512), rand(pages, PAGE, 1, 64)) for _ in range(LAYERS)]
        self.weights = [((1 + 0.3 * torch.randn(512, generator=g)).to(dtype), (1 + 0.3 * torch.randn(NOPE + 64, generator=g)).to(dtype))
                        for _ in range(LAYERS)]
        i = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
        self.d = {"table": i32(self.table).cuda(), "refs": i32(self.refs).cuda(), "lens": i32(self.lens).cuda(),
                  "lengths": i(batch), "new": i(batch), "ends": i(batch), "parents": i(batch), "src": i(batch), "dst": i(batch),
                  "tokens": i(batch), "missing": i(1), "msrc": i(pages), "mdst": i(pages), "count": i(1),
                  "group_ends": i32([batch]).cuda(), "prefix": i32([0]).cuda()}
        self.d_caches = [(a.cuda(), b.cuda()) for a, b in self.caches]
        self.d_weights = [(a.cuda(), b.cuda()) for a, b in self.weights]

    def rows(self, new):
        """A step's projections and angles, for every layer."""
        total = sum(new)
        rand = lambda *s: torch.randn(*s, generator=self.g).to(self.dtype)  # noqa: E731
        angle = (torch.rand(total, 32, generator=self.g) * 6.283).repeat_interleave(2, 1)
        return [{"query": rand(total, HEADS, NOPE + 64), "latent": 2 * rand(total, HEADS, 512), "kv": rand(total, 576),
                 "cos": angle.cos().to(self.dtype), "sin": angle.sin().to(self.dtype)} for _ in range(LAYERS)]

    def outputs(self, rows):
        total = rows[0]["query"].shape[0]
        return [{**{k: v.cuda() for k, v in r.items()},
                 "query_rope": torch.zeros(total, HEADS, 64, dtype=self.dtype, device="cuda"),
                 "query_nope": torch.zeros(total, HEADS, NOPE, dtype=self.dtype, device="cuda"),
                 "out": torch.zeros(total, HEADS, 512, dtype=self.dtype, device="cuda")} for r in rows]

    def set_step(self, new, parents, prefix):
        d = self.d
        d["new"].copy_(i32(new))
        d["ends"].copy_(i32(new).cumsum(0))
        d["parents"].copy_(i32(parents))
        d["prefix"].copy_(i32([prefix]))

    def step(self, layers):
        d, p = self.d, api()
        p.pages_branch(d["lens"], d["new"], d["table"], d["refs"], d["src"], d["dst"], d["tokens"], d["missing"],
                       parents=d["parents"])
        p.pages_copy(d["src"], d["dst"], [c for pair in self.d_caches for c in pair], tokens=d["tokens"])
        torch.add(d["lens"], d["new"], out=d["lengths"])
        for (kv_cache, k_rope), (kv_weight, query_weight), r in zip(self.d_caches, self.d_weights, layers):
            p.norm_rope_append(r["query"], r["kv"], r["cos"], r["sin"], kv_weight, d["ends"], d["lengths"], d["table"],
                               k_rope, kv_cache, r["query_rope"], query_norm_weight=query_weight, query_nope=r["query_nope"])
            p.shared_prefix_attention(r["query_rope"], r["latent"], d["ends"], d["lengths"], d["table"], k_rope, kv_cache,
                                      SCALE, r["out"], prefix_request_ends=d["group_ends"], prefix_lengths=d["prefix"])
        d["lens"].copy_(d["lengths"])

    def check(self, new, parents, rows, layers):
        """The oracle's step from the state before, against what the GPU left."""
        self.lens, self.table, self.refs, copies, missing = O.branch(self.lens, new, self.table, self.refs, parents)
        assert missing == 0 and self.d["missing"].item() == 0
        assert self.d["table"].tolist() == self.table and self.d["refs"].tolist() == self.refs
        lengths = [a + n for a, n in zip(self.lens, new)]
        assert self.d["lens"].tolist() == lengths
        table, ends = i32(self.table), i32(new).cumsum(0).to(torch.int32)
        for layer, (r, got) in enumerate(zip(rows, layers)):
            kv_cache, k_rope = self.caches[layer]
            for cache in (kv_cache, k_rope):
                O.copy(cache, [c[:2] for c in copies], [c[2] for c in copies])
            kv_weight, query_weight = self.weights[layer]
            put, rope, nope = O.norm_rope(r["query"], r["kv"], r["cos"], r["sin"], kv_weight, ends, i32(lengths), table,
                                          query_weight, 1e-6)
            new_kv, new_rope = (c.cpu() for c in self.d_caches[layer])
            off = HALF_STEP[self.dtype] + 2.0 ** -13
            for (page, row), (latent, turned) in put.items():
                assert ((new_kv[page, row, 0].double() - latent).abs() <= latent.abs() * off + 2.0 ** -24).all()
                size = turned.abs() + turned.unflatten(-1, (-1, 2)).flip(-1).flatten(-2).abs()
                assert ((new_rope[page, row, 0].double() - turned).abs() <= turned.abs() * off + size * 2.0 ** -20 + 2.0 ** -24).all()
                # The rows as they were stored: what the attention and the next steps read.
                kv_cache[page, row], k_rope[page, row] = new_kv[page, row], new_rope[page, row]
            # Every page that somebody holds is the same, byte for byte.
            for p, holders in enumerate(self.refs):
                if holders > 0:
                    assert torch.equal(new_kv[p].view(torch.int16), kv_cache[p].view(torch.int16)), (layer, p)
                    assert torch.equal(new_rope[p].view(torch.int16), k_rope[p].view(torch.int16)), (layer, p)
            turned_q = got["query_rope"].cpu()
            c = {"query": r["latent"], "query_rope": turned_q, "ends": ends, "lengths": i32(lengths), "table": table,
                 "kv_cache": kv_cache, "k_rope": k_rope, "out": torch.zeros_like(r["latent"])}
            check_attention(got["out"].cpu(), c)
        self.lens = lengths

    def compact(self):
        d, p = self.d, api()
        p.pages_compact(d["table"], d["refs"], d["msrc"], d["mdst"], d["count"])
        p.pages_copy(d["msrc"], d["mdst"], [c for pair in self.d_caches for c in pair], count=d["count"])
        self.table, self.refs, moves = O.compact(self.table, self.refs)
        assert d["table"].tolist() == self.table and d["refs"].tolist() == self.refs
        assert d["count"].item() == len(moves)
        for pair in self.caches:
            for cache in pair:
                O.copy(cache, moves)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_sampling_from_one_prompt(dtype):
    """Eight continuations of one prompt: all take it over, go on, are replaced
    by the better ones, and the cache is brought together in between."""
    rng = random.Random(7)
    s = Serving(8, 700, 64, 9, dtype, 5)
    parents, prefix = [0] * 8, 640
    for step in range(5):
        new = [1] * 8 if step != 3 else [1, 2, 1, 4, 1, 1, 3, 1]  # (drafted tokens)
        print(f"TOGETHER {dtype} step {step}", flush=True)
        rows = s.rows(new)
        layers = s.outputs(rows)
        s.set_step(new, parents, prefix)
        s.step(layers)
        torch.cuda.synchronize()
        s.check(new, parents, rows, layers)
        if step == 2:
            s.compact()
        parents = [rng.randrange(8) for _ in range(8)] if step % 2 == 0 else list(range(8))


def test_a_captured_step():
    """One graph of the whole step, replayed on other rows and parents, with
    eager work between."""
    s = Serving(6, 300, 40, 6, torch.bfloat16, 9)
    new, parents = [1] * 6, [0] * 6
    rows = s.rows(new)
    layers = s.outputs(rows)
    s.set_step(new, parents, 256)
    s.step(layers)
    torch.cuda.synchronize()
    s.check(new, parents, rows, layers)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.step(layers)
    for step in range(4):
        parents = [(i * 5 + step) % 6 for i in range(6)]
        rows = s.rows(new)
        for r, d in zip(rows, layers):
            for k, v in r.items():
                d[k].copy_(v)
        s.set_step(new, parents, 256 if step % 2 == 0 else 0)
        graph.replay()
        (s.d["lens"].sum() + 1).item()
        torch.cuda.synchronize()
        s.check(new, parents, rows, layers)


def test_offsets_past_32_bits():
    """Pages whose bytes lie behind 2^32 of the cache: rows, copies and attention."""
    pages, far = 33000, [32990, 32771, 32999, 1]
    kv_cache = torch.empty(pages, PAGE, 1, 512, dtype=torch.bfloat16, device="cuda")
    k_rope = torch.empty(pages, PAGE, 1, 64, dtype=torch.bfloat16, device="cuda")
    assert kv_cache.numel() * 2 > 1 << 32
    c = make_queries(make_cache([256], [2], [100, 60], 40, torch.bfloat16), [1, 2], 16, 41)
    small = sorted({p for row in c["table"].tolist() for p in row if p >= 0})
    to = dict(zip(small, far))
    assert len(small) == 4
    for p, q in to.items():
        kv_cache[q], k_rope[q] = c["kv_cache"][p].cuda(), c["k_rope"][p].cuda()
    d = {k: v.cuda() for k, v in c.items()}
    d["table"] = i32([[to.get(p, p) for p in row] for row in c["table"].tolist()]).cuda()
    attend = lambda table: api().shared_prefix_attention(  # noqa: E731
        d["query_rope"], d["query"], d["ends"], d["lengths"], table, k_rope, kv_cache, SCALE, d["out"],
        prefix_request_ends=d["group_ends"], prefix_lengths=d["prefix"])
    attend(d["table"])
    check_attention(d["out"].cpu(), c)
    dst = [32768, 32769, 32770, 2]
    api().pages_copy(i32(far).cuda(), i32(dst).cuda(), [kv_cache, k_rope])
    for a, b in zip(far, dst):
        assert torch.equal(kv_cache[a].view(torch.int16), kv_cache[b].view(torch.int16))
    moved = dict(zip(far, dst))
    d["out"].fill_(7.0)
    attend(i32([[moved.get(p, p) for p in row] for row in d["table"].tolist()]).cuda())
    check_attention(d["out"].cpu(), c)


def test_many_keys():
    """One row over 131072 slots, cut into as many parts as there are."""
    n = 131072
    c = make_queries(make_cache([], [], [n], 42, torch.bfloat16, size=0.5), [1], 2, 43, size=0.5)
    d = {k: v.cuda() for k, v in c.items()}
    call_attention(d, groups=False)
    check_attention(d["out"].cpu(), c)


@pytest.mark.parametrize("group_ends", [[4, 0, 4, 0, 4], [3, 1, 4], [-5, 99], [0, 0, 0], [4, 2, 4, 2, 4, 2, 4], [2, 4]])
def test_group_ends_in_any_order(group_ends):
    """Groups that overlap: a request counts with one at most, and is right."""
    c = make_queries(make_cache([512], [4], [9, 8, 7, 6], 44, torch.bfloat16), [1, 1, 1, 1], 64, 45)
    c["group_ends"], c["prefix"] = i32(group_ends), i32([512] * len(group_ends))
    d = {k: v.cuda() for k, v in c.items()}
    call_attention(d)
    check_attention(d["out"].cpu(), c)


def test_row_ends_that_decrease_stay_within_the_buffers():
    """Not allowed: rows of two requests, whose values nobody knows.  The rows of
    the first request alone are its own."""
    c = make_queries(make_cache([512], [4], [9, 8, 7, 6], 46, torch.bfloat16), [1, 1, 1, 1], 64, 47, pad=3)
    d = {k: v.cuda() for k, v in c.items()}
    d["ends"].copy_(i32([2, 1, 4, 4]))
    call_attention(d)
    torch.cuda.synchronize()
    assert (d["out"][4:] == 7.0).all() and not d["out"][:4].isnan().any()
