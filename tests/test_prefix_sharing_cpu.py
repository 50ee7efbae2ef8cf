"""The prefix-sharing operators without a GPU: refusals of the C ABI, the
operators' registration, and the oracle's own rules."""

from __future__ import annotations

import ctypes
import random

import pytest
import torch

from _prefix import PAGE, i32, make_cache, make_pages, make_queries
from oracle import prefix_oracle as O

BF16, F16, I32, F32 = 2, 1, 0, 3


def _desc(shape, dtype, device=0, contiguous=1, data=0x1000):
    from nanovllm_amd import _lib

    assert (_lib.INT32, _lib.FLOAT16, _lib.BFLOAT16, _lib.FLOAT32) == (I32, F16, BF16, F32)
    d = _lib.NvdsaTensor()
    d.data, d.dtype, d.ndim, d.contiguous, d.device = data, dtype, len(shape), contiguous, device
    for i, s in enumerate(shape):
        d.shape[i] = s
    return d


def _ref(d):
    return None if d is None else ctypes.byref(d)


def _lib():
    from nanovllm_amd import _lib as L

    return L


def _paged(B=2, C=3, blocks=7):
    return {"ends": _desc((B,), I32), "lengths": _desc((B,), I32), "table": _desc((B, C), I32),
            "k_rope": _desc((blocks, 128, 1, 64), BF16), "kv_cache": _desc((blocks, 128, 1, 512), BF16)}


def _norm_args(T=5, N=4, nope=128):
    return {**_paged(), "query": _desc((T, N, nope + 64), BF16), "kv": _desc((T, 576), BF16), "cos": _desc((T, 64), BF16),
            "sin": _desc((T, 64), BF16), "kv_weight": _desc((512,), BF16), "query_rope": _desc((T, N, 64), BF16),
            "query_weight": _desc((nope + 64,), BF16), "query_nope": _desc((T, N, nope), BF16)}


def _norm(a, eps=1e-6):
    order = ("query", "kv", "cos", "sin", "kv_weight", "ends", "lengths", "table", "k_rope", "kv_cache", "query_rope",
             "query_weight", "query_nope")
    return _lib().lib.nvdsa_norm_rope_append(*[_ref(a[k]) for k in order], eps, None), _lib().last_error()


def _attention_args(T=5, N=4, S=2):
    return {**_paged(), "query": _desc((T, N, 512), BF16), "query_rope": _desc((T, N, 64), BF16),
            "out": _desc((T, N, 512), BF16), "group_ends": _desc((S,), I32), "prefix": _desc((S,), I32)}


def _attention(a, ws=0x1000, nbytes=1 << 50):
    x = [_ref(a[k]) for k in ("query_rope", "query", "ends", "lengths", "table", "k_rope", "kv_cache")]
    y = [_ref(a[k]) for k in ("out", "group_ends", "prefix")]
    return _lib().lib.nvdsa_shared_prefix_attention(*x, 0.1, *y, ws, nbytes, None), _lib().last_error()


def _branch_args(B=2, C=3, P=7):
    vectors = {k: _desc((B,), I32) for k in ("lengths", "new", "src", "dst", "tokens", "parents")}
    return {**vectors, "table": _desc((B, C), I32), "refs": _desc((P,), I32), "missing": _desc((1,), I32)}


def _branch(a, ws=0x1000, nbytes=1 << 40):
    order = ("lengths", "new", "table", "refs", "src", "dst", "tokens", "missing", "parents")
    return _lib().lib.nvdsa_pages_branch(*[_ref(a[k]) for k in order], ws, nbytes, None), _lib().last_error()


def _compact_args(B=2, C=3, P=7):
    return {"table": _desc((B, C), I32), "refs": _desc((P,), I32), "src": _desc((P,), I32), "dst": _desc((P,), I32),
            "count": _desc((1,), I32)}


def _compact(a, ws=0x1000, nbytes=1 << 40):
    order = ("table", "refs", "src", "dst", "count")
    return _lib().lib.nvdsa_pages_compact(*[_ref(a[k]) for k in order], ws, nbytes, None), _lib().last_error()


def _copy_args(P=7, pairs=3):
    return {"src": _desc((pairs,), I32), "dst": _desc((pairs,), I32), "tokens": _desc((pairs,), I32),
            "count": _desc((1,), I32), "cache": _desc((P, 128, 1, 512), BF16), "other": _desc((P, 128, 1, 64), BF16)}


def _copy(a, n=2):
    caches = (_lib().NvdsaTensor * 2)(a["cache"], a["other"])
    return _lib().lib.nvdsa_pages_copy(_ref(a["src"]), _ref(a["dst"]), caches, n, _ref(a["tokens"]), _ref(a["count"]),
                                       None), _lib().last_error()


def _set(name, field, value):
    return lambda a: setattr(a[name], field, value)


def _shape(name, i, value):
    return lambda a: a[name].shape.__setitem__(i, value)


def _none(*names):
    return lambda a: a.update({n: None for n in names})


def _refused(call, args, mutate, code, msg):
    mutate(args)
    got, text = call(args)
    assert got == code and msg in text, (got, text)


PAGED_FAULTS = [
    (_set("kv_cache", "ndim", 3), 1, "kv_cache"),
    (_shape("kv_cache", 1, 64), 1, "kv_cache"),
    (_shape("kv_cache", 2, 2), 1, "kv_cache"),
    (_shape("kv_cache", 3, 576), 1, "kv_cache"),
    (_shape("kv_cache", 0, 6), 1, "k_rope"),
    (_shape("k_rope", 3, 128), 1, "k_rope"),
    (_set("k_rope", "dtype", F16), 2, "16-bit dtype"),
    (_set("kv_cache", "dtype", F32), 2, "16-bit dtype"),
    (_shape("table", 0, 3), 1, "block_table must be"),
    (_shape("table", 1, 0), 1, "block_table must be"),
    (_shape("table", 1, (1 << 14) + 1), 1, "<= 16384"),
    (_set("table", "dtype", F32), 2, "block_table must be int32"),
    (_set("ends", "ndim", 2), 1, "actual_seq_lengths_query"),
    (_shape("lengths", 0, 3), 1, "actual_seq_lengths_kv"),
    (_set("lengths", "dtype", F32), 2, "must be int32"),
    (_set("kv_cache", "contiguous", 0), 3, "contiguous"),
    (_set("table", "contiguous", 0), 3, "contiguous"),
    (_set("k_rope", "data", 0x1008), 3, "16-byte aligned"),
    (_set("ends", "device", 1), 4, "same device"),
    (_set("kv_cache", "device", -1), 4, "device"),
    (_set("kv_cache", "data", None), 7, "null data"),
    (_none("table"), 7, "null tensor"),
]


@pytest.mark.parametrize("mutate,code,msg", PAGED_FAULTS + [
    (_none("query_weight"), 7, "go together"),
    (_none("query_nope"), 7, "go together"),
    (_shape("query", 2, 60), 1, "query must be"),
    (_shape("query", 2, 196), 1, "query must be"),
    (_shape("query", 2, 640), 1, "query must be"),
    (_shape("query", 1, 0), 1, "query must be"),
    (_shape("query", 1, 1025), 1, "query must be"),
    (_shape("query", 0, 1 << 24), 1, "too many rows"),
    (_shape("kv", 1, 512), 1, "kv must be"),
    (_shape("kv", 0, 4), 1, "kv must be"),
    (_shape("cos", 1, 32), 1, "cos and sin"),
    (_shape("sin", 0, 4), 1, "cos and sin"),
    (_shape("kv_weight", 0, 576), 1, "kv_norm_weight"),
    (_shape("query_weight", 0, 128), 1, "query_norm_weight"),
    (_shape("query_nope", 2, 192), 1, "query_nope"),
    (_shape("query_rope", 1, 5), 1, "query_rope"),
    (_set("kv", "dtype", F16), 2, "kv_cache's dtype"),
    (_set("query_weight", "dtype", F32), 2, "kv_cache's dtype"),
    (_set("query_nope", "data", 0x1004), 3, "16-byte aligned"),
    (_set("query_nope", "contiguous", 0), 3, "contiguous"),
    (_set("query_weight", "device", 1), 4, "same device"),
])
def test_norm_rope_append_refuses(mutate, code, msg):
    _refused(_norm, _norm_args(), mutate, code, msg)


@pytest.mark.parametrize("eps", [-1e-9, 1.5, float("nan")])
def test_norm_rope_append_refuses_eps(eps):
    code, text = _norm(_norm_args(), eps)
    assert code == 7 and "eps" in text


@pytest.mark.parametrize("mutate,code,msg", PAGED_FAULTS + [
    (_none("group_ends"), 7, "go together"),
    (_none("prefix"), 7, "go together"),
    (_shape("query", 2, 576), 1, "query must be"),
    (_shape("query", 1, 1025), 1, "query_rope must be"),
    (_shape("query_rope", 2, 32), 1, "query_rope must be"),
    (_shape("query_rope", 0, 4), 1, "query_rope must be"),
    (_shape("out", 1, 5), 1, "attention_out"),
    (_shape("prefix", 0, 3), 1, "prefix_lengths"),
    (_shape("group_ends", 0, 65537), 1, "at most 65536 groups"),
    (_set("group_ends", "dtype", F32), 2, "must be int32"),
    (_set("query", "dtype", F16), 2, "kv_cache's dtype"),
    (_set("out", "dtype", F32), 2, "kv_cache's dtype"),
    (_set("out", "data", 0x1002), 3, "16-byte aligned"),
    (_set("out", "contiguous", 0), 3, "contiguous"),
    (_set("prefix", "device", 1), 4, "same device"),
])
def test_shared_prefix_attention_refuses(mutate, code, msg):
    _refused(_attention, _attention_args(), mutate, code, msg)


def test_shared_prefix_attention_refuses_heads_and_rows():
    for T, N, msg in ((5, 1025, "1024 heads"), (1 << 20, 4, "too many query rows"), (1 << 17, 512, "too many query rows")):
        code, text = _attention(_attention_args(T, N))
        assert code == 1 and msg in text, (T, N, text)


def test_shared_prefix_attention_needs_its_workspace():
    size = _lib().lib.nvdsa_shared_prefix_attention_workspace_size(5, 4, 2, 2)
    assert size > 0
    for ws, nbytes in ((None, 1 << 40), (0x1000, size - 1), (0x1000, 0)):
        code, text = _attention(_attention_args(), ws, nbytes)
        assert code != 0 and "workspace too small" in text
    assert _lib().lib.nvdsa_shared_prefix_attention_workspace_size(-1, 4, 2, 2) == 0
    # It grows with every argument, and holds two sums of every pair of a small call.
    sizes = [_lib().lib.nvdsa_shared_prefix_attention_workspace_size(r, h, b, g)
             for r, h, b, g in ((1, 1, 1, 0), (5, 1, 1, 0), (5, 64, 1, 0), (5, 64, 5, 0), (5, 64, 5, 9))]
    assert sizes == sorted(sizes)
    assert sizes[-1] >= 2 * 5 * 64 * 512 * 4


def test_calls_without_rows_do_nothing():
    assert _attention(_attention_args(T=0), None, 0)[0] == 0


PAGES_FAULTS = [
    (_set("table", "ndim", 1), 1, "block_table must be"),
    (_shape("table", 1, 0), 1, "block_table must be"),
    (_shape("table", 1, (1 << 14) + 1), 1, "<= 16384"),
    (_shape("table", 0, (1 << 14) + 1), 1, "at most 16384"),
    (_shape("refs", 0, 0), 1, "page_refs must be"),
    (_shape("refs", 0, 1 << 24), 1, "page_refs must be"),
    (_set("refs", "dtype", F32), 2, "must be int32"),
    (_set("table", "contiguous", 0), 3, "contiguous"),
    (_set("table", "device", 1), 4, "same device"),
    (_set("refs", "device", -1), 4, "device"),
    (_none("table"), 7, "null tensor"),
]


@pytest.mark.parametrize("mutate,code,msg", PAGES_FAULTS + [
    (_shape("lengths", 0, 3), 1, "seq_lens must be"),
    (_shape("new", 0, 1), 1, "new_tokens must be"),
    (_shape("src", 0, 1), 1, "copy_src must be"),
    (_shape("dst", 0, 1), 1, "copy_dst must be"),
    (_shape("tokens", 0, 1), 1, "copy_tokens must be"),
    (_shape("missing", 0, 2), 1, "missing must be"),
    (_shape("parents", 0, 3), 1, "parents must be"),
    (_set("parents", "dtype", F32), 2, "must be int32"),
    (_set("parents", "device", 1), 4, "same device"),
])
def test_pages_branch_refuses(mutate, code, msg):
    _refused(_branch, _branch_args(), mutate, code, msg)


@pytest.mark.parametrize("mutate,code,msg", PAGES_FAULTS + [
    (_shape("src", 0, 6), 1, "move_src must be"),
    (_shape("dst", 0, 8), 1, "move_dst must be"),
    (_shape("count", 0, 2), 1, "move_count must be"),
    (_set("src", "dtype", F32), 2, "must be int32"),
])
def test_pages_compact_refuses(mutate, code, msg):
    _refused(_compact, _compact_args(), mutate, code, msg)


def test_page_operators_need_their_workspace():
    for call, args, size in ((_branch, _branch_args, _lib().lib.nvdsa_pages_branch_workspace_size(7)),
                             (_compact, _compact_args, _lib().lib.nvdsa_pages_compact_workspace_size(7))):
        assert size > 0
        for ws, nbytes in ((None, 1 << 30), (0x1000, size - 1)):
            code, text = call(args(), ws, nbytes)
            assert code != 0 and "workspace too small" in text


@pytest.mark.parametrize("mutate,code,msg", [
    (_set("src", "ndim", 2), 1, "src_ids must be"),
    (_shape("src", 0, 1 << 24), 1, "src_ids must be"),
    (_shape("dst", 0, 2), 1, "dst_ids must be"),
    (_shape("tokens", 0, 2), 1, "tokens must be"),
    (_shape("count", 0, 3), 1, "count must be"),
    (_set("dst", "dtype", F32), 2, "must be int32"),
    (_set("src", "device", -1), 4, "device"),
    (_set("count", "device", 1), 4, "same device"),
    (_shape("other", 0, 6), 1, "same number of pages"),
    (_shape("cache", 0, 0), 1, "caches must be"),
    (_set("cache", "ndim", 1), 1, "caches must be"),
    (_set("cache", "ndim", 5), 1, "caches must be"),
    (_set("other", "dtype", 77), 2, "caches must be"),
    (_set("other", "contiguous", 0), 3, "contiguous"),
    (_set("other", "device", 1), 4, "same device"),
    (_set("other", "data", None), 7, "null data"),
    (_set("cache", "data", 0x1002), 3, "multiples of 4 bytes"),
    (_shape("cache", 3, 1 << 24), 3, "below 1 GiB"),
    (_shape("other", 3, 3), 3, "multiples of 4 bytes"),
    (_none("src"), 7, "null tensor"),
])
def test_pages_copy_refuses(mutate, code, msg):
    _refused(_copy, _copy_args(), mutate, code, msg)


@pytest.mark.parametrize("n", [0, -1, 17])
def test_pages_copy_refuses_a_number_of_caches(n):
    from nanovllm_amd import prefix_sharing

    code, text = _copy(_copy_args(), n)
    assert code == 7 and "1 to 16 caches" in text
    with pytest.raises(RuntimeError, match="1 to 16 caches"):
        prefix_sharing._pages_copy(i32([0]), i32([1]), [torch.zeros(2, 128, 4)] * max(n, 0))


def test_operators_are_registered():
    from nanovllm_amd import prefix_sharing

    for name, schema in prefix_sharing.SCHEMAS.items():
        op = getattr(torch.ops.nanovllm_dsa, name).default
        assert str(op._schema).startswith(f"nanovllm_dsa::{name}(")
        outputs = [a.name for a in op._schema.arguments if a.alias_info is not None and a.alias_info.is_write]
        assert outputs, schema
        assert callable(getattr(prefix_sharing, name)) and name in prefix_sharing.__all__


def test_cpu_tensors_are_refused():
    from nanovllm_amd import prefix_sharing

    c = make_queries(make_cache([128], [2], [1, 2], 1, torch.bfloat16), [1, 1], 4, 1)
    with pytest.raises((RuntimeError, NotImplementedError)):
        prefix_sharing.shared_prefix_attention(c["query_rope"], c["query"], c["ends"], c["lengths"], c["table"],
                                               c["k_rope"], c["kv_cache"], 0.1, c["out"])


def test_meta_calls_return_nothing():
    c = make_queries(make_cache([128], [2], [1, 2], 1, torch.bfloat16), [1, 1], 4, 1)
    m = {k: v.to("meta") for k, v in c.items()}
    from nanovllm_amd import prefix_sharing

    assert prefix_sharing.shared_prefix_attention(m["query_rope"], m["query"], m["ends"], m["lengths"], m["table"],
                                                  m["k_rope"], m["kv_cache"], 0.1, m["out"]) is None
    assert prefix_sharing.pages_copy(m["ends"], m["lengths"], [m["kv_cache"], m["k_rope"]]) is None


def test_outputs_count_as_written(monkeypatch):
    """Autograd refuses a backward pass through values that a call overwrote,
    and only outputs count as written."""
    from contextlib import nullcontext
    from types import SimpleNamespace

    from nanovllm_amd import prefix_sharing as P

    calls = {f"nvdsa_{n}": lambda *a: 0 for n in P.SCHEMAS}
    monkeypatch.setattr(P, "_C", SimpleNamespace(**calls))
    monkeypatch.setattr(P, "_device_of", lambda t: nullcontext())
    monkeypatch.setattr(P, "_stream_of", lambda t: 0)
    c = make_queries(make_cache([128], [2], [1, 2], 1, torch.bfloat16), [1, 1], 4, 1)
    c.update({k: i32([0] * n) for k, n in (("lens", 2), ("new", 2), ("src", 2), ("dst", 2), ("tokens", 2), ("missing", 1),
                                            ("refs", 5), ("msrc", 5), ("mdst", 5), ("count", 1))})
    c.update({k: torch.zeros(*s, dtype=torch.bfloat16) for k, s in (
        ("q", (2, 4, 192)), ("kv", (2, 576)), ("cos", (2, 64)), ("sin", (2, 64)), ("w", (512,)), ("qw", (192,)),
        ("nope", (2, 4, 128)), ("turned", (2, 4, 64)))})

    def written(call):
        before = {k: v._version for k, v in c.items()}
        call()
        return {k for k, v in c.items() if v._version > before[k]}

    norm = [c[k] for k in ("q", "kv", "cos", "sin", "w", "ends", "lengths", "table", "k_rope", "kv_cache", "turned")]
    assert written(lambda: P._norm_rope_append(*norm)) == {"k_rope", "kv_cache", "turned"}
    assert written(lambda: P._norm_rope_append(*norm, c["qw"], c["nope"])) == {"k_rope", "kv_cache", "turned", "nope"}
    attend = [c[k] for k in ("query_rope", "query", "ends", "lengths", "table", "k_rope", "kv_cache")]
    assert written(lambda: P._shared_prefix_attention(*attend, 0.1, c["out"], c["group_ends"], c["prefix"])) == {"out"}
    branch = [c[k] for k in ("lens", "new", "table", "refs", "src", "dst", "tokens", "missing")]
    assert written(lambda: P._pages_branch(*branch)) == {"lens", "table", "refs", "src", "dst", "tokens", "missing"}
    compact = [c[k] for k in ("table", "refs", "msrc", "mdst", "count")]
    assert written(lambda: P._pages_compact(*compact)) == {"table", "refs", "msrc", "mdst", "count"}
    assert written(lambda: P._pages_copy(c["src"], c["dst"], [c["kv_cache"], c["k_rope"]])) == {"kv_cache", "k_rope"}


# ------------------------------------------------------------------ the oracle
def test_oracle_attention_is_softmax_over_the_slots():
    c = make_queries(make_cache([256], [2], [5, 40], 3, torch.float16), [2, 1], 3, 4)
    out, _, _ = O.attention(c["query_rope"], c["query"], c["ends"], c["lengths"], c["table"], c["k_rope"], c["kv_cache"], 0.05)
    for t, b, sees in ((0, 0, 260), (1, 0, 261), (2, 1, 296)):
        page = [int(c["table"][b, s // PAGE]) for s in range(sees)]
        k = torch.stack([torch.cat([c["kv_cache"][p, s % PAGE, 0], c["k_rope"][p, s % PAGE, 0]]) for s, p in enumerate(page)]).double()
        for h in range(3):
            q = torch.cat([c["query"][t, h], c["query_rope"][t, h]]).double()
            w = (k @ q * 0.05).exp()
            want = (w[:, None] * k[:, :512]).sum(0) / w.sum()
            assert torch.allclose(out[t, h], want, rtol=1e-9, atol=1e-12)


@pytest.mark.parametrize("seed", range(4))
def test_oracle_branch_keeps_its_counts(seed):
    """Counts are the entries that name a page, rows own what they write to, and
    nobody's older rows are lost."""
    rng = random.Random(seed)
    lengths = [rng.randrange(0, 5 * PAGE) for _ in range(9)]
    table, refs = make_pages(lengths, 90, 6, seed)
    parents = [rng.randrange(-1, 9) for _ in range(9)]
    new = [rng.choice([0, 1, 130]) for _ in range(9)]
    cache = torch.arange(90 * PAGE).view(90, PAGE, 1).clone()
    old = lambda t, n: [int(cache[t[s // PAGE], s % PAGE, 0]) for s in range(n)]  # noqa: E731
    want = [old(table[p], lengths[p]) if p >= 0 else [] for p in parents]
    lens2, table2, refs2, copies, missing = O.branch(lengths, new, table, refs, parents)
    assert missing == 0
    counts = [0] * 90
    for row in table2:
        for p in row:
            if p >= 0:
                counts[p] += 1
    assert counts == refs2
    O.copy(cache, [c[:2] for c in copies], [c[2] for c in copies])
    assert [old(t, n) for t, n in zip(table2, lens2)] == want
    for row, length, n in zip(table2, lens2, new):
        for c in range(length // PAGE, -(-min(length + n, 6 * PAGE) // PAGE) if n else 0):
            assert refs2[row[c]] == 1


def test_oracle_compact_keeps_every_row():
    table, refs = make_pages([300, 500, 0, 129], 40, 6, 5)
    cache = torch.arange(40 * PAGE).view(40, PAGE, 1).clone()
    before = [[cache[p].clone() for p in row if p >= 0] for row in table]
    table2, refs2, moves = O.compact(table, refs)
    O.copy(cache, moves)
    live = sum(r > 0 for r in refs)
    assert all(r > 0 for r in refs2[:live]) and not any(refs2[live:])
    for row, pages in zip(table2, before):
        assert all(torch.equal(cache[p], x) for p, x in zip([p for p in row if p >= 0], pages))
