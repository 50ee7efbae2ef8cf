"""The 8-bit latent cache without a GPU: refusals of the C ABI, the
operators' registration, and the oracle's own rules."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from _latent8 import i32, make_cache, oracle_attention, queries, same_codes
from oracle import latent8_oracle as O

F8 = 4


def _desc(shape, dtype, device=0, contiguous=1, data=0x1000):
    from nanovllm_amd._lib import NvdsaTensor

    d = NvdsaTensor()
    d.data, d.dtype, d.ndim, d.contiguous, d.device = data, dtype, len(shape), contiguous, device
    for i, s in enumerate(shape):
        d.shape[i] = s
    return d


def _common(B=2, C=3, G=2, blocks=7):
    from nanovllm_amd._lib import FLOAT32, INT32

    return {"seq_q": _desc((B,), INT32), "seq_kv": _desc((B,), INT32), "table": _desc((B, C), INT32),
            "cache": _desc((blocks, 128, G, 576), F8), "scale": _desc((blocks, G), FLOAT32),
            "entries": _desc((B,), INT32), "positions_pool": _desc((5, C * 128), INT32),
            "weights_pool": _desc((5, C * 128), FLOAT32)}


def _append_args(T=4, G=2):
    from nanovllm_amd._lib import BFLOAT16, INT32

    return {**_common(G=G), "kv": _desc((T, G, 512), BFLOAT16), "rope": _desc((T, G, 64), BFLOAT16),
            "positions": _desc((T,), INT32)}


def _ref(d):
    return None if d is None else ctypes.byref(d)


def _append(a):
    from nanovllm_amd import _lib

    order = ("kv", "rope", "seq_q", "seq_kv", "table", "cache", "scale", "positions", "entries", "positions_pool",
             "weights_pool")
    return _lib.lib.nvdsa_latent8_append(*[_ref(a[k]) for k in order], None), _lib.last_error()


def _attention_args(T=4, N=8):
    from nanovllm_amd._lib import FLOAT16

    return {**_common(), "q": _desc((T, N, 512), FLOAT16), "qr": _desc((T, N, 64), FLOAT16), "topk": None,
            "out": _desc((T, N, 512), FLOAT16)}


def _attention(a, ws=0x1000, nbytes=None):
    from nanovllm_amd import _lib

    if nbytes is None:
        nbytes = 1 << 40
    order = ("qr", "q", "seq_q", "seq_kv", "table", "cache", "scale", "topk", "entries", "weights_pool")
    return _lib.lib.nvdsa_latent8_attention(*[_ref(a[k]) for k in order], 0.1, _ref(a["out"]), ws, nbytes, None), \
        _lib.last_error()


def _evict_args(B=2, C=3):
    from nanovllm_amd._lib import INT32

    return {**_common(B, C), "budgets": _desc((B,), INT32), "src": _desc((B, C * 128), INT32),
            "dst": _desc((B, C * 128), INT32), "counts": _desc((B,), INT32), "kept": _desc((B,), INT32)}


def _evict(a, first=0, last=0, ws=0x1000, nbytes=1 << 30):
    from nanovllm_amd import _lib

    x = [_ref(a[k]) for k in ("seq_kv", "budgets", "table", "entries", "cache", "scale", "positions_pool",
                              "weights_pool")]
    y = [_ref(a[k]) for k in ("src", "dst", "counts", "kept")]
    return _lib.lib.nvdsa_latent8_evict(*x, first, last, *y, ws, nbytes, None), _lib.last_error()


def _set(name, field, value):
    return lambda a: setattr(a[name], field, value)


def _shape(name, i, value):
    return lambda a: a[name].shape.__setitem__(i, value)


def _none(*names):
    return lambda a: a.update({n: None for n in names})


CACHE_FAULTS = [
    (_set("cache", "ndim", 3), 1, "latent_cache must be"),
    (_shape("cache", 0, 0), 1, "latent_cache must be"),
    (_shape("cache", 0, 1 << 24), 1, "too many blocks"),
    (_shape("cache", 1, 64), 1, "latent_cache must be"),
    (_shape("cache", 3, 512), 1, "latent_cache must be"),
    (_set("cache", "dtype", 2), 2, "float8_e4m3fn"),
    (_shape("scale", 1, 1), 1, "cache_scale must be"),
    (_set("scale", "dtype", 2), 2, "cache_scale must be float32"),
    (_shape("table", 0, 3), 1, "block_table must be"),
    (_shape("table", 1, 0), 1, "block_table must be"),
    (_set("table", "dtype", 3), 2, "block_table must be int32"),
    (_shape("seq_kv", 0, 3), 1, "actual_seq_lengths_kv must be [B]"),
    (_set("seq_kv", "dtype", 3), 2, "must be int32"),
    (_set("cache", "contiguous", 0), 3, "contiguous"),
    (_set("cache", "data", 0x1008), 3, "16-byte aligned"),
    (_set("table", "device", 1), 4, "same device"),
    (_set("table", "data", None), 7, "null data"),
    (_shape("entries", 0, 3), 1, "req_pool_entries must be [B]"),
    (_shape("weights_pool", 1, 128), 1, "token_weights must be"),
    (_set("weights_pool", "dtype", 0), 2, "token weights float32"),
    (_set("weights_pool", "contiguous", 0), 3, "contiguous"),
    (_set("weights_pool", "device", 1), 4, "same device"),
]


@pytest.mark.parametrize("mutate,code,msg", CACHE_FAULTS + [
    (_none("kv"), 7, "null tensor"),
    (_none("positions"), 7, "go together"),
    (_none("entries"), 7, "req_pool_entries goes with"),
    (_none("positions", "positions_pool", "weights_pool"), 7, "req_pool_entries goes with"),
    (_set("seq_q", "ndim", 2), 1, "rank one"),
    (_shape("kv", 1, 1), 1, "kv must be"),
    (_shape("kv", 2, 576), 1, "kv must be"),
    (_shape("rope", 0, 3), 1, "k_rope must be"),
    (_set("kv", "dtype", 3), 2, "16-bit"),
    (_set("rope", "dtype", 1), 2, "16-bit"),
    (_set("rope", "data", 0x1002), 3, "aligned"),
    (_shape("positions", 0, 3), 1, "positions must be [T]"),
    (_set("positions_pool", "dtype", 3), 2, "token positions must be int32"),
    (_shape("positions_pool", 0, 4), 1, "one shape"),
])
def test_append_refusals(mutate, code, msg):
    a = _append_args()
    mutate(a)
    status, text = _append(a)
    assert (status, msg in text) == (code, True), (status, text)


@pytest.mark.parametrize("mutate,code,msg", CACHE_FAULTS + [
    (_none("out"), 7, "null tensor"),
    (_none("entries"), 7, "go together"),
    (_none("weights_pool"), 7, "go together"),
    (lambda a: a.update(topk=_desc((4, 2048), 0)), 7, "not with topk_ids"),
    (lambda a: a.update(topk=_desc((3, 2048), 0), entries=None, weights_pool=None), 1, "topk_ids must be"),
    (lambda a: a.update(topk=_desc((4, 0), 0), entries=None, weights_pool=None), 1, "topk_ids must be"),
    (lambda a: a.update(topk=_desc((4, 16), 3), entries=None, weights_pool=None), 2, "topk_ids must be int32"),
    (_shape("q", 2, 576), 1, "query must be"),
    (_shape("qr", 1, 4), 1, "query_rope must be"),
    (lambda a: [a[k].shape.__setitem__(1, 7) for k in ("q", "qr", "out")], 1, "multiple of the latent heads"),
    (lambda a: [a[k].shape.__setitem__(1, 2048) for k in ("q", "qr", "out")], 1, "at most 1024"),
    (_shape("out", 0, 5), 1, "attention_out must match"),
    (_set("out", "dtype", 2), 2, "16-bit"),
    (_set("q", "data", 0x1004), 3, "aligned"),
])
def test_attention_refusals(mutate, code, msg):
    a = _attention_args()
    mutate(a)
    status, text = _attention(a)
    assert (status, msg in text) == (code, True), (status, text)


@pytest.mark.parametrize("rows,topk", [((1 << 20) - 1, False), ((1 << 20) - 1, True)])
def test_attention_refuses_more_items_than_it_counts(rows, topk):
    """1,024 latent heads of one head each: an item for every row and head."""
    a = _attention_args(T=rows, N=1024)
    B = 1 << 15
    for key, i, n in (("cache", 2, 1024), ("scale", 1, 1024), ("table", 0, B), ("seq_q", 0, B), ("seq_kv", 0, B),
                      ("entries", 0, B)):
        a[key].shape[i] = n
    if topk:
        a.update(topk=_desc((rows, 16), 0), entries=None, weights_pool=None)
    status, text = _attention(a)
    assert (status, "too many query rows and heads" in text) == (1, True), (status, text)


def test_attention_workspace_refusals():
    from nanovllm_amd import _lib

    a = _attention_args()
    need = _lib.lib.nvdsa_latent8_attention_workspace_size(4, 8, 1)
    assert need == _lib.lib.nvdsa_latent8_attention_workspace_size(4, 8, 0) + 4 * 4 * 8
    assert _attention(a, 0x1000, need - 1)[0] == 5
    assert _attention(a, None, need)[0] == 5


# (The eviction takes its batch from actual_seq_lengths_kv, so another length there is the table's fault.)
@pytest.mark.parametrize("mutate,code,msg", [f for f in CACHE_FAULTS if "actual_seq_lengths_kv" not in f[2]] + [
    (_shape("seq_kv", 0, 3), 1, "block_table must be"),
    (_none("kept"), 7, "null tensor"),
    (_shape("budgets", 0, 3), 1, "budgets must be [B]"),
    (_shape("counts", 0, 3), 1, "move_counts must be [B]"),
    (_set("kept", "dtype", 3), 2, "must be int32"),
    (_shape("src", 1, 128), 1, "move_src_slots and"),
    (_shape("dst", 0, 1), 1, "move_src_slots and"),
    (_set("dst", "dtype", 3), 2, "move lists must be int32"),
    (_shape("positions_pool", 0, 4), 1, "one shape"),
])
def test_evict_refusals(mutate, code, msg):
    a = _evict_args()
    mutate(a)
    status, text = _evict(a)
    assert (status, msg in text) == (code, True), (status, text)


def test_evict_scalar_and_workspace_refusals():
    from nanovllm_amd import _lib

    assert _evict(_evict_args(), first=-1)[0] == 7
    assert _evict(_evict_args(), last=1 << 31)[0] == 7
    need = _lib.lib.nvdsa_latent8_evict_workspace_size(2, 3, 2)
    assert _evict(_evict_args(), nbytes=need - 1)[0] == 5
    assert _evict(_evict_args(), ws=None)[0] == 5


def test_nothing_to_do_launches_nothing():
    """No rows or no requests: accepted before any HIP call."""
    a = _append_args(T=0)
    assert _append(a)[0] == 0
    a = _attention_args(T=0)
    assert _attention(a)[0] == 0
    a = _evict_args(B=0)
    assert _evict(a)[0] == 0


def test_operators_are_registered():
    from nanovllm_amd import latent_cache

    for name, schema in latent_cache.SCHEMAS.items():
        op = getattr(torch.ops.nanovllm_dsa, name).default
        assert schema.split("(")[0] == name and str(op._schema).startswith("nanovllm_dsa::" + name)
    cache, scale = latent_cache.empty_latent_cache(3, 2, "cpu")
    assert cache.shape == (3, 128, 2, 576) and cache.dtype == torch.float8_e4m3fn
    assert scale.tolist() == [[1.0, 1.0]] * 3
    with pytest.raises((RuntimeError, NotImplementedError)):  # no CPU implementation
        latent_cache.latent8_append(torch.zeros(1, 2, 512, dtype=torch.bfloat16),
                                    torch.zeros(1, 2, 64, dtype=torch.bfloat16), i32([1]), i32([1]), i32([[0]]), cache,
                                    scale)
    meta = {k: v.to("meta") for k, v in {"cache": cache, "scale": scale, "one": i32([1]), "table": i32([[0]])}.items()}
    latent_cache.latent8_append(torch.zeros(1, 2, 512, dtype=torch.bfloat16, device="meta"),
                                torch.zeros(1, 2, 64, dtype=torch.bfloat16, device="meta"), meta["one"], meta["one"],
                                meta["table"], meta["cache"], meta["scale"])


@pytest.mark.parametrize("amax,expect", [(448.0, 1.0), (448.0 * 1.0001, 2.0), (1.75, 2.0 ** -8), (1.76, 2.0 ** -7),
                                         (0.0, 2.0 ** -126), (1e-45, 2.0 ** -126), (3.3895e38, 2.0 ** 120),
                                         (1.0, 2.0 ** -8), (2.0, 2.0 ** -7)])
def test_oracle_scale_rule(amax, expect):
    s = O.least_scale(amax)
    assert s == expect
    assert amax / s <= 448.0
    assert s == 2.0 ** -126 or amax / (s / 2) > 448.0


def test_oracle_append_grows_and_keeps():
    """A page whose scale grows keeps its values (powers of two only shift)."""
    c = make_cache([100], 1, seed=1, exponents=(-7, -6))
    before = c["cache"][c["table"][0, 0]].float() * c["scale"][c["table"][0, 0], 0]
    kv = torch.full((1, 1, 512), 10.0, dtype=torch.bfloat16)
    O.append(kv, torch.zeros(1, 1, 64, dtype=torch.bfloat16), i32([1]), i32([101]), c["table"], c["cache"], c["scale"])
    page = int(c["table"][0, 0])
    after = c["cache"][page].float() * c["scale"][page, 0]
    assert float(c["scale"][page, 0]) == 2.0 ** -5
    assert torch.allclose(after[:100], before[:100], rtol=0, atol=2.0 ** -5 * 2.0 ** -10)
    assert (after[100, 0, :512] == 10.0).all()


def test_oracle_attention_by_differences():
    """Weights sum to one per row and head; the output is their mean of rows."""
    c = make_cache([70, 0, 5], 2, seed=3)
    qr, q, ends = queries([2, 1, 1], 4, torch.bfloat16, 3)
    out, sums, _, _ = oracle_attention(qr, q, ends, c)
    assert math.isclose(float(sums[0].sum()), 8.0, rel_tol=1e-12) and float(sums[1].sum()) == 0.0
    assert (out[2] == 0).all() and not out.isnan().any()
    every = torch.arange(128, dtype=torch.int32).expand(4, 128).contiguous()
    listed, _, _, _ = oracle_attention(qr, q, ends, c, every)
    assert torch.equal(out, listed)


def test_oracle_evict_keeps_the_heaviest():
    c = make_cache([300], 1, seed=4)
    weights, positions = torch.rand(2, 384), torch.arange(384, dtype=torch.int32).repeat(2, 1)
    w0, rows0 = weights.clone(), c["cache"].clone()
    moves, kept = O.evict(c["lengths"], i32([200]), c["table"], i32([1]), c["cache"], c["scale"], positions, weights,
                          2, 10)
    assert kept == [200] and len(moves[0]) > 10
    survivors = sorted(positions[1, :200].tolist())
    free = [t for t in range(2, 290)]
    best = sorted(free, key=lambda t: -float(w0[1, t]))[:188]
    assert survivors == sorted([0, 1, *best, *range(290, 300)])
    assert not same_codes(rows0, c["cache"])


def test_outputs_count_as_written(monkeypatch):
    """Autograd refuses a backward pass through values that a call overwrote,
    and only outputs count as written."""
    from contextlib import nullcontext
    from types import SimpleNamespace

    from nanovllm_amd import latent_cache as L

    calls = {f"nvdsa_latent8_{n}": lambda *a: 0 for n in ("append", "attention", "evict")}
    monkeypatch.setattr(L, "_C", SimpleNamespace(**calls))
    monkeypatch.setattr(L, "_device_of", lambda t: nullcontext())
    monkeypatch.setattr(L, "_stream_of", lambda t: 0)
    cache, scale = L.empty_latent_cache(3, 1, "cpu")
    f16 = lambda *shape: torch.zeros(*shape, dtype=torch.float16)  # noqa: E731
    t = {"kv": f16(2, 1, 512), "rope": f16(2, 1, 64), "ends": i32([2]), "lens": i32([2]), "table": i32([[0, 1]]),
         "cache": cache, "scale": scale, "row_pos": i32([0, 1]), "entries": i32([0]),
         "positions": torch.zeros(1, 256, dtype=torch.int32), "weights": torch.zeros(1, 256), "q": f16(2, 4, 512),
         "qr": f16(2, 4, 64), "out": f16(2, 4, 512), "budgets": i32([1]), "src": torch.zeros(1, 256, dtype=torch.int32),
         "dst": torch.zeros(1, 256, dtype=torch.int32), "counts": i32([0]), "kept": i32([0])}
    factor = torch.ones_like(t["out"], requires_grad=True)
    loss = (t["out"] * factor).sum()

    def written(call):
        before = {k: v._version for k, v in t.items()}
        call()
        return {k for k, v in t.items() if v._version > before[k]}

    a = [t[k] for k in ("kv", "rope", "ends", "lens", "table", "cache", "scale")]
    assert written(lambda: L._append(*a)) == {"cache", "scale"}
    records = [t[k] for k in ("row_pos", "entries", "positions", "weights")]
    assert written(lambda: L._append(*a, *records)) == {"cache", "scale", "positions", "weights"}
    a = [t[k] for k in ("qr", "q", "ends", "lens", "table", "cache", "scale")]
    assert written(lambda: L._attention(*a, 0.1, t["out"])) == {"out"}
    assert written(lambda: L._attention(*a, 0.1, t["out"], None, t["entries"], t["weights"])) == {"out", "weights"}
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    a = [t[k] for k in ("lens", "budgets", "table", "entries", "cache", "scale", "positions", "weights", "src", "dst",
                        "counts", "kept")]
    assert written(lambda: L._evict(*a, 0, 0)) == {"cache", "scale", "positions", "weights", "src", "dst", "counts", "kept"}
    with torch.inference_mode():
        t["out"] = f16(2, 4, 512)
        a = [t[k] for k in ("qr", "q", "ends", "lens", "table", "cache", "scale")]
        L._attention(*a, 0.1, t["out"])  # (no counter to raise)
    L._attention(*a, 0.1, t["out"])
