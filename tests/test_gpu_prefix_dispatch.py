"""The prefix-sharing functions take tensors in every form that the dispatcher
resolves, and are seen by whatever traces them."""

from __future__ import annotations

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from _prefix import PAGE, SCALE, api, i32, norm_inputs

pytestmark = pytest.mark.gpu

NAMES = ["pages_branch", "pages_copy", "norm_rope_append", "shared_prefix_attention", "pages_compact"]
OUTPUTS = ("kv_cache", "k_rope", "query_rope", "query_nope", "out", "lens", "table", "refs", "src", "dst", "tokens",
           "missing", "msrc", "mdst", "count")


def _state(seed=61):
    """Two requests on one page of 128 tokens and a page with 30 more that both write on."""
    s = norm_inputs([1, 1], [158, 158], 4, 128, torch.bfloat16, seed)
    s = {k: v for k, v in s.items()}
    table = i32([[0, 1, -1], [0, 1, -1]])
    g = torch.Generator().manual_seed(seed)
    s.update(table=table, refs=i32([2, 2, 0, 0, 0, 0]), lens=i32([158, 158]), new=i32([1, 1]),
             src=i32([9, 9]), dst=i32([9, 9]), tokens=i32([9, 9]), missing=i32([9]),
             msrc=i32([9] * 6), mdst=i32([9] * 6), count=i32([9]), parents=i32([0, 0]),
             kv_cache=torch.randn(6, PAGE, 1, 512, generator=g).bfloat16(),
             k_rope=torch.randn(6, PAGE, 1, 64, generator=g).bfloat16(),
             latent=torch.randn(2, 4, 512, generator=g).bfloat16(), out=torch.zeros(2, 4, 512).bfloat16(),
             group_ends=i32([2]), prefix=i32([128]))
    return {k: v.cuda() for k, v in s.items()}


def _calls(s):
    p = api()
    p.pages_branch(s["lens"], s["new"], s["table"], s["refs"], s["src"], s["dst"], s["tokens"], s["missing"],
                   parents=s["parents"])
    p.pages_copy(s["src"], s["dst"], [s["kv_cache"], s["k_rope"]], tokens=s["tokens"])
    p.norm_rope_append(s["query"], s["kv"], s["cos"], s["sin"], s["kv_weight"], s["ends"], s["lengths"], s["table"],
                       s["k_rope"], s["kv_cache"], s["query_rope"], query_norm_weight=s["query_weight"],
                       query_nope=s["query_nope"])
    p.shared_prefix_attention(s["query_rope"], s["latent"], s["ends"], s["lengths"], s["table"], s["k_rope"],
                              s["kv_cache"], SCALE, s["out"], prefix_request_ends=s["group_ends"], prefix_lengths=s["prefix"])
    p.pages_compact(s["table"], s["refs"], s["msrc"], s["mdst"], s["count"])


def _same(a, b):
    for k in OUTPUTS:
        x, y = (t[k].view(torch.int16) if t[k].dtype == torch.bfloat16 else t[k] for t in (a, b))
        if k in ("msrc", "mdst"):   # (what lies behind the count is nobody's)
            n = int(a["count"])
            x, y = x[:n], y[:n]
        assert torch.equal(x, y), k


def test_a_dispatch_mode_sees_the_calls():
    class Seen(TorchDispatchMode):
        names: list[str] = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(func._schema.name.split("::")[-1])
            return func(*args, **(kwargs or {}))

    with Seen() as mode:
        _calls(_state())
    assert [n for n in mode.names if n in NAMES] == NAMES


def test_tracing_records_the_calls():
    from torch.fx.experimental.proxy_tensor import make_fx

    s = _state()
    keys = list(s)
    graph = make_fx(lambda *values: _calls(dict(zip(keys, values))))(*s.values())
    found = [n.target._schema.name.split("::")[-1] for n in graph.graph.nodes
             if n.op == "call_function" and "nanovllm_dsa" in str(n.target)]
    assert found == NAMES


@pytest.mark.parametrize("which", [("query",), ("kv", "cos"), ("latent",), ("kv_weight", "query_weight", "sin")])
def test_negated_views(which):
    plain, negated = _state(), _state()
    for k in which:
        negated[k] = torch._neg_view(-negated[k])
        assert negated[k].is_neg() and torch.equal(negated[k], plain[k])
    _calls(plain)
    _calls(negated)
    _same(plain, negated)


@pytest.mark.parametrize("which", ["latent", "kv_cache", "group_ends"])
def test_wrapped_tensors_do_not_reach_the_kernels(which):
    """Tensors without memory of their own end in the operator's meta form,
    wherever among the arguments they stand."""
    from torch._subclasses import FakeTensorMode

    s = _state()
    before = s["out"].clone()
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        s[which] = mode.from_tensor(s[which])
    api().shared_prefix_attention(s["query_rope"], s["latent"], s["ends"], s["lengths"], s["table"], s["k_rope"],
                                  s["kv_cache"], SCALE, s["out"], prefix_request_ends=s["group_ends"],
                                  prefix_lengths=s["prefix"])
    assert torch.equal(before, s["out"])


def test_compiled_calls_write_the_same():
    plain, compiled = _state(), _state()
    _calls(plain)
    torch.compile(_calls, backend="aot_eager", fullgraph=True)(compiled)
    _same(plain, compiled)


def test_tensors_elsewhere_are_refused():
    s = _state()
    for k in ("latent", "table", "prefix"):
        t = dict(s)
        t[k] = s[k].cpu()
        with pytest.raises((RuntimeError, NotImplementedError)):
            api().shared_prefix_attention(t["query_rope"], t["latent"], t["ends"], t["lengths"], t["table"], t["k_rope"],
                                          t["kv_cache"], SCALE, t["out"], prefix_request_ends=t["group_ends"],
                                          prefix_lengths=t["prefix"])
    strided = s["latent"].transpose(0, 1).contiguous().transpose(0, 1)
    with pytest.raises(RuntimeError, match="contiguous"):
        api().shared_prefix_attention(s["query_rope"], strided, s["ends"], s["lengths"], s["table"], s["k_rope"],
                                      s["kv_cache"], SCALE, s["out"])
    with pytest.raises(RuntimeError, match="contiguous"):
        api().pages_copy(s["src"], s["dst"], [s["kv_cache"][:, ::2]])
