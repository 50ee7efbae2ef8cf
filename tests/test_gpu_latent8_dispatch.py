"""The 8-bit latent cache's functions take tensors in every form that the
dispatcher resolves, and are seen by whatever traces them."""

from __future__ import annotations

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from _latent8 import PAGE, SCALE, i32, make_cache, queries, same_codes

pytestmark = pytest.mark.gpu


def _state(seed=51):
    c = make_cache([300, 140], 1, seed=seed)
    qr, q, ends = queries([1, 2], 8, torch.bfloat16, seed)
    s = {k: v.cuda() for k, v in {"qr": qr, "q": q, "ends": ends, "lens": c["lengths"], "table": c["table"],
                                  "cache": c["cache"], "scale": c["scale"], "entries": i32([1, 0])}.items()}
    g = torch.Generator().manual_seed(seed)
    s["kv"], s["rope"] = (torch.randn(3, 1, n, generator=g).bfloat16().cuda() for n in (512, 64))
    s["weights"] = torch.rand(2, c["cols"] * PAGE, generator=g).cuda()
    s["positions"] = torch.arange(c["cols"] * PAGE, dtype=torch.int32).repeat(2, 1).cuda()
    s["out"] = torch.zeros_like(s["q"])
    s["src"], s["dst"] = (torch.zeros(2, c["cols"] * PAGE, dtype=torch.int32, device="cuda") for _ in range(2))
    s["counts"], s["kept"] = (torch.zeros(2, dtype=torch.int32, device="cuda") for _ in range(2))
    s["budgets"] = i32([200, 128]).cuda()
    return s


def _calls(s):
    from nanovllm_amd.latent_cache import latent8_append, latent8_attention, latent8_evict

    latent8_append(s["kv"], s["rope"], s["ends"], s["lens"], s["table"], s["cache"], s["scale"])
    latent8_attention(s["qr"], s["q"], s["ends"], s["lens"], s["table"], s["cache"], s["scale"], SCALE, s["out"],
                      req_pool_entries=s["entries"], token_weights=s["weights"])
    latent8_evict(s["lens"], s["budgets"], s["table"], s["entries"], s["cache"], s["scale"], s["positions"],
                  s["weights"], s["src"], s["dst"], s["counts"], s["kept"], protect_first=2, protect_last=9)


NAMES = ["latent8_append", "latent8_attention", "latent8_evict"]


def test_a_dispatch_mode_sees_the_calls():
    class Seen(TorchDispatchMode):
        names: list[str] = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(func._schema.name.split("::")[-1])
            return func(*args, **(kwargs or {}))

    with Seen() as mode:
        _calls(_state())
    assert [n for n in mode.names if n.startswith("latent8")] == NAMES


def test_tracing_records_the_calls():
    from torch.fx.experimental.proxy_tensor import make_fx

    s = _state()
    keys = list(s)
    graph = make_fx(lambda *values: _calls(dict(zip(keys, values))))(*s.values())
    assert [n.target._schema.name.split("::")[-1] for n in graph.graph.nodes
            if n.op == "call_function" and "latent8" in str(n.target)] == NAMES


@pytest.mark.parametrize("which", [("kv",), ("rope",), ("q",), ("qr",), ("kv", "rope", "q", "qr")])
def test_negated_views(which):
    plain, negated = _state(), _state()
    for k in which:
        negated[k] = torch._neg_view(-negated[k])
        assert negated[k].is_neg() and torch.equal(negated[k], plain[k])
    _calls(plain)
    _calls(negated)
    assert same_codes(plain["cache"], negated["cache"]) and torch.equal(plain["out"], negated["out"])
    for k in ("scale", "weights", "positions", "kept", "counts"):
        assert torch.equal(plain[k], negated[k])


def test_wrapped_tensors_do_not_reach_the_kernels():
    """Tensors without memory of their own end in an error or in the operator's
    meta form, wherever among the arguments they stand."""
    from torch._subclasses import FakeTensorMode

    for k in ("kv", "ends", "scale"):
        s = _state()
        before = s["cache"].view(torch.uint8).clone()
        with FakeTensorMode(allow_non_fake_inputs=True) as mode:
            s[k] = mode.from_tensor(s[k])
        from nanovllm_amd.latent_cache import latent8_append

        latent8_append(s["kv"], s["rope"], s["ends"], s["lens"], s["table"], s["cache"], s["scale"])
        assert torch.equal(before, s["cache"].view(torch.uint8))


def test_compiled_calls_write_the_same():
    plain, compiled = _state(), _state()
    _calls(plain)
    torch.compile(_calls, backend="aot_eager", fullgraph=True)(compiled)
    assert same_codes(plain["cache"], compiled["cache"])
    for k in ("out", "scale", "weights", "positions", "src", "dst", "counts", "kept"):
        assert torch.equal(plain[k], compiled[k]), k
