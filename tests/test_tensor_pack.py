"""The native descriptors hold what those read through Python attributes hold,
for every form of tensor a caller may pass."""

from __future__ import annotations

import pytest
import torch

FORMS = [
    lambda d: torch.zeros(3, device=d), lambda d: torch.zeros((), device=d),
    lambda d: torch.zeros(0, 4, dtype=torch.bfloat16, device=d), lambda d: torch.zeros(2, 3, 4, 5, dtype=torch.float16, device=d),
    lambda d: torch.zeros(1, 2, 3, 4, 5, device=d), lambda d: torch.zeros(4, 6, device=d).t()[1:],
    lambda d: torch.zeros(2, dtype=torch.int64, device=d), lambda d: torch.zeros(8, dtype=torch.int32, device=d)[3:],
    lambda d: torch.zeros(2, 8, device=d).to(torch.float8_e4m3fn), lambda d: torch.zeros(5, 1, 7, device=d).expand(5, 3, 7),
    lambda d: torch.nn.Parameter(torch.zeros(4, 4, device=d)), lambda d: torch.zeros(3, 3, device=d, requires_grad=True) * 2,
]


def _fields(at):
    from nanovllm_amd import _lib

    t = _lib.NvdsaTensor.from_address(at)
    return [t.data, t.dtype, t.ndim, list(t.shape), t.contiguous, t.device]


def _compare(tensors):
    from nanovllm_amd import _lib

    assert _lib._native_pack is not None, "the extension is not built"
    native = _lib._native_pack(*tensors)
    buf, at = _lib.pack(*tensors)
    plain_buf, plain = _lib.pack_plain(*tensors)
    assert native is not None and type(at) is type(plain) is list and len(at) == len(tensors)
    for t, a, b in zip(tensors, at, plain):
        assert (a is None) == (b is None) == (t is None)
        if t is not None:
            assert _fields(a) == _fields(b)
    assert bytes(buf) == bytes(plain_buf)
    with pytest.raises(IndexError):
        _lib.pack(*[tensors[0]] * (_lib._MAX_PACKED + 1))


def test_host_tensors():
    tensors = [make("cpu") for make in FORMS]
    _compare([*tensors, None, tensors[0]])
    _compare([None])
    _compare([tensors[3]] * 24)


def test_what_is_no_tensor_goes_the_plain_way():
    from nanovllm_amd import _lib

    assert _lib._native_pack(torch.zeros(2), 3) is None
    assert _lib._native_pack(torch.zeros(2, device="meta")) is None
    for wrong in (3, "x", [torch.zeros(1)]):
        with pytest.raises(AttributeError):
            _lib.pack(torch.zeros(2), wrong)
    buf, at = _lib.pack()
    assert at == [] and len(bytes(buf)) == 0


def test_buffers_are_their_callers():
    """Two packs at once do not share memory, and none is kept."""
    import sys

    from nanovllm_amd import _lib

    x, y = torch.zeros(2), torch.zeros(3, 4)
    before = sys.getrefcount(x)
    first = _lib.pack(x, y)
    second = _lib.pack(y, x)
    assert _fields(first[1][0]) == _fields(second[1][1]) != _fields(second[1][0])
    for _ in range(1000):
        _lib.pack(x, None, y)
    assert sys.getrefcount(x) == before


@pytest.mark.gpu
def test_device_tensors():
    tensors = [make("cuda") for make in FORMS]
    _compare([*tensors, None, torch.zeros(7).pin_memory(), torch.zeros(7)])
