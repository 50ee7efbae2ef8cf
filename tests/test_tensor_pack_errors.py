"""What the native descriptors leave to the plain way: tensors whose fields are
computed in Python, and fail there."""

from __future__ import annotations

import pytest
import torch


class Refusing(torch.Tensor):
    """Has sizes and strides of its own making, and refuses to make them."""

    @staticmethod
    def __new__(cls, x, policy):
        return torch.Tensor._make_wrapper_subclass(cls, x.shape, dtype=x.dtype, device=x.device,
                                                   dispatch_sizes_strides_policy=policy)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise ValueError("not these sizes")


@pytest.mark.parametrize("policy", ["sizes", "strides", None])
def test_an_error_in_python_is_the_callers(policy):
    from nanovllm_amd import _lib

    t = Refusing(torch.zeros(3, 4), policy)
    assert _lib._native_pack(torch.zeros(2), t) is None
    with pytest.raises((ValueError, RuntimeError)):   # (not SystemError: the fields' own error, or that it has no memory)
        _lib.pack(torch.zeros(2), t)
    assert _lib._native_pack(torch.zeros(2)) is not None
