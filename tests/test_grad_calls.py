"""What the Python side of the gradient operators hands to the library, on the CPU: tensors that say they are on a
device, and a codec whose calls are written down instead of made."""
import math

import pytest
import torch

import streamvbyte_amd as svb


class OnDevice(torch.Tensor):
    """A host tensor that the checks take for one on a device; its detached copies and views are of its kind."""
    is_cuda = property(lambda self: True)


def dev(t):
    return t.as_subclass(OnDevice)


@pytest.fixture
def codec():
    c = object.__new__(svb.DeviceCodec)
    c.torch, c.lib, c.device, c.max_count = torch, svb.load(), torch.device("cpu"), 1 << 20
    c.ws_bytes = c.lib.svbgpu_workspace_bytes(c.max_count)
    c.ws, c.res = torch.zeros(c.ws_bytes, dtype=torch.uint8), torch.zeros(8, dtype=torch.int64)
    c.calls = []
    c._call = lambda what, *args: c.calls.append((what, args))
    return c


def test_a_given_norm_is_of_any_kind(codec):
    """It is read, so the kind that would be worked out does not matter: a norm of another order can be clipped by."""
    x = [dev(torch.ones(5))]
    given = torch.tensor([3.0])
    assert codec.clip_grads(x, 1.0, norm_type=3.0, norm=given) is given
    assert len(codec.calls) == 1 and codec.calls[0][0] == "svbgpu_grad_clip"
    for p in (3.0, 0, "fro"):
        with pytest.raises(ValueError, match="norm_type"):
            codec.clip_grads(x, 1.0, norm_type=p)
        with pytest.raises(ValueError, match="norm_type"):
            codec.grad_norm(x, p)
    for p in (1, 2, math.inf):
        codec.clip_grads(x, 1.0, norm_type=p, norm=given)
        codec.clip_grads(x, 1.0, norm_type=p)
    assert len(codec.calls) == 7


def moved(codec, grads, owner):
    """Whether the set is refused once `owner`'s storage has given its memory back."""
    codec.grad_norm(grads)
    owner.untyped_storage().resize_(0)
    try:
        codec.grad_norm(grads)
    except ValueError as e:
        assert "moved" in str(e)
        return True
    return False


def test_memory_given_back_is_noticed(codec):
    """One tensor a storage is compared; an empty one has no address that could tell.  (The results are compared by
    themselves: a failed assert would print tensors that have no memory any more.)"""
    def buffers():
        return torch.randn(100), torch.randn(100)
    seen = {}
    x, _ = buffers()
    seen["two views"] = moved(codec, svb.GradSet([dev(x[:40]), dev(x[40:])]), x)
    x, _ = buffers()
    seen["empty views beside it"] = moved(codec, svb.GradSet([dev(x[:0]), dev(x), dev(x[7:7])]), x)
    x, y = buffers()
    seen["an empty output in an input's storage"] = moved(codec, svb.GradSet([dev(x), dev(y[:0])], out=[dev(y), dev(x[:0])]), x)
    x, y = buffers()
    seen["and the other way round"] = moved(codec, svb.GradSet([dev(x), dev(y[:0])], out=[dev(y), dev(x[:0])]), y)
    x, y = buffers()
    seen["another tensor's"] = not moved(codec, svb.GradSet([dev(x), dev(x[:0])]), y)
    assert seen == dict.fromkeys(seen, True)
