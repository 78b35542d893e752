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
    c._index = -1  # what a host tensor says
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


def versions(*tensors):
    return [t._version for t in tensors]


def test_what_is_written_counts_as_written(codec):
    """The library writes behind torch's back: every tensor of the caller's that a call writes has its version counted on,
    so that a graph that saved one refuses its backward pass, as after an in-place operation of torch's own."""
    a, b = torch.randn(10), torch.randn(3, 3)
    grads = [dev(a), dev(b)]
    was = versions(a, b)
    codec.grad_norm(grads)
    assert versions(a, b) == was                    # only read
    codec.clip_grads(grads, 1.0)
    assert all(v > w for v, w in zip(versions(a, b), was))
    was = versions(a, b)
    outs = [torch.empty(10), torch.empty(3, 3)]
    outs_were = versions(*outs)
    codec.clip_grads(svb.GradSet(grads, out=[dev(t) for t in outs]), 1.0)
    assert versions(a, b) == was and all(v > w for v, w in zip(versions(*outs), outs_were))
    # views of one bucket
    bucket = torch.randn(100)
    kept = svb.GradSet([dev(t) for t in bucket.split(10)])
    spare = svb.GradSet([dev(t) for t in torch.randn(100).split(10)], out=[dev(t) for t in bucket.split(10)])
    for s in (kept, spare):
        for _ in range(2):
            was = bucket._version
            codec.clip_grads(s, 1.0)
            assert bucket._version > was
    # norms and residuals
    word = torch.zeros(1)
    codec.grad_norm(grads, out=word)
    assert word._version == 1
    codec.clip_grads(grads, 1.0, norm=word)
    assert word._version == 1                       # only read
    g, r, new, out = torch.randn(8), torch.zeros(8), torch.zeros(8), torch.zeros(100, dtype=torch.uint8)
    codec.quantize_feedback_encode(g, 4.0, r, norm=word)
    assert versions(g, r, word) == [0, 1, 1]
    codec.quantize_feedback_encode(g, 4.0, r, out=out, residual_out=new)
    assert versions(g, r, new, out) == [0, 1, 1, 1]


def test_a_saved_gradient_is_not_changed_unseen(codec):
    w = torch.randn(6, requires_grad=True)
    for change in (lambda g: codec.clip_grads([dev(g)], 1.0),
                   lambda g: codec.clip_grads(svb.GradSet([dev(torch.ones(6))], out=[dev(g)]), 1.0),
                   lambda g: codec.quantize_feedback_encode(torch.ones(6), 4.0, g)):
        g = torch.randn(6)
        loss = (w * g).sum()
        change(g)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_tensors_without_versions(codec):
    """Tensors made in inference mode have none; ordinary ones have theirs there too."""
    with torch.inference_mode():
        a, r = torch.randn(10), torch.zeros(10)
        for _ in range(2):
            codec.clip_grads([dev(a)], 1.0)
            codec.quantize_feedback_encode(a, 4.0, r)
    codec.clip_grads([dev(a)], 1.0)
    codec.quantize_feedback_encode(a, 4.0, r)
    b = torch.randn(10)
    with torch.inference_mode():
        codec.clip_grads([dev(b)], 1.0)
    assert b._version == 1 and len(codec.calls) == 7


def test_lazily_negated_tensors_are_refused(codec):
    """What such a tensor's memory holds is not its values."""
    z = torch.complex(torch.tensor([1.0]), torch.tensor([2.0]))
    x = z.conj().imag                               # -2, of which memory holds 2
    assert x.is_neg() and x.is_contiguous() and float(x) == -2.0
    plain = torch.zeros(1)
    for wrong in (lambda: svb.GradSet([dev(x)]), lambda: svb.GradSet([dev(plain)], out=[dev(x)]),
                  lambda: svb.GradSet([dev(plain), dev(x)])):
        with pytest.raises(ValueError, match="negated"):
            wrong()
    for change in (dict(grad=x), dict(residual=x), dict(residual_out=x)):
        with pytest.raises(ValueError, match="negated"):
            codec.quantize_feedback_encode(**dict(dict(grad=plain, scale=4.0, residual=torch.zeros(1)), **change))
    with pytest.raises(ValueError, match="negated"):
        codec.grad_norm([dev(plain)], out=x)
    with pytest.raises(ValueError, match="negated"):
        codec.clip_grads([dev(plain)], 1.0, norm=x)
    assert not codec.calls
    y = x.resolve_neg()
    codec.grad_norm([dev(y)])
    codec.quantize_feedback_encode(y, 4.0, plain)
    assert len(codec.calls) == 2


def test_versions_are_counted_once_a_buffer():
    """A set that is kept holds one tensor for every version that its calls count on."""
    bucket = torch.randn(100)
    views = [dev(t) for t in bucket.split(10)]
    others = [dev(torch.randn(10)) for _ in range(10)]
    assert len(svb.GradSet(views).written) == 1 and len(svb.GradSet(others).written) == 10
    assert len(svb.GradSet(others, out=views).written) == 1 and len(svb.GradSet(views, out=others).written) == 10
    with torch.inference_mode():
        made = [dev(t) for t in torch.randn(100).split(10)]
    assert len(svb.GradSet(made).written) == 0
