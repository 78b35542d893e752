"""What the gradient operators refuse, checked without a GPU: argument errors come before any device work, and a call
whose arguments are all right gets as far as the missing device (-2) here."""
import ctypes as C

import pytest
import torch

import streamvbyte_amd as svb
from streamvbyte_amd._lib import GradTensor

EINVAL, ENODEVICE, EWORKSPACE = -1, -2, -3
F32, F16, BF16 = 0, 1, 2
WS = 0x7000_0000_0000
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are made up")


def tensors(*rows):
    t = (GradTensor * max(len(rows), 1))()
    for i, (addr, count, kind) in enumerate(rows):
        t[i] = GradTensor(addr, count, kind)
    return t, len(rows)


def norm(rows, kind=2, d_norm=0x1000, ws=WS, ws_bytes=None):
    lib = svb.load()
    t, n = tensors(*rows)
    return lib.svbgpu_grad_norm(kind, t, n, d_norm, ws, lib.svbgpu_grad_workspace_bytes(n) if ws_bytes is None else ws_bytes, None)


def clip(rows, outs=None, limit=1.0, kind=2, given=0, d_norm=0x1000, ws=WS, ws_bytes=None):
    lib = svb.load()
    t, n = tensors(*rows)
    o = None if outs is None else (C.c_void_p * max(n, 1))(*outs)
    return lib.svbgpu_grad_clip(kind, t, n, o, limit, given, d_norm, ws,
                                lib.svbgpu_grad_workspace_bytes(n) if ws_bytes is None else ws_bytes, None)


A, B = 0x10_0000, 0x20_0000


def test_norm_arguments():
    assert norm([(A, 10, F32), (B, 3, BF16)]) == ENODEVICE
    assert norm([]) == ENODEVICE and norm([(None, 0, F32)]) == ENODEVICE
    assert norm([(A, 10, F32), (A, 10, F32)]) == ENODEVICE          # read only: may overlap
    assert norm([(A + 2, 10, F16)]) == ENODEVICE
    assert norm([(A, 10, 3)]) == EINVAL and norm([(A, 10, -1)]) == EINVAL
    assert norm([(A, 10, F32)], kind=3) == EINVAL and norm([(A, 10, F32)], kind=-1) == EINVAL
    assert norm([(A + 2, 10, F32)]) == EINVAL and norm([(A + 1, 10, BF16)]) == EINVAL
    assert norm([(None, 10, F32)]) == EINVAL
    assert norm([(A, 1 << 37, F32)]) == EINVAL and norm([(1 << 56, 1, F32)]) == EINVAL
    assert norm([(A, 10, F32)], d_norm=None) == EINVAL and norm([(A, 10, F32)], d_norm=0x1002) == EINVAL
    assert norm([(A, 10, F32)], ws=None) == EWORKSPACE and norm([(A, 10, F32)], ws=WS + 128) == EWORKSPACE
    assert norm([(A, 10, F32)], ws_bytes=256) == EWORKSPACE
    assert svb.load().svbgpu_grad_norm(2, None, 3, 0x1000, WS, 1 << 20, None) == EINVAL


def test_clip_arguments():
    ok = [(A, 10, F32), (B, 3, BF16)]
    assert clip(ok) == ENODEVICE and clip([]) == ENODEVICE
    assert clip(ok, limit=0.0) == ENODEVICE and clip(ok, limit=float("inf")) == ENODEVICE
    assert clip(ok, limit=-1.0) == EINVAL and clip(ok, limit=float("nan")) == EINVAL
    assert clip(ok, kind=7) == EINVAL
    assert clip(ok, ws=None) == EWORKSPACE and clip(ok, ws=None, given=1) == ENODEVICE
    assert clip([(A + 1, 4, F16)]) == EINVAL


def test_clip_writes_nothing_twice():
    assert clip([(A, 10, F32), (A + 40, 10, F32)]) == ENODEVICE    # neighbours
    assert clip([(A + 40, 10, F32), (A, 10, F32)]) == ENODEVICE    # in any order
    assert clip([(A, 10, F32), (A, 10, F32)]) == EINVAL
    assert clip([(A, 10, F32), (A + 36, 10, F32)]) == EINVAL
    assert clip([(A + 36, 10, F32), (B, 1, F32), (A, 10, F32)]) == EINVAL
    assert clip([(A, 10, F32), (A, 0, F32)]) == ENODEVICE          # empty tensors are nowhere
    many = [(A + 64 * i, 16, F32) for i in range(300)]
    assert clip(many) == ENODEVICE and clip(many[::-1]) == ENODEVICE
    assert clip(many + [(A + 64 * 150 + 60, 2, F16)]) == EINVAL


def test_clip_outputs():
    rows = [(A, 10, F32), (A + 100, 10, F32)]
    assert clip(rows, outs=[B, B + 40]) == ENODEVICE
    assert clip(rows, outs=[A, A + 100]) == ENODEVICE               # themselves
    assert clip(rows, outs=[A, B]) == ENODEVICE
    assert clip(rows, outs=[A + 100, A]) == EINVAL                  # each other
    assert clip(rows, outs=[B, A]) == EINVAL
    assert clip(rows, outs=[A + 4, B]) == EINVAL                    # itself, shifted
    assert clip(rows, outs=[B, B]) == EINVAL and clip(rows, outs=[B, B + 36]) == EINVAL
    assert clip(rows, outs=[B, None]) == EINVAL and clip(rows, outs=[B, B + 42]) == EINVAL
    assert clip([(A, 10, F32), (A, 10, F32)], outs=[B, B + 40]) == ENODEVICE  # read twice, written apart
    assert clip([(A, 10, F32), (A, 10, F32)], outs=[A, B]) == EINVAL
    assert clip([(A, 10, F32), (None, 0, F32)], outs=[B, None]) == ENODEVICE


def test_the_norm_lies_apart():
    """It is read while tensors are written."""
    rows = [(A, 10, F32), (B, 3, BF16)]
    for d_norm in (A, A + 36, B, B + 4):
        assert clip(rows, d_norm=d_norm) == EINVAL, hex(d_norm)
        assert clip(rows, outs=[0x30_0000, 0x31_0000], d_norm=d_norm) == EINVAL
        assert norm(rows, d_norm=d_norm) == ENODEVICE               # written when everything is read
    assert clip(rows, d_norm=A + 40) == ENODEVICE and clip(rows, d_norm=B + 8) == ENODEVICE
    assert clip(rows, outs=[0x30_0000, 0x31_0000], d_norm=0x30_0000 + 36) == EINVAL
    assert clip(rows, outs=[0x30_0000, 0x31_0000], d_norm=0x31_0004, given=1) == EINVAL


def test_feedback_arguments():
    lib = svb.load()
    n = 1000
    room = svb.streamvbyte_max_compressedbytes(n)
    at = dict(variant=1, kind=F32, grad=A, count=n, norm=None, limit=1.0, scale=64.0, r=B, r_out=B, out=0x40_0000, ws=WS,
              ws_bytes=lib.svbgpu_workspace_bytes(n))

    def call(**change):
        k = dict(at, **change)
        return lib.svbgpu_quantize_feedback_encode(k["variant"], k["kind"], k["grad"], k["count"], k["norm"], k["limit"], k["scale"],
                                                   k["r"], k["r_out"], k["out"], k["ws"], k["ws_bytes"], None, None)
    assert call() == ENODEVICE
    assert call(r_out=0x30_0000) == ENODEVICE and call(kind=BF16, grad=A + 2) == ENODEVICE and call(out=0x40_0003) == ENODEVICE
    assert call(norm=0x1000) == ENODEVICE and call(limit=float("nan")) == ENODEVICE  # without a norm the limit is not looked at
    assert call(count=0, grad=None, r=None, r_out=None, out=None) == 0
    assert call(variant=2) == EINVAL and call(kind=5) == EINVAL
    for scale in (0.0, -1.0, float("inf"), float("nan"), 1e-39, 3e38):
        assert call(scale=scale) == EINVAL, scale
    assert call(norm=0x1000, limit=-0.5) == EINVAL and call(norm=0x1000, limit=float("nan")) == EINVAL and call(norm=0x1002) == EINVAL
    for missing in ("grad", "r", "r_out", "out"):
        assert call(**{missing: None}) == EINVAL, missing
    assert call(grad=A + 2) == EINVAL and call(kind=F16, grad=A + 1) == EINVAL and call(r=B + 2) == EINVAL and call(r_out=B + 1) == EINVAL
    assert call(r_out=B + 4) == EINVAL and call(r_out=B + 4 * n) == ENODEVICE          # shifted, and just behind
    assert call(grad=B) == EINVAL and call(grad=B + 4 * n - 4) == EINVAL               # the residual is written
    assert call(out=A + 4 * n - 1) == EINVAL and call(out=A + 4 * n) == ENODEVICE
    assert call(out=B - room + 1) == EINVAL and call(out=B - room) == ENODEVICE
    assert call(r_out=0x30_0000, out=0x30_0000 + 4 * n - 1) == EINVAL
    assert call(norm=B) == EINVAL and call(norm=B + 4 * n - 4) == EINVAL and call(norm=B + 4 * n) == ENODEVICE
    assert call(norm=0x40_0000) == EINVAL and call(norm=A) == ENODEVICE                # a gradient may hold it


def test_sets_look_their_tensors_over():
    with pytest.raises(ValueError, match="not a dense tensor on a device"):
        svb.GradSet([torch.zeros(3)])
    assert len(svb.GradSet([])) == 0
    for wrong in ([None], [torch.zeros(3), 1.0], torch.zeros(2, 3).numpy()):  # a gradient that was never made
        with pytest.raises(ValueError, match="tensors, not"):
            svb.GradSet(wrong)
    with pytest.raises(ValueError, match="0 tensors, but 1 outputs"):
        svb.GradSet([], out=[torch.zeros(3)])
    from streamvbyte_amd import _dense, _grad_type
    x = torch.zeros(4, 6, 5)
    for t in (x, x.permute(2, 0, 1), x[1:3], x[2], x[:, :1, :][:1], torch.zeros(()), torch.zeros(0, 3), x.view(-1)[7:9]):
        assert _dense(t), t.stride()
    for t in (x[:, :3], x[::2], x[:, :, 0], torch.zeros(1).expand(4), torch.zeros(3, 1).expand(3, 2), x.as_strided((3, 3), (1, 1))):
        assert not _dense(t), t.stride()
    assert [_grad_type(torch, t) for t in (torch.float32, torch.float16, torch.bfloat16)] == [F32, F16, BF16]
    for t in (torch.float64, torch.int32, torch.uint8):
        with pytest.raises(ValueError):
            _grad_type(torch, t)
