"""The largest sets of the gradient operators, by arguments alone: nothing here needs a GPU, for every call is refused
before any device work, or gets as far as the missing device (-2)."""
import pytest
import torch

import streamvbyte_amd as svb
from test_grad_refusals import A, EINVAL, ENODEVICE, F16, F32, clip, norm

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are made up")


def test_bytes_of_a_set():
    """A norm's chunks grow with the set up to 2^31 bytes, and the workspace has a word for each of 4096 of them and one
    more a tensor: past 2^43 bytes there would be more chunks than words.  A tensor may be given often, so a set can be
    larger than any memory."""
    longest = (1 << 37) - 1  # elements of a tensor, at most
    assert norm([(A, longest, F32)] * 16) == ENODEVICE                       # 2^43 - 64 bytes
    assert norm([(A, longest, F32)] * 16 + [(A, 16, F32)]) == ENODEVICE      # 2^43 exactly
    assert norm([(A, longest, F32)] * 16 + [(A, 17, F32)]) == EINVAL
    assert norm([(A, longest, F32)] * 16 + [(A, 16, F32), (A, 1, F16)]) == EINVAL
    assert norm([(A, longest, F16)] * 33) == EINVAL
    assert norm([(A, longest, F32)] * 120) == EINVAL
    room = [(A, longest, F32)] * 15 + [(A, 16, F32)] * 1000                  # more tensors, fewer bytes
    assert norm(room) == ENODEVICE
    assert clip([(1 << 40, longest, F32)], given=1) == ENODEVICE


def test_any_number_of_tensors():
    """Chunks are counted anew in every launch, so the number of tensors is bounded by the 32 bits of all chunks alone."""
    import ctypes as C
    from streamvbyte_amd._lib import GradTensor
    lib = svb.load()
    n = (1 << 22) + 1
    table = (GradTensor * n)()  # all empty
    for i in (0, n // 2, n - 1):
        table[i] = GradTensor(A + 4096 * i, 3, F32)
    room = lib.svbgpu_grad_workspace_bytes(n)
    assert room >= 8 * (4096 + n)
    ws = 0x7000_0000_0000
    assert lib.svbgpu_grad_norm(2, table, n, 0x1000, ws, room, None) == ENODEVICE
    assert lib.svbgpu_grad_norm(2, table, n, 0x1000, ws, room - 256, None) == -3
    assert lib.svbgpu_grad_clip(2, table, n, None, 1.0, 0, 0x1000, ws, room, None) == ENODEVICE
    # beyond the limit the table is not even read
    assert lib.svbgpu_grad_norm(2, C.c_void_p(1 << 12), (1 << 31) + 1, 0x1000, ws, 1 << 40, None) == EINVAL
    assert lib.svbgpu_grad_workspace_bytes((1 << 32) - 1) >= 8 * (4096 + (1 << 32) - 1)


def test_a_given_norm_needs_no_kind_and_no_workspace():
    rows = [(A, 10, F32)]
    for kind in (2, 1, 0, 3, -1):
        assert clip(rows, kind=kind, ws=None, given=1) == ENODEVICE, kind
    assert clip(rows, kind=3) == EINVAL and clip(rows, kind=-1) == EINVAL
