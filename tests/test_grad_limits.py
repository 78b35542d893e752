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
