"""The encoder with error feedback under hostile timing: the build whose look-back publishes late and out of order
(csrc/svb_lookback.h: lb_stress_delay), in a child process, as in test_gpu_lookback_stress.py."""
import os
import subprocess
import sys

import numpy as np
import pytest

from grad_util import factor, feedback, same_bits
from oracle import V1234, V0124

pytestmark = pytest.mark.gpu
CHILD = os.environ.get("SVB_STRESS_CHILD") == "1"


@pytest.mark.skipif(CHILD, reason="this is the child")
def test_feedback_cases_pass_in_the_stress_build():
    from streamvbyte_amd.build import STRESS_LIB
    assert os.path.exists(STRESS_LIB), "stress build missing: python -m streamvbyte_amd.build"
    env = dict(os.environ, SVB_LIB_PATH=STRESS_LIB, SVB_STRESS_CHILD="1")
    out = subprocess.run([sys.executable, "-m", "pytest", os.path.abspath(__file__), "-x", "-q", "-m", "gpu",
                          "--timeout", "300", "--timeout-method", "thread", "-p", "no:cacheprovider"],
                         env=env, capture_output=True, text=True, timeout=600,
                         cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert out.returncode == 0 and " passed" in out.stdout, (out.stdout[-3000:], out.stderr[-2000:])


@pytest.mark.skipif(not CHILD, reason="runs in the child process, against the stress build")
@pytest.mark.parametrize("n,variant", [(7001, V0124), (700001, V1234), ((1 << 21) + 77, V0124), ((1 << 22) + 5, V1234),
                                       ((1 << 23) + 9, V0124), ((1 << 24) + 1, V0124)])
def test_feedback_is_exact_under_delays(oracle, n, variant):
    import torch
    import streamvbyte_amd as svb
    lib = svb.load()
    assert lib.svbgpu_build_has(b"lookback_stress") == 1, "not the stress build"
    codec = svb.DeviceCodec(n, "cuda:0")
    gen = torch.Generator().manual_seed(n)
    g = (torch.randn(n, generator=gen) * 0.05).to(torch.bfloat16)
    r = (torch.rand(n, generator=gen) - 0.5) / 64
    norm = torch.tensor([3.0], device="cuda")
    q, left = feedback(g, r.numpy(), factor(3.0, 2.0), 64.0)
    want = oracle.encode(variant, oracle.zigzag_encode(q))
    assert lib.svbgpu_set_option(b"debug_ablate", 64) == 0
    try:
        for _ in range(18):  # past the stress build's sixteen look-back tags
            d_r = r.cuda()
            out, size, _ = codec.quantize_feedback_encode(g.cuda(), 64.0, d_r, norm=norm, max_norm=2.0, variant=variant)
            codec.check()
            assert int(size.item()) == want.size and np.array_equal(out[:want.size].cpu().numpy(), want)
            assert same_bits(d_r, torch.from_numpy(left))
    finally:
        lib.svbgpu_set_option(b"debug_ablate", 0)
