"""The gradient kernels keep their state in registers: no scratch, and the occupancy their launches count on (sixteen
waves of the encoder a CU; eight a SIMD for the kernels that stream)."""
import os
import re
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_gradient_kernels_do_not_spill():
    out = subprocess.run([sys.executable, os.path.join(ROOT, "tools", "kernel_resources.py"), "--unit", "svb_grad"],
                         capture_output=True, text=True, timeout=600).stdout
    rows = re.findall(r"^(k_\w+)<\S.*?>\s+vgpr=\s*\d+\s+agpr=\s*\d+\s+sgpr=\s*\d+\s+scratch=\s*(\d+)\s+lds=\s*(\d+)\s+occ=(\d+)", out, flags=re.M)
    assert {name for name, *_ in rows} == {"k_grad_norm", "k_grad_finish", "k_grad_scale", "k_grad_small", "k_feedback_encode"}, out[-2000:]
    for name, scratch, lds, occ in rows:
        assert int(scratch) == 0, (name, scratch)
        assert int(lds) <= 160 * 1024
        assert int(occ) >= (4 if name == "k_feedback_encode" else 8), (name, occ)
