"""The gradient operators in numpy: norms in 64 bits, the factor, clipping and error feedback with every rounding of
their definitions (include/streamvbyte_gpu.h)."""
import math

import numpy as np
import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def f64(t):
    return t.detach().cpu().to(torch.float64).numpy().reshape(-1)


def norm64(tensors, p):
    """Norm of all elements in 64 bits, sums exactly rounded."""
    parts = [f64(t) for t in tensors]
    x = np.abs(np.concatenate(parts)) if parts else np.zeros(0)
    if not x.size:
        return 0.0
    if np.isnan(x).any():
        return math.nan
    if p == math.inf:
        return float(x.max())
    if np.isinf(x).any():
        return math.inf
    return math.sqrt(math.fsum(x * x)) if p == 2 else math.fsum(x)


def factor(norm32, limit):
    n = np.float64(np.float32(norm32)) + 1e-6
    if n <= limit:
        return np.float32(1.0)
    with np.errstate(invalid="ignore"):
        return np.float32(np.float64(limit) / n)


def to_type(x32, dtype):
    """float32 array -> tensor of the type, rounded to nearest even"""
    return torch.from_numpy(np.ascontiguousarray(x32, dtype=np.float32)).to(dtype)


def clipped(t, c):
    """t * c, rounded to float32 and then to t's type."""
    with np.errstate(all="ignore"):
        x = t.detach().cpu().to(torch.float32).numpy().reshape(-1) * np.float32(c)
    return to_type(x, t.dtype)


def feedback(g, r, c, scale):
    """(q int32, new residual float32) of the flattened gradient g."""
    with np.errstate(all="ignore"):
        g = g.detach().cpu().to(torch.float32).numpy().reshape(-1)
        r = np.asarray(r, dtype=np.float32)
        scale, one = np.float32(scale), np.float32(1.0)
        step = one / scale
        e = (g * np.float32(c)).astype(np.float32) + r
        f = np.rint(e * scale)
        finite = np.isfinite(e)
        f = np.where(finite, f, np.float32(0))
        q = np.where(f >= np.float32(2.0 ** 31), 2 ** 31 - 1, np.maximum(f, np.float32(-2.0 ** 31)).astype(np.float64)).astype(np.int64)
        q = q.astype(np.int32)
        left = e - q.astype(np.float32) * step
        return q, np.where(finite, left, r).astype(np.float32)


def same_bits(a, b):
    """Bitwise equality of two tensors of one type, any NaN equal to any other."""
    a, b = a.detach().cpu().reshape(-1), b.detach().cpu().reshape(-1)
    assert a.dtype == b.dtype and a.shape == b.shape
    nan = torch.isnan(a) & torch.isnan(b)
    kind = torch.int32 if a.dtype == torch.float32 else torch.int16
    return bool(((a.view(kind) == b.view(kind)) | nan).all())
