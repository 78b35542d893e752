"""The gradient operators, as they are measured: the global norm of many tensors, clipping by it, and the
quantising encoder that carries its error over to the next step.

With `own` false, `run` computes them in elementary torch operations; with `own` true it makes the calls a
training program makes of streamvbyte_amd.  Both sides get what `prepare` returns.

The shapes: `flat` is one bucket of gradients, as data-parallel training keeps them; `layers` the separate weight
gradients of a decoder stack (attention projections, a gated feed-forward, two norms a layer, an embedding);
`ragged` many tensors of all sizes, most of them small, as biases, norms and adapters are.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
MIXED = ("f32", "bf16", "f16")
LARGEST = 1 << 28  # values of the repository's longest stream
LARGEST_FEEDBACK = 1 << 26  # values of its gradient workload
EPS = 1e-6  # added to the norm before it divides


def listed():
    return [
        # the norm of a handful of small tensors (the head of a model, a probe): latency is all there is
        {"name": "norm_few", "op": "norm", "set": "ragged", "tensors": 4, "n": 1021, "shapes": 1, "dtype": "f32", "p": 2.0},
        # a decoder stack's weight gradients as the backward pass leaves them, one tensor per weight
        {"name": "norm_layers", "op": "norm", "set": "layers", "layers": 12, "hidden": 1024, "ff": 2816, "vocab": 32000,
         "dtype": "bf16", "p": 2.0},
        # several hundred adapters, biases and norms in mixed types; the largest entry instead of the sum
        {"name": "norm_ragged_max", "op": "norm", "set": "ragged", "tensors": 613, "n": 65521, "shapes": 2, "dtype": "mixed",
         "p": math.inf},
        # one flat float32 bucket of the repository's full stream length
        {"name": "norm_flat", "op": "norm", "set": "flat", "n": 1 << 28, "dtype": "f32", "p": 2.0},
        # clipping the same four kinds; into other tensors, so that a pass can be repeated on the same gradients
        {"name": "clip_few", "op": "clip", "set": "ragged", "tensors": 5, "n": 2039, "shapes": 3, "dtype": "f32", "p": 2.0,
         "limit": 0.25},
        {"name": "clip_layers", "op": "clip", "set": "layers", "layers": 12, "hidden": 1024, "ff": 2816, "vocab": 32000,
         "dtype": "bf16", "p": 2.0, "limit": 0.25},
        {"name": "clip_ragged", "op": "clip", "set": "ragged", "tensors": 613, "n": 65521, "shapes": 4, "dtype": "mixed", "p": 2.0,
         "limit": 0.25},
        {"name": "clip_flat", "op": "clip", "set": "flat", "n": (1 << 28) - 5, "dtype": "f32", "p": 2.0, "limit": 0.25},
        # the gradient workload of the repository's benchmark (2^26 values, most of them 0 after quantising), clipped on the way
        {"name": "feedback_f32", "op": "feedback", "n": 1 << 26, "dtype": "f32", "variant": 1, "limit": 0.25},
        # a bfloat16 bucket of odd length, one byte a value at least
        {"name": "feedback_bf16", "op": "feedback", "n": (1 << 24) + 3, "dtype": "bf16", "variant": 0, "limit": 0.25},
        # one mid-sized weight
        {"name": "feedback_f16", "op": "feedback", "n": 1024 * 2816 + 1, "dtype": "f16", "variant": 1, "limit": 64.0},
        # a bias: latency again
        {"name": "feedback_few", "op": "feedback", "n": 4099, "dtype": "f32", "variant": 1, "limit": 0.25},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(("norm", "clip", "feedback"))
    limit = rng.choice((0.015625, 0.25, 1.0, 64.0))  # far below, below, near and above the norms that prepare makes
    if op == "feedback":
        return {"op": op, "n": _log_int(rng, 1, LARGEST_FEEDBACK), "dtype": rng.choice(MIXED), "variant": rng.randint(0, 1),
                "limit": limit}
    case = {"op": op, "set": rng.choice(("flat", "layers", "ragged")), "dtype": rng.choice(MIXED + ("mixed",)),
            "p": rng.choice((2.0, 2.0, 1.0, math.inf))}
    if case["set"] == "flat":
        case["n"] = _log_int(rng, 1, LARGEST - 5)
        if case["dtype"] == "mixed":
            case["dtype"] = "f32"
    elif case["set"] == "layers":
        hidden = 64 * _log_int(rng, 1, 24)
        ff, vocab = 8 * rng.randint(hidden // 8, hidden // 2), _log_int(rng, 128, 32000)
        fit = (LARGEST - 5 - vocab * hidden - hidden) // (4 * hidden * hidden + 3 * hidden * ff + 2 * hidden)
        case.update(layers=min(_log_int(rng, 1, 16), fit), hidden=hidden, ff=ff, vocab=vocab)
    else:
        case.update(tensors=_log_int(rng, 1, 1500), n=_log_int(rng, 1, 100000), shapes=rng.randint(0, 1 << 20))
    if op == "clip":
        case["limit"] = limit
    return case


def _counts(case):
    """Elements of every tensor of the set."""
    if case["op"] == "feedback" or case["set"] == "flat":
        return [case["n"]]
    if case["set"] == "layers":
        h, f = case["hidden"], case["ff"]
        return [case["vocab"] * h] + [h * h, h * h, h * h, h * h, h * f, h * f, f * h, h, h] * case["layers"] + [h]
    rng = random.Random(case["shapes"])
    return [_log_int(rng, 1, case["n"]) for _ in range(case["tensors"])]


def _types(case, tensors):
    return [case["dtype"] if case["dtype"] != "mixed" else MIXED[i % 3] for i in range(tensors)]


def work(case):
    counts = _counts(case)
    total = sum(counts)
    inputs = sum(c * BYTES[t] for c, t in zip(counts, _types(case, len(counts))))
    if case["op"] == "norm":
        return {"bytes": inputs + 4, "flops": 2 * total}
    if case["op"] == "clip":
        return {"bytes": 2 * inputs + 4, "flops": 3 * total}
    data = 0.6 if case["variant"] == 1 else 1.0  # bytes a value, as the inputs of prepare come out
    return {"bytes": int(inputs + 8 * total + (total + 3) // 4 + data * total), "flops": 8 * total}


class _State:
    pass


def _buckets(tensors, make=None):
    """The tensors of each type one behind the other (or what `make` makes of that)."""
    out = []
    for t in DTYPES.values():
        of_type = [x for x in tensors if x.dtype == t]
        if of_type:
            out.append(torch.cat(of_type) if make is None else make(torch.cat(of_type)))
    return out


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed * 1000003 + 17)
    s = _State()
    s.case = case
    counts = _counts(case)
    total = sum(counts)
    if case["op"] == "feedback":
        # most gradients below the quantisation step 1/64, one in a thousand far above it; the residual of earlier steps
        n = case["n"]
        g = torch.randn(n, generator=gen, device=dev) * (0.8 / 64)
        far = torch.rand(n, generator=gen, device=dev) < 0.001
        g = torch.where(far, g * 16384.0, g) if case["dtype"] != "f16" else torch.where(far, g * 1024.0, g)
        s.grad = g.to(DTYPES[case["dtype"]])
        s.residual = (torch.rand(n, generator=gen, device=dev) - 0.5) / 64
        s.scale = 64.0
        # a norm near the limits that are drawn: the factor is below 1 for the small limits, 1 for the largest
        s.norm = 0.3 + torch.rand(1, generator=gen, device=dev)
        bytes_out = (n + 3) // 4 + 4 * n + 16
        s.stream = torch.zeros(bytes_out, dtype=torch.uint8, device=dev)
        s.residual_out = torch.zeros(n, device=dev)
        if own:
            import streamvbyte_amd as svb
            s.codec = svb.DeviceCodec(n)
        return s
    # tensors of different magnitude whose 2-norm comes out at about 1
    scale = 1.0 / math.sqrt(max(total, 1))
    s.grads = []
    for c, t in zip(counts, _types(case, len(counts))):
        k = (0.5 + torch.rand(1, generator=gen, device=dev)) * scale
        s.grads.append((torch.randn(c, generator=gen, device=dev) * k).to(DTYPES[t]))
    s.limit = case.get("limit", 0.0)
    if case["p"] == 1.0:
        s.limit *= math.sqrt(max(total, 1))  # the 1-norm of the same tensors is that much larger
    elif case["p"] == math.inf:
        s.limit *= 4.0 * scale
    if case["op"] == "clip":
        # the clipped gradients lie in one bucket a type, one behind the other: what the exchange takes
        s.buckets = _buckets(s.grads, torch.empty_like)
        room = {b.dtype: list(b.split([g.numel() for g in s.grads if g.dtype == b.dtype])) for b in s.buckets}
        s.clipped = [room[g.dtype].pop(0) for g in s.grads]
    if own:
        import streamvbyte_amd as svb
        s.codec = svb.DeviceCodec(1)
        s.set = svb.GradSet(s.grads, out=s.clipped) if case["op"] == "clip" else svb.GradSet(s.grads)
    return s


# ---- plain forms --------------------------------------------------------------------------------------
def _plain_norm(grads, p):
    parts = []
    for g in grads:
        x = g.to(torch.float32).abs()
        if p == math.inf:
            parts.append(x.max().to(torch.float64))
        elif p == 1.0:
            parts.append(x.sum(dtype=torch.float64))
        else:
            d = x.to(torch.float64)
            parts.append((d * d).sum())
    parts = torch.stack(parts)
    if p == math.inf:
        return parts.max().reshape(1).to(torch.float32)
    total = parts.sum().reshape(1)
    return (total if p == 1.0 else total.sqrt()).to(torch.float32)


def _plain_factor(norm, limit):
    n = norm.to(torch.float64) + EPS
    return torch.where(n <= limit, torch.ones_like(n), limit / n).to(torch.float32)


def _plain_clip(grads, clipped, buckets, limit, p):
    norm = _plain_norm(grads, p)
    c = _plain_factor(norm, limit)
    for g, y in zip(grads, clipped):
        y.copy_(g.to(torch.float32) * c)
    return norm, buckets


def _plain_feedback(grad, residual, scale, norm, limit, variant):
    n = grad.numel()
    c = _plain_factor(norm, limit)
    e = grad.to(torch.float32) * c
    e = e + residual
    f = torch.round(e * scale)
    top = f >= 2147483648.0
    finite = torch.isfinite(e)
    q = torch.where(finite, f, torch.zeros_like(f)).clamp(min=-2147483648.0, max=2147483520.0).to(torch.int64)
    q = torch.where(top & finite, torch.full_like(q, 2147483647), q)
    r = torch.where(finite, e - q.to(torch.float32) * (1.0 / scale), residual)  # the scale is a power of two
    u = torch.where(q < 0, -2 * q - 1, 2 * q)
    if variant == 1:
        code = (u > 0).to(torch.int64) + (u > 0xFF) + (u > 0xFFFF)
        size = (1 << code) >> 1
    else:
        code = (u > 0xFF).to(torch.int64) + (u > 0xFFFF) + (u > 0xFFFFFF)
        size = code + 1
    keys = (n + 3) // 4
    padded = torch.zeros(4 * keys, dtype=torch.int64, device=grad.device)
    padded[:n] = code
    k = padded.view(keys, 4)
    room = keys + 4 * n + 16
    out = torch.zeros(room + 1, dtype=torch.uint8, device=grad.device)
    out[:keys] = (k[:, 0] + 4 * k[:, 1] + 16 * k[:, 2] + 64 * k[:, 3]).to(torch.uint8)
    ends = torch.cumsum(size, 0)
    start = ends - size + keys
    for b in range(4):  # bytes that a value does not have go to the one place past the end
        out.scatter_(0, torch.where(size > b, start + b, torch.full_like(start, room)), ((u >> (8 * b)) & 255).to(torch.uint8))
    return out[:room], (ends[-1:] + keys), r


def run(state):
    case = state.case
    if case["op"] == "norm":
        return state.codec.grad_norm(state.set, case["p"]) if own else _plain_norm(state.grads, case["p"])
    if case["op"] == "clip":
        if own:
            return state.codec.clip_grads(state.set, state.limit, case["p"]), state.buckets
        return _plain_clip(state.grads, state.clipped, state.buckets, state.limit, case["p"])
    if own:
        return state.codec.quantize_feedback_encode(state.grad, state.scale, state.residual, norm=state.norm, max_norm=case["limit"],
                                                    out=state.stream, residual_out=state.residual_out, variant=case["variant"])
    return _plain_feedback(state.grad, state.residual, state.scale, state.norm, case["limit"], case["variant"])


# ---- the definition in 64 bits ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] != "feedback":
        p = case["p"]
        total = 0.0
        for g in s.grads:
            for piece in g.split(1 << 25):
                v = float(torch.linalg.vector_norm(piece.to(torch.float64), p))
                total = max(total, v) if p == math.inf else total + (v * v if p == 2.0 else v)
        norm = math.sqrt(total) if p == 2.0 else total
        norm_out = torch.tensor([norm], dtype=torch.float64, device="cuda")
        if case["op"] == "norm":
            return norm_out
        c = min(1.0, s.limit / (norm + EPS))
        return norm_out, [b.to(torch.float64) * c for b in _buckets(s.grads)]
    if case["n"] > 1 << 25:
        return None
    # every rounding of the definition, on the host
    import numpy as np
    n = case["n"]
    norm = float(s.norm.item()) + EPS
    c = np.float64(np.float32(1.0 if norm <= case["limit"] else case["limit"] / norm))
    g = s.grad.to(torch.float64).cpu().numpy()
    r = s.residual.cpu().numpy().astype(np.float64)
    e = ((g * c).astype(np.float32).astype(np.float64) + r).astype(np.float32).astype(np.float64)
    q = np.clip(np.rint((e * s.scale).astype(np.float32).astype(np.float64)), -2.0 ** 31, 2.0 ** 31 - 1).astype(np.int64)
    left = e - q.astype(np.float32).astype(np.float64) / s.scale
    u = ((q << 1) ^ (q >> 63)).astype(np.uint32)
    widths = np.zeros(n, dtype=np.int64)
    for bits in (0, 8, 16) if case["variant"] == 1 else (8, 16, 24):
        widths += (u.astype(np.uint64) >> np.uint64(bits)) > 0
    lengths = np.array([0, 1, 2, 4] if case["variant"] == 1 else [1, 2, 3, 4])[widths]
    codes = np.zeros(-(-n // 4) * 4, dtype=np.uint8)
    codes[:n] = widths
    keys = (codes.reshape(-1, 4) << np.array([0, 2, 4, 6], dtype=np.uint8)).sum(axis=1).astype(np.uint8)
    data = u.astype("<u4").view(np.uint8).reshape(n, 4)[np.arange(4)[None, :] < lengths[:, None]]
    stream = np.zeros(keys.size + 4 * n + 16, dtype=np.uint8)
    stream[:keys.size] = keys
    stream[keys.size:keys.size + data.size] = data
    size = torch.tensor([keys.size + data.size], dtype=torch.int64, device="cuda")
    return torch.from_numpy(stream).cuda(), size, torch.from_numpy(left).cuda()
