"""The forms of the gradient kernels that sizes, types and cache policy choose between, each against the definitions
(grad_util) and the oracle's streams; and what a GradSet stands for.  Norms within half a float32 step, 2^-24, of the sum
in 64 bits (its own error, at most n * 2^-53, is below 2^-8 of that); everything elementwise bit for bit."""
import math

import numpy as np
import pytest

from grad_util import TYPES, clipped, factor, feedback, norm64, same_bits
from oracle import V1234, V0124
from test_gpu_grad_ops import SETS, close_norm, expected, gradients, guarded, untouched

pytestmark = pytest.mark.gpu
INF = math.inf


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


@pytest.fixture(scope="module")
def codec(torch):
    import streamvbyte_amd as svb
    return svb.DeviceCodec(1 << 16, "cuda:0")


@pytest.fixture(params=[0, 3], ids=["plain", "nontemporal"])
def policy(request):
    """Every access plain, or every access non-temporal, whatever the size."""
    import streamvbyte_amd as svb
    lib = svb.load()
    assert lib.svbgpu_set_option(b"nt_force", request.param) == 0
    yield request.param
    assert lib.svbgpu_set_option(b"nt_force", -1) == 0


@pytest.mark.parametrize("name", list(SETS))
def test_clip_under_either_policy(torch, codec, policy, name):
    import streamvbyte_amd as svb
    sizes, dtypes = SETS[name]
    src, views, buffers = guarded(torch, sizes, dtypes, seed=21)
    _, outs, out_buffers = guarded(torch, sizes, dtypes, seed=22)
    for limit in (0.37, INF):
        norm = codec.clip_grads(svb.GradSet(views, out=outs), limit)
        assert close_norm(norm, norm64(src, 2))
        c = factor(norm.item(), limit)
        for s, v, y in zip(src, views, outs):
            assert same_bits(v, s)
            assert same_bits(y, clipped(s, c)), (s.numel(), s.dtype, limit)
    assert untouched(out_buffers, outs) and untouched(buffers, views)
    norm = codec.clip_grads(views, 0.37)
    for s, v in zip(src, views):
        assert same_bits(v, clipped(s, factor(norm.item(), 0.37)))
    assert untouched(buffers, views)


@pytest.mark.parametrize("p", [2, 1, INF])
def test_a_set_larger_than_the_cache(torch, codec, p):
    """Two launches of the norm and two of the clip.  The last 256 MiB are read to stay in the cache, what is before them is
    not: the reads change within the second launch.  The clip writes elsewhere, with non-temporal stores."""
    import streamvbyte_amd as svb
    gen = torch.Generator(device="cuda").manual_seed(31)
    sizes = [50_000 + 2 * i for i in range(240)] + [1_800_002 + 998 * i for i in range(60)]
    kinds = [torch.float32, torch.float32, torch.bfloat16, torch.float16]
    grads = [torch.randn(n, generator=gen, device="cuda").to(kinds[i % 4]) for i, n in enumerate(sizes)]
    size = [g.numel() * g.element_size() for g in grads]
    first, passing = sum(size[:240]), sum(size) - (256 << 20)
    assert first < passing < sum(size)
    buf = torch.full((sum(size),), 9, dtype=torch.uint8, device="cuda")  # in this order: the library's is that of what is written
    outs = [b.view(g.dtype) for b, g in zip(buf.split(size), grads)]
    kept = [g.clone() for g in grads]
    parts = torch.stack([g.to(torch.float64).abs().max() if p == INF else (g.to(torch.float64).abs() ** p).sum() for g in grads])
    want = float(parts.max()) if p == INF else float(parts.sum()) ** (1.0 / p)
    both = svb.GradSet(grads, out=outs)
    norm = codec.clip_grads(both, want / 5, p)
    assert close_norm(norm, want)
    c = torch.tensor(factor(norm.item(), want / 5), device="cuda")
    for g, k, y in zip(grads, kept, outs):
        assert torch.equal(g, k) and torch.equal(y, (k.to(torch.float32) * c).to(k.dtype))
    assert torch.equal(codec.grad_norm(both, p), norm)
    assert close_norm(codec.grad_norm(grads, p), want)


FORMS = [(3 << 19) + 7, (7 << 19) + 5, (15 << 19) - 5, (15 << 19) + 6, (1 << 24) + 7]


@pytest.mark.parametrize("n", FORMS)
@pytest.mark.parametrize("dtype", list(TYPES))
def test_feedback_forms(torch, oracle, n, dtype):
    """Every type in every tile form, one size each, both variants."""
    import streamvbyte_amd as svb
    codec = svb.DeviceCodec(n, "cuda:0")
    g, r = gradients(torch, n, dtype, seed=n % 997, far=3000.0)
    norm = torch.tensor([1.25], device="cuda")
    q, left = feedback(g, r.numpy(), factor(1.25, 1.0), 64.0)
    left, zz, d_g = torch.from_numpy(left).cuda(), oracle.zigzag_encode(q), g.cuda()
    out = torch.empty((n + 3) // 4 + 4 * n + 16, dtype=torch.uint8, device="cuda")
    for variant in (V0124, V1234):
        want = oracle.encode(variant, zz)
        out.fill_(0xA5)
        d_r = r.cuda()
        _, size, _ = codec.quantize_feedback_encode(d_g, 64.0, d_r, norm=norm, max_norm=1.0, out=out, variant=variant)
        codec.check()
        assert int(size.item()) == want.size
        assert torch.equal(out[:want.size], torch.from_numpy(want).cuda()) and bool((out[want.size:] == 0xA5).all())
        assert torch.equal(d_r.view(torch.int32), left.view(torch.int32))


def test_two_graphs_in_any_order(torch, oracle):
    """Two graphs hold one codec's workspaces; whatever the order, stream and residual are those of the norm that was read."""
    import streamvbyte_amd as svb
    n = 50001
    codec = svb.DeviceCodec(n, "cuda:0")
    side = torch.cuda.Stream()
    parts = []
    for i in range(2):
        g, r = gradients(torch, n - 20000 * i, "f32", seed=400 + i)
        d = dict(g=g.cuda(), r=r.cuda(), new=torch.zeros_like(r).cuda(), norm=torch.zeros(1, device="cuda"),
                 size=torch.zeros(1, dtype=torch.int64, device="cuda"))
        d["out"] = torch.zeros(svb.streamvbyte_max_compressedbytes(g.numel()), dtype=torch.uint8, device="cuda")
        d["set"] = svb.GradSet([d["g"]])
        parts.append((d, g, r))
    graphs = []
    for d, *_ in parts:
        def step():
            codec.grad_norm(d["set"], out=d["norm"])
            z = codec.quantize_feedback_encode(d["g"], 64.0, d["r"], norm=d["norm"], max_norm=0.5, out=d["out"], residual_out=d["new"])[1]
            d["size"].copy_(z)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                step()
        torch.cuda.current_stream().wait_stream(side)
        graphs.append(graph)
    for order in ((0, 1), (1, 0), (1, 1, 0, 0), (0, 1, 0)):
        for d, *_ in parts:
            d["out"].zero_(), d["new"].zero_(), d["norm"].zero_(), d["size"].zero_()
        for i in order:
            graphs[i].replay()
        torch.cuda.synchronize()
        for d, g, r in parts:
            assert close_norm(d["norm"], norm64([g], 2))
            want, left = expected(oracle, V0124, g, r, factor(d["norm"].item(), 0.5), 64.0)
            assert int(d["size"].item()) == want.size and np.array_equal(d["out"][:want.size].cpu().numpy(), want)
            assert same_bits(d["new"], torch.from_numpy(left))
        assert torch.equal(codec.grad_norm([parts[0][0]["g"]]), parts[0][0]["norm"])  # and eager calls in between
    codec.check()


def test_a_set_stands_for_memory(torch, codec):
    """A tensor that is given other memory later is not followed: the set keeps the memory that it was made of, reads and
    writes that, and leaves the tensor's new memory alone.  A set made again takes the new one."""
    import streamvbyte_amd as svb
    x = torch.full((5000,), 2.0, device="cuda")
    first = x.detach()
    kept = svb.GradSet([x])
    x.data = torch.full((5000,), 8.0, device="cuda")
    norm = codec.clip_grads(kept, 1.0)
    assert close_norm(norm, math.sqrt(20000.0))
    assert same_bits(first, clipped(torch.full((5000,), 2.0), factor(norm.item(), 1.0)))
    assert bool((x == 8.0).all())
    # gradients that are dropped and made anew are other tensors
    w = torch.ones(7, device="cuda", requires_grad=True)
    (3.0 * w).sum().backward()
    kept = svb.GradSet([w.grad])
    w.grad = None
    (5.0 * w).sum().backward()
    codec.clip_grads(kept, 1.0)
    assert bool((w.grad == 5.0).all())
    norm = codec.clip_grads([w.grad], 1.0)
    assert close_norm(norm, math.sqrt(7 * 25.0))
    assert same_bits(w.grad, clipped(torch.full((7,), 5.0), factor(norm.item(), 1.0)))
    # zeroed instead, they keep their memory, and the set stays right
    kept = svb.GradSet([w.grad])
    for k in (1.0, 2.0):
        w.grad.zero_()
        (k * w).sum().backward()
        assert close_norm(codec.grad_norm(kept), math.sqrt(7.0) * k)


def test_writes_are_seen_by_autograd(torch, codec):
    import streamvbyte_amd as svb
    w = torch.ones(3000, device="cuda", requires_grad=True)
    for change in (lambda g: codec.clip_grads([g], 1e-3), lambda g: codec.clip_grads(svb.GradSet([w.detach()], out=[g]), 1e-3),
                   lambda g: codec.quantize_feedback_encode(w.detach(), 4.0, g)):
        g = torch.randn(3000, device="cuda")
        loss = (w * g).sum()
        change(g)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    g = torch.randn(3000, device="cuda")
    loss = (w * g).sum()
    codec.grad_norm([g])
    loss.backward()
    assert torch.equal(w.grad, g)
