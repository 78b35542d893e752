"""Gradient operators on the device: norm over many tensors, clipping, the encoder with error feedback -- against the
numpy forms of grad_util (64-bit norms; every rounding of the elementwise definitions) and the oracle's streams.

Tolerances: a norm is one rounding to float32 of a sum in 64 bits, so at most half a float32 step off, 2^-24 of it; the
64-bit sum of n terms adds at most n * 2^-53 of it, 2^-33 for the largest n here, which the factor 1 + 2^-8 covers.
Everything elementwise is defined to the last rounding and has to be equal bit for bit."""
import math

import numpy as np
import pytest

from grad_util import HALF_STEP, TYPES, clipped, factor, f64, feedback, norm64, same_bits, to_type
from oracle import V1234, V0124

pytestmark = pytest.mark.gpu
NORM_TOL = 2.0 ** -24 * (1 + 2.0 ** -8)
CHUNK = 64 * 1024  # bytes of the smallest piece a workgroup takes
INF = math.inf


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


@pytest.fixture(scope="module")
def codec(torch):
    import streamvbyte_amd as svb
    return svb.DeviceCodec(1 << 21, "cuda:0")


def make(torch, sizes, dtypes, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * spread * (1 + i % 3)).to(TYPES[dtypes[i % len(dtypes)]]).cuda() for i, n in enumerate(sizes)]


def close_norm(got, want):
    got = float(got)
    if math.isnan(want):
        return math.isnan(got)
    if want >= 2.0 ** 128 - 2.0 ** 103:  # rounds past the largest float32
        return got == INF
    return abs(got - want) <= NORM_TOL * want


SETS = {
    "none": ([], ["f32"]),
    "empty": ([0, 0], ["f32", "bf16"]),
    "one": ([1], ["f32"]),
    "one_between_empties": ([0, 1, 0], ["f16"]),
    "vector_edges": ([1, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 33], ["f32", "f16", "bf16"]),
    "chunk_edges_f32": ([CHUNK // 4 - 1, CHUNK // 4, CHUNK // 4 + 1, 2 * CHUNK // 4 + 3], ["f32"]),
    "chunk_edges_16": ([CHUNK // 2 - 1, CHUNK // 2, CHUNK // 2 + 1, CHUNK + 5], ["bf16", "f16"]),
    "table_edges": ([5 + i % 11 for i in range(160)], ["f32", "bf16"]),
    "over_one_table": ([3 + i % 17 for i in range(161)], ["bf16", "f32", "f16"]),
    "over_two_tables": ([1 + (i * 37) % 301 for i in range(481)], ["f16", "f32", "bf16"]),
    # the set that one workgroup still takes, and the first that it does not
    "small_by_bytes": ([CHUNK], ["f32"]),
    "beyond_small_by_bytes": ([CHUNK + 1], ["f32"]),
    "small_by_tensors": ([1 + 16 * i for i in range(64)], ["f32", "f16"]),
    "beyond_small_by_tensors": ([1 + 16 * i for i in range(65)], ["f32", "f16"]),
    "beyond_small_by_chunks": ([1025] * 33, ["f32"]),
    "small_chunk_edges": ([1023, 1024, 1025, 2047, 2048, 2049, 4097], ["f32", "bf16"]),
    "with_holes": ([0 if i % 5 == 0 else i for i in range(300)], ["f32"]),
    "weights": ([1 << 20, 1024, 300007, 1, 65537], ["bf16", "f32"]),
}


@pytest.mark.parametrize("p", [2, 1, INF])
@pytest.mark.parametrize("name", list(SETS))
def test_norm(torch, codec, name, p):
    sizes, dtypes = SETS[name]
    grads = make(torch, sizes, dtypes, seed=len(name))
    want = norm64(grads, p)
    got = codec.grad_norm(grads, p)
    assert got.shape == (1,) and got.dtype == torch.float32
    assert close_norm(got, want), (float(got), want)
    if p == INF:
        assert float(got) == want  # a maximum is not rounded
    assert torch.equal(got, codec.grad_norm(grads, p)), "another result the second time"


@pytest.mark.parametrize("dtype", list(TYPES))
def test_norm_of_extremes(torch, codec, dtype):
    """Squares of the largest and of the smallest numbers neither overflow nor vanish; infinities and NaN come out."""
    t = TYPES[dtype]
    top, tiny = torch.finfo(t).max, torch.finfo(t).smallest_normal
    smallest = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}[dtype]  # subnormal
    for n in (1, 8, 9, 70001):
        x = torch.zeros(n, dtype=t)
        for value in (top / 512, tiny, smallest):
            x.fill_(value)
            for p in (2, 1, INF):
                want = norm64([x], p)
                got = codec.grad_norm([x.cuda()], p)
                if want < 2.0 ** -126:  # a subnormal result: half a step of the smallest numbers
                    assert abs(float(got) - want) <= 2.0 ** -150, (n, value, p)
                else:
                    assert close_norm(got, want), (n, value, p, float(got), want)
        x.fill_(1.0)
        for place in (0, n // 2, n - 1):
            for bad in (INF, -INF, math.nan):
                y = x.clone()
                y[place] = bad
                for p in (2, 1, INF):
                    got = float(codec.grad_norm([x.cuda(), y.cuda(), x.cuda()], p))
                    assert math.isnan(got) if math.isnan(bad) else got == INF, (n, place, bad, p)
    if dtype == "f32":  # beyond float32: infinite, not wrapped
        x = torch.full((16,), top, dtype=t).cuda()
        assert float(codec.grad_norm([x], 2)) == INF and float(codec.grad_norm([x], INF)) == top


def test_norm_takes_overlapping_and_strided_tensors(torch, codec):
    base = torch.randn(64, 48).cuda()
    views = [base, base, base.t(), base[3:9], base.view(-1)[5:2000], base.view(4, 16, 6, 8).permute(2, 0, 3, 1)]
    assert close_norm(codec.grad_norm(views), norm64(views, 2))
    for dtype in TYPES.values():  # aligned to the element and to nothing more
        x = torch.randn(70003).to(dtype).cuda()
        for off in range(1, 9):
            assert close_norm(codec.grad_norm([x[off:], x[:off]]), norm64([x], 2)), (dtype, off)


def guarded(torch, sizes, dtypes, seed):
    """Tensors with sentinel elements around each, all in one buffer a type, starts off every alignment."""
    src = make(torch, sizes, dtypes, seed, spread=3.0)
    views, buffers = [], []
    for i, t in enumerate(src):
        lead = 9 + i % 8
        buf = torch.full((t.numel() + lead + 16,), 7.0, dtype=t.dtype, device="cuda")
        buf[lead:lead + t.numel()] = t
        views.append(buf[lead:lead + t.numel()])
        buffers.append((buf, lead))
    return src, views, buffers


def untouched(buffers, views):
    return all(bool((b[:lead] == 7.0).all()) and bool((b[lead + v.numel():] == 7.0).all()) for (b, lead), v in zip(buffers, views))


@pytest.mark.parametrize("limit", [0.0, 0.37, 1e9, INF])
@pytest.mark.parametrize("name", list(SETS))
def test_clip(torch, codec, name, limit):
    import streamvbyte_amd as svb
    sizes, dtypes = SETS[name]
    src, views, buffers = guarded(torch, sizes, dtypes, seed=3)
    outs_src, outs, out_buffers = guarded(torch, sizes, dtypes, seed=4)
    # into other tensors first: the gradients stay
    norm = codec.clip_grads(svb.GradSet(views, out=outs), limit)
    assert close_norm(norm, norm64(src, 2))
    c = factor(norm.item(), limit)
    for s, v, y in zip(src, views, outs):
        assert same_bits(v, s)
        assert same_bits(y, clipped(s, c)), (s.numel(), s.dtype)
    assert untouched(out_buffers, outs)
    # in place: the same bits
    norm2 = codec.clip_grads(views, limit)
    assert torch.equal(norm, norm2)
    for v, y in zip(views, outs):
        assert same_bits(v, y)
    assert untouched(buffers, views)


@pytest.mark.parametrize("p", [1, INF])
def test_clip_by_other_norms(torch, codec, p):
    src = make(torch, [1000, 3, 70001], ["f32", "f16", "bf16"], seed=9)
    grads = [t.clone() for t in src]
    want = norm64(src, p)
    norm = codec.clip_grads(grads, want / 3, p)
    assert close_norm(norm, want)
    for s, g in zip(src, grads):
        assert same_bits(g, clipped(s, factor(norm.item(), want / 3)))
        # and the value itself: factor, product and type are a rounding each, over a norm that is one off already
        exact = f64(s) / 3 * want / (want + 1e-6)
        tol = 3 * 2.0 ** -24 + HALF_STEP[s.dtype]
        small = np.abs(exact) < {2.0 ** -24: 2.0 ** -120, 2.0 ** -11: 2.0 ** -13, 2.0 ** -8: 2.0 ** -120}[HALF_STEP[s.dtype]]
        assert (np.abs(f64(g) - exact) <= np.where(small, 2.0 ** -24, tol * np.abs(exact))).all()


def test_clip_with_a_norm_that_is_given(torch, codec):
    """A rank that holds a shard clips by the norm of all: what is read is the tensor, and it stays."""
    src = make(torch, [5000, 77], ["f32", "bf16"], seed=11)
    for value in (0.0, 1.0, 1.0 - 1e-6, 3.5, 1e30, INF, math.nan):
        grads = [t.clone() for t in src]
        given = torch.tensor([value], dtype=torch.float32, device="cuda")
        back = codec.clip_grads(grads, 1.0, norm=given)
        assert back is given and same_bits(given, torch.tensor([value], dtype=torch.float32))
        for s, g in zip(src, grads):
            assert same_bits(g, clipped(s, factor(value, 1.0))), value


def test_a_given_norm_and_outputs(torch, codec):
    """The two together, on a set larger and one smaller than one workgroup takes."""
    import streamvbyte_amd as svb
    for sizes in ([700, 3], [90001, 17, 4096], [2, 5] * 100):
        src = make(torch, sizes, ["bf16", "f32", "f16"], seed=len(sizes))
        keep = [t.clone() for t in src]
        outs = [torch.full_like(t, 9.0) for t in src]
        given = torch.tensor(7.0, device="cuda")  # without a dimension
        codec.clip_grads(svb.GradSet(src, out=outs), 2.0, norm=given)
        for k, t, y in zip(keep, src, outs):
            assert same_bits(t, k) and same_bits(y, clipped(k, factor(7.0, 2.0)))


def test_what_the_methods_refuse(torch, codec):
    import streamvbyte_amd as svb
    x, h = torch.randn(100).cuda(), torch.randn(64, 64).cuda()
    keep = x.clone()
    for wrong in ([x, x], [x, x[10:20]], [h[:8], h[7:]]):
        with pytest.raises(svb.SvbError, match="invalid argument"):
            codec.clip_grads(wrong, 1e-3)
    for wrong in ([h[:, 3]], [h[::2]], [x[:1].expand(9)], [x.double()], [x.int()], [x.cpu()], [torch.eye(4).to_sparse().cuda()]):
        for call in (codec.grad_norm, lambda g: codec.clip_grads(g, 1.0)):
            with pytest.raises(ValueError):
                call(wrong)
    for p in (0, 3, -1, "fro"):
        with pytest.raises(ValueError):
            codec.grad_norm([x], p)
    for limit in (-1.0, math.nan):
        with pytest.raises(ValueError):
            codec.clip_grads([x], limit)
    for out in ([h], [x, x], [x.half()], [torch.empty(50, 2, device="cuda")]):
        with pytest.raises(ValueError):
            svb.GradSet([x], out=out)
    with pytest.raises(svb.SvbError):  # shifted against itself
        codec.clip_grads(svb.GradSet([x[:50]], out=[x[1:51]]), 1e-3)
    for norm in (torch.zeros(2, device="cuda"), torch.zeros(1), torch.zeros(1, device="cuda", dtype=torch.float64)):
        with pytest.raises(ValueError):
            codec.clip_grads([x], 1.0, norm=norm)
        with pytest.raises(ValueError):
            codec.grad_norm([x], out=norm)
    r = torch.zeros(100, device="cuda")
    for change in (dict(grad=x.double()), dict(grad=x[::2]), dict(residual=r[:50]), dict(residual=r.half()), dict(residual=r.cpu()),
                   dict(out=torch.empty(10, dtype=torch.uint8, device="cuda")), dict(out=torch.empty(1000, device="cuda")),
                   dict(residual_out=r[1:]), dict(norm=torch.zeros(2, device="cuda")), dict(grad=torch.zeros((1 << 21) + 1, device="cuda"))):
        with pytest.raises(ValueError):
            codec.quantize_feedback_encode(**dict(dict(grad=x, scale=64.0, residual=r), **change))
    for change in (dict(scale=0.0), dict(scale=-1.0), dict(scale=INF), dict(variant=2), dict(residual=x), dict(norm=r[5:6], max_norm=1.0),
                   dict(norm=torch.ones(1, device="cuda"), max_norm=-1.0)):
        with pytest.raises(svb.SvbError):
            codec.quantize_feedback_encode(**dict(dict(grad=x, scale=64.0, residual=r), **change))
    torch.cuda.synchronize()
    assert torch.equal(x, keep) and not bool(r.any())  # nothing ran


def test_clip_of_what_is_not_finite(torch, codec):
    for bad in (INF, math.nan):
        src = make(torch, [100, 33000], ["f32", "f16"], seed=12)
        src[1][32999] = bad
        grads = [t.clone() for t in src]
        norm = codec.clip_grads(grads, 1.0)
        assert math.isnan(norm.item()) if math.isnan(bad) else norm.item() == INF
        for s, g in zip(src, grads):
            assert same_bits(g, clipped(s, factor(bad, 1.0)))
        if bad == INF:  # an infinite limit leaves even that alone
            grads = [t.clone() for t in src]
            codec.clip_grads(grads, INF)
            assert all(same_bits(s, g) for s, g in zip(src, grads))


def test_clip_output_may_be_the_tensor_itself(torch, codec):
    import streamvbyte_amd as svb
    src = make(torch, [4097, 9], ["bf16", "f32"], seed=13)
    a, b = [t.clone() for t in src], [t.clone() for t in src]
    other = torch.empty_like(b[1])
    codec.clip_grads(a, 0.5)
    codec.clip_grads(svb.GradSet(b, out=[b[0], other]), 0.5)
    assert same_bits(a[0], b[0]) and same_bits(a[1], other) and same_bits(b[1], src[1])


def test_clip_of_permuted_tensors(torch, codec):
    x = torch.randn(6, 5, 7).cuda()
    y = x.clone().permute(2, 0, 1)
    codec.clip_grads([y], 1.0)
    n = codec.grad_norm([x])
    assert same_bits(y.permute(1, 2, 0).contiguous(), clipped(x, factor(n.item(), 1.0)))


def test_set_is_refused_after_a_tensor_moved(torch, codec):
    import streamvbyte_amd as svb
    x = torch.randn(100).cuda()
    s = svb.GradSet([x])
    x.data = torch.zeros(100, device="cuda")  # the set still holds the tensor it was made of
    assert float(codec.grad_norm(s)) > 0
    s.tensors[0].untyped_storage().resize_(0)
    with pytest.raises(ValueError, match="moved"):
        codec.grad_norm(s)


@pytest.mark.parametrize("case", [("f32", (1 << 30) + 7), ("bf16", (1 << 31) + 9)])
def test_offsets_past_32_bits(torch, codec, case):
    """A tensor of more than 4 GiB: everything counts once, and its ends are scaled."""
    dtype, n = case
    x = torch.full((n,), 2.0, dtype=TYPES[dtype], device="cuda")
    x[-3:] = 1024.0
    total = 4.0 * (n - 3) + 3 * 1024.0 ** 2
    assert close_norm(codec.grad_norm([x]), math.sqrt(total))
    assert float(codec.grad_norm([x], INF)) == 1024.0
    norm = codec.clip_grads([x], math.sqrt(total) / 4)
    c = factor(norm.item(), math.sqrt(total) / 4)
    two, far = clipped(torch.full((1,), 2.0, dtype=TYPES[dtype]), c).cuda(), clipped(torch.full((1,), 1024.0, dtype=TYPES[dtype]), c).cuda()
    assert bool((x[:-3] == two).all()) and bool((x[-3:] == far).all())


# ---- quantise with feedback -------------------------------------------------------------------------------
def gradients(torch, n, dtype, seed, far=300.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, generator=g) * 0.02
    x = torch.where(torch.rand(n, generator=g) < 0.01, x * far, x).to(TYPES[dtype])
    r = (torch.rand(n, generator=g) - 0.5) / 64
    return x, r


def expected(oracle, variant, g, r, c, scale):
    q, left = feedback(g, r.numpy(), c, scale)
    return oracle.encode(variant, oracle.zigzag_encode(q)), left


@pytest.mark.parametrize("variant", [V0124, V1234])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_feedback_encode(torch, codec, oracle, dtype, variant):
    sizes = (0, 1, 2, 3, 4, 5, 63, 255, 257, 1023, 1024, 1025, 2047, 2049, 4095, 16383, 16384, 16385, 32767, 32769, 100003, 300000, (1 << 20) + 5)
    for k, n in enumerate(sizes):
        scale = (64.0, 7.5, 1000.0)[k % 3]
        g, r = gradients(torch, n, dtype, seed=n + variant)
        limit, value = ((INF, None), (1.0, 3.7), (5.0, 3.7))[k % 3]
        c = np.float32(1.0) if value is None else factor(value, limit)
        want, left = expected(oracle, variant, g, r, c, scale)
        norm = None if value is None else torch.tensor([value], device="cuda")
        room = (n + 3) // 4 + 4 * n + 16
        buf = torch.full((room + 64,), 0xA5, dtype=torch.uint8, device="cuda")
        lead = k % 7  # streams start anywhere
        d_g = torch.full((n + 8,), 1.0, dtype=TYPES[dtype], device="cuda")
        d_g[k % 3:k % 3 + n] = g.cuda()
        d_r, d_new = r.cuda(), torch.full((n + 4,), 9.0, device="cuda")
        out, size, new = codec.quantize_feedback_encode(d_g[k % 3:k % 3 + n], scale, d_r, norm=norm, max_norm=limit,
                                                        out=buf[lead:lead + room], residual_out=d_new[1:1 + n], variant=variant)
        codec.check()
        assert int(size.item()) == want.size, n
        host = buf.cpu().numpy()
        assert np.array_equal(host[lead:lead + want.size], want), n
        assert (host[:lead] == 0xA5).all() and (host[lead + want.size:] == 0xA5).all(), n  # nothing but the stream
        assert same_bits(new, torch.from_numpy(left)), n
        assert d_new[0] == 9.0 and bool((d_new[1 + n:] == 9.0).all()) and same_bits(d_r, r)
        # in place
        out, size, new = codec.quantize_feedback_encode(d_g[k % 3:k % 3 + n], scale, d_r, norm=norm, max_norm=limit, variant=variant)
        assert new is d_r and int(size.item()) == want.size and same_bits(d_r, torch.from_numpy(left))
        assert np.array_equal(out[:want.size].cpu().numpy(), want)


@pytest.mark.parametrize("n,dtype,variant", [
    ((1 << 19) - 1, "f32", V0124), (1 << 19, "f16", V1234), ((3 << 19) - 1, "bf16", V0124), ((3 << 19) + 3, "f32", V1234),
    ((7 << 19) - 1, "f32", V0124), (7 << 19, "f16", V0124), ((6 << 20) - 2, "bf16", V1234), ((6 << 20) + 1, "f32", V0124),
    ((15 << 19) - 3, "f32", V0124), ((15 << 19) + 1, "f32", V1234), ((15 << 19) + 2, "f16", V0124),
    ((1 << 24) - 1, "bf16", V0124), ((1 << 24) + 5, "f32", V0124), ((1 << 24) + 30719, "bf16", V1234)])
def test_feedback_of_every_tile_shape(torch, oracle, n, dtype, variant):
    """The tile, the waves a tile and the cache policy change with the size: whole streams on both sides of each change,
    gradients from far below a step to thousands of steps."""
    import streamvbyte_amd as svb
    codec = svb.DeviceCodec(n, "cuda:0")
    g, r = gradients(torch, n, dtype, seed=n % 1000, far=3000.0)
    norm = torch.tensor([1.25], device="cuda")
    want, left = expected(oracle, variant, g, r, factor(1.25, 1.0), 64.0)
    out = torch.full(((n + 3) // 4 + 4 * n + 16,), 0xA5, dtype=torch.uint8, device="cuda")
    for _ in range(2):  # the second call finds the first one's words in the workspace
        d_r = r.cuda()
        _, size, _ = codec.quantize_feedback_encode(g.cuda(), 64.0, d_r, norm=norm, max_norm=1.0, out=out, variant=variant)
        codec.check()
        assert int(size.item()) == want.size
        assert torch.equal(out[:want.size], torch.from_numpy(want).cuda())
        assert bool((out[want.size:] == 0xA5).all())
        assert same_bits(d_r, torch.from_numpy(left))


@pytest.mark.parametrize("variant", [V0124, V1234])
def test_feedback_of_incompressible_gradients(torch, codec, oracle, variant):
    """Every width of integer up to four bytes in every group, beyond 2^22 too: the worst case of a tile's bytes."""
    n = 150001
    rng = np.random.default_rng(5)
    x = (rng.standard_normal(n) * 2.0 ** rng.integers(0, 31, n)).astype(np.float32)
    g, r = torch.from_numpy(x), torch.zeros(n)
    want, left = expected(oracle, variant, g, r, np.float32(1.0), 1.0)
    out, size, new = codec.quantize_feedback_encode(g.cuda(), 1.0, r.cuda(), variant=variant)
    assert int(size.item()) == want.size and np.array_equal(out[:want.size].cpu().numpy(), want)
    assert same_bits(new, torch.from_numpy(left))
    big = torch.full((n,), -1.5e9)  # four bytes each
    want, left = expected(oracle, variant, big, r, np.float32(1.0), 1.0)
    out, size, new = codec.quantize_feedback_encode(big.cuda(), 1.0, r.cuda(), variant=variant)
    assert int(size.item()) == want.size == (n + 3) // 4 + 4 * n and np.array_equal(out[:want.size].cpu().numpy(), want)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("scale", [64.0, 7.3, 1e4])
def test_feedback_against_64_bits(torch, codec, dtype, scale):
    """What is sent plus what is left is what came in, g c + r, worked out in 64 bits.  Half a float32 step, h = 2^-24 of the
    value, is lost at: the factor and the product (2 h |g c|), the sum e (h |e|), the step 1 / scale and the product
    q step (2 h |q step|) and the difference (h |r'|); the scale itself is rounded once (h |q step|, as step is its
    inverse).  And what is left is at most half a step: the product e scale is rounded before it is (h |e scale|)."""
    h = 2.0 ** -24 * (1 + 2.0 ** -10)
    for n in (5, 1027, 70001):
        g, r = gradients(torch, n, dtype, seed=n + 7, far=100.0)
        norm = torch.tensor([3.3], device="cuda")
        out, size, new = codec.quantize_feedback_encode(g.cuda(), scale, r.cuda(), norm=norm, max_norm=1.1)
        step = np.float32(1) / np.float32(scale)
        sent, _ = codec.decode_dequantize(out, n, float(step))
        gc = f64(g) * (1.1 / (f64(norm)[0] + 1e-6))
        e, qs, left = gc + f64(r), f64(sent), f64(new)
        assert (np.abs(qs + left - e) <= h * (2 * np.abs(gc) + np.abs(e) + 3 * np.abs(qs) + np.abs(left))).all()
        assert (np.abs(left) <= 0.5 / scale + h * (4 * np.abs(e) + 4 * np.abs(qs) + 4 / scale)).all()


def test_feedback_of_extremes(torch, codec, oracle):
    """Saturation at both ends of int32, infinities and NaN in gradient, residual and factor: such an element sends 0
    and keeps its residual; its neighbours do not notice."""
    big = [3e38, -3e38, 2.0 ** 31, -2.0 ** 31, 2.0 ** 31 - 128, -2.0 ** 31 - 256, 1e-45, -1e-45, 0.0, -0.0, 0.5, -0.5, 1.5, 2.5,
           INF, -INF, math.nan, 16777217.0, 33554433.0]
    for n in (len(big), 1024 + len(big), 40000):
        g = torch.zeros(n)
        g[-len(big):] = torch.tensor(big)
        g[:5] = torch.tensor(big[:5])
        for bad_r in (0.0, 0.25, 3e38, INF, math.nan):
            r = torch.full((n,), 0.125)
            r[::7] = bad_r
            for value in (None, 2.0, INF, math.nan):
                c = np.float32(1.0) if value is None else factor(value, 1.0)
                norm = None if value is None else torch.tensor([value], device="cuda")
                want, left = expected(oracle, V0124, g, r, c, 1.0)
                out, size, new = codec.quantize_feedback_encode(g.cuda(), 1.0, r.cuda(), norm=norm, max_norm=1.0)
                assert int(size.item()) == want.size and np.array_equal(out[:want.size].cpu().numpy(), want), (n, bad_r, value)
                assert same_bits(new, torch.from_numpy(left)), (n, bad_r, value)


def test_feedback_keeps_the_sign_of_zero(torch, codec, oracle):
    for dtype in TYPES:
        g = torch.tensor([-0.0, 0.0, -0.0, 0.0, -1.0, 1.0] * 200).to(TYPES[dtype])
        r = torch.tensor([-0.0, -0.0, 0.0, 0.0, -0.0, 0.0] * 200)
        for value in (None, INF):  # a factor of 1 and of 0
            c = np.float32(1.0) if value is None else factor(value, 1.0)
            want, left = expected(oracle, V1234, g, r, c, 1.0)
            norm = None if value is None else torch.tensor([value], device="cuda")
            out, size, new = codec.quantize_feedback_encode(g.cuda(), 1.0, r.cuda(), norm=norm, max_norm=1.0, variant=V1234)
            assert same_bits(new, torch.from_numpy(left)), (dtype, value)
            assert np.array_equal(out[:want.size].cpu().numpy(), want)


def test_feedback_sends_everything_in_the_end(torch, codec):
    """Gradients of a thirtieth of a step: the plain quantiser never sends one; with feedback what was sent plus what is
    left is what came in.  Each step rounds e and r' once, relative to at most a step and a half (fl(1/30) + residual), so
    T steps are off by at most 2 T half-steps of numbers below 2^-5: T * 2 * 2^-5 * 2^-24."""
    n, T, scale = 5000, 90, 64.0
    g = torch.full((n,), 1.0 / (30 * 64)).cuda()
    r, got, acc = torch.zeros(n, device="cuda"), None, torch.zeros(n, device="cuda")
    import streamvbyte_amd as svb
    reader = svb.DeviceCodec(n, "cuda:0")
    for _ in range(T):
        out, size, r = codec.quantize_feedback_encode(g, scale, r)
        reader.decode_dequantize(out, n, 1.0 / scale, out=acc, accumulate=True)
    plain, _ = codec.quantize_encode(g, scale)
    zero, _ = reader.decode_dequantize(plain, n, 1.0 / scale)
    assert bool((zero == 0).all())
    exact = T * f64(g)
    # the sum of whole steps in acc is exact; T roundings of e and of r' each
    assert (np.abs(f64(acc) + f64(r) - exact) <= T * 2 * 2.0 ** -29).all()
    assert float(acc.min()) > 0


def test_feedback_of_a_long_stream(torch, oracle):
    """Over 4 GiB of residuals, against the same steps in torch, and decoded again."""
    import streamvbyte_amd as svb
    n = (1 << 30) + 5
    codec = svb.DeviceCodec(n, "cuda:0")
    gen = torch.Generator(device="cuda").manual_seed(5)
    g = (torch.randn(n, generator=gen, device="cuda") * 0.02).to(torch.bfloat16)
    r = (torch.rand(n, generator=gen, device="cuda") - 0.5) / 64
    e = g.to(torch.float32) + r
    q = torch.round(e * 64)
    left = e - q / 64
    del e
    out, size, r = codec.quantize_feedback_encode(g, 64.0, r)
    codec.check()
    assert torch.equal(r, left)
    del left, g
    assert bool((codec.validate(out, int(size.item()), n, variant=V0124) & 1).item())
    back, used = codec.decode_dequantize(out, n, 1.0)
    assert int(used.item()) == int(size.item())
    assert torch.equal(back, q)


# ---- together, on streams, in graphs ---------------------------------------------------------------------------
def test_a_training_exchange(torch, oracle):
    """What the operators are for: every worker clips its own gradients by their norm while it encodes its bucket with
    feedback; the receiver sums the streams, clips the sum and hands it on.  Against numpy step by step."""
    import streamvbyte_amd as svb
    shapes = [(64, 33), (33,), (129, 7), (1,)]
    sizes = [int(np.prod(s)) for s in shapes]
    n, workers, scale, limit = sum(sizes), 3, 256.0, 1.0
    codecs = [svb.DeviceCodec(n, "cuda:0") for _ in range(workers)]
    residual = [torch.zeros(n, device="cuda") for _ in range(workers)]
    want_r = [np.zeros(n, dtype=np.float32) for _ in range(workers)]
    for step in range(4):
        total, want_total = torch.zeros(n, device="cuda"), np.zeros(n, dtype=np.float32)
        for w in range(workers):
            gen = torch.Generator().manual_seed(100 * step + w)
            bucket = (torch.randn(n, generator=gen) * 0.1).to(torch.bfloat16).cuda()
            grads = [v.view(s) for v, s in zip(bucket.split(sizes), shapes)]
            norm = codecs[w].grad_norm(grads)
            out, size, _ = codecs[w].quantize_feedback_encode(bucket, scale, residual[w], norm=norm, max_norm=limit)
            codecs[w].decode_dequantize(out, n, 1.0 / scale, out=total, accumulate=True)
            q, want_r[w] = feedback(bucket, want_r[w], factor(norm.item(), limit), scale)
            stream = oracle.encode(V0124, oracle.zigzag_encode(q))
            assert int(size.item()) == stream.size and np.array_equal(out[:stream.size].cpu().numpy(), stream)
            assert same_bits(residual[w], torch.from_numpy(want_r[w]))
            want_total = want_total + q.astype(np.float32) / np.float32(scale)
        assert same_bits(total, torch.from_numpy(want_total))
        norm = codecs[0].clip_grads(list(total.split(sizes)), 2.0)
        assert same_bits(total, clipped(torch.from_numpy(want_total), factor(norm.item(), 2.0)))


def test_captured_and_replayed(torch, oracle):
    """Norm, clip and encoder recorded once and replayed on new gradients in the same buffers, with eager calls of the
    same codec and synchronisations between the replays."""
    import streamvbyte_amd as svb
    n = 70001
    codec = svb.DeviceCodec(n, "cuda:0")
    grads = [torch.zeros(n, device="cuda"), torch.zeros(333, dtype=torch.bfloat16, device="cuda")]
    clip_to = [torch.empty_like(t) for t in grads]
    residual, residual_out = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    out = torch.zeros((n + 3) // 4 + 4 * n + 16, dtype=torch.uint8, device="cuda")
    norm = torch.zeros(1, device="cuda")
    a_set, b_set = svb.GradSet(grads), svb.GradSet(grads, out=clip_to)
    size = torch.zeros(1, dtype=torch.int64, device="cuda")

    def step():
        codec.grad_norm(a_set, out=norm)
        codec.clip_grads(b_set, 0.5)
        _, z, _ = codec.quantize_feedback_encode(grads[0], 64.0, residual, norm=norm, max_norm=0.5, out=out, residual_out=residual_out)
        size.copy_(z)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
    torch.cuda.current_stream().wait_stream(side)
    for k in range(4):
        g0, r0 = gradients(torch, n, "f32", seed=50 + k)
        g1 = to_type(np.linspace(-1, 1, 333).astype(np.float32) * (k + 1), torch.bfloat16)
        grads[0].copy_(g0), grads[1].copy_(g1), residual.copy_(r0)
        graph.replay()
        torch.cuda.synchronize()
        assert close_norm(norm, norm64([g0, g1], 2))
        c = factor(norm.item(), 0.5)
        assert same_bits(clip_to[0], clipped(g0, c)) and same_bits(clip_to[1], clipped(g1, c))
        want, left = expected(oracle, V0124, g0, r0, c, 64.0)
        assert int(size.item()) == want.size and np.array_equal(out[:want.size].cpu().numpy(), want)
        assert same_bits(residual_out, torch.from_numpy(left))
        # eager calls in between
        e_norm = codec.grad_norm(grads)
        assert torch.equal(e_norm, norm)
        e_out, e_size, e_new = codec.quantize_feedback_encode(grads[0], 64.0, residual, norm=norm, max_norm=0.5,
                                                              residual_out=torch.empty_like(residual))
        assert int(e_size.item()) == want.size and np.array_equal(e_out[:want.size].cpu().numpy(), want)
    codec.check()


def test_two_graphs_of_one_codec(torch, oracle):
    """Both hold the codec's workspaces; replayed in turn on one stream, in any order, each gives what it gave."""
    import streamvbyte_amd as svb
    n = 50001
    codec = svb.DeviceCodec(n, "cuda:0")
    side = torch.cuda.Stream()
    parts = []
    for i in range(2):
        g, r = gradients(torch, n - 20000 * i, "f32", seed=200 + i)
        d = dict(g=g.cuda(), r=r.cuda(), new=torch.zeros_like(r).cuda(), norm=torch.zeros(1, device="cuda"), size=torch.zeros(1, dtype=torch.int64, device="cuda"))
        d["out"] = torch.zeros(svb.streamvbyte_max_compressedbytes(g.numel()), dtype=torch.uint8, device="cuda")
        d["set"] = svb.GradSet([d["g"]])
        want, left = expected(oracle, V0124, g, r, factor(norm64([g], 2), 0.5), 64.0)
        parts.append((d, want, left, norm64([g], 2)))
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
    for order in ((0, 1), (1, 0), (1, 1, 0, 0)):
        for d, *_ in parts:
            d["out"].zero_(), d["new"].zero_(), d["norm"].zero_(), d["size"].zero_()
        for i in order:
            graphs[i].replay()
        torch.cuda.synchronize()
        for d, want, left, n64 in parts:
            assert close_norm(d["norm"], n64)
            c = factor(d["norm"].item(), 0.5)
            if c == factor(n64, 0.5):  # the float32 norm is the nearest one, so it nearly always is
                assert int(d["size"].item()) == want.size and np.array_equal(d["out"][:want.size].cpu().numpy(), want)
                assert same_bits(d["new"], torch.from_numpy(left))
        assert float(codec.grad_norm([parts[0][0]["g"]])) == float(parts[0][0]["norm"])  # and eager calls in between
    codec.check()


def test_from_several_threads(torch, oracle):
    """A codec, a stream and buffers a thread, all at once."""
    import threading
    import streamvbyte_amd as svb
    n, failures = 120007, []
    g, r = gradients(torch, n, "bf16", seed=300)
    want, left = expected(oracle, V1234, g, r, factor(2.0, 1.0), 64.0)

    def work():
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                codec = svb.DeviceCodec(n, "cuda:0")
                d_g, norm = g.cuda(), torch.tensor([2.0], device="cuda")
                for _ in range(10):
                    out, size, new = codec.quantize_feedback_encode(d_g, 64.0, r.cuda(), norm=norm, max_norm=1.0, variant=V1234)
                    ok = int(size.item()) == want.size and np.array_equal(out[:want.size].cpu().numpy(), want)
                    ok = ok and same_bits(new, torch.from_numpy(left)) and close_norm(codec.grad_norm([d_g, d_g]), norm64([g, g], 2))
                    if not ok:
                        failures.append("wrong")
        except Exception as e:  # noqa: BLE001 -- reported by the test
            failures.append(repr(e))
    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures[:3]


def test_a_graph_outlives_a_larger_eager_call(torch):
    """A later call on more tensors takes a larger workspace; the captured one's stays what it is."""
    import streamvbyte_amd as svb
    codec = svb.DeviceCodec(1, "cuda:0")
    small = make(torch, [200000, 300001], ["f32"], seed=90)
    s, norm = svb.GradSet(small), torch.zeros(1, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        codec.grad_norm(s, out=norm)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            codec.grad_norm(s, out=norm)
    torch.cuda.current_stream().wait_stream(side)
    want = norm64(small, 2)
    many = [torch.ones(3, device="cuda") for _ in range(9000)]
    assert close_norm(codec.grad_norm(many), math.sqrt(27000))
    bystanders = [torch.zeros(1 << 13, device="cuda") for _ in range(64)]  # what a freed workspace would be given to
    for _ in range(3):
        norm.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert close_norm(norm, want)
        assert close_norm(codec.grad_norm(many), math.sqrt(27000))
    assert not any(bool(b.any()) for b in bystanders)


def test_on_streams_of_their_own(torch):
    """Two codecs on two streams at once, each with its workspace."""
    import streamvbyte_amd as svb
    codecs = [svb.DeviceCodec(1 << 18, "cuda:0") for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    sets = [make(torch, [200000, 4099, 17], ["f32", "bf16"], seed=70 + i) for i in range(2)]
    keep = [[t.clone() for t in s] for s in sets]
    torch.cuda.synchronize()
    norms = []
    for _ in range(5):
        for c, st, s in zip(codecs, streams, sets):
            with torch.cuda.stream(st):
                norms.append((c.clip_grads(s, 10.0), c))
    torch.cuda.synchronize()
    for s, k in zip(sets, keep):
        first = factor(float(codecs[0].grad_norm(k)), 10.0)
        x = [clipped(t, first) for t in k]
        for _ in range(4):  # clipped again: the norm is 10 now, give or take a rounding
            x = [clipped(t, factor(float(codecs[0].grad_norm([y.cuda() for y in x])), 10.0)) for t in x]
        for got, want in zip(s, x):
            assert same_bits(got, want)
