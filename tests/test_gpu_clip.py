"""GPU parity of clip_grad_norm_ (g2v_clip_gradients) against the formula in float64.

Tolerances.  Squares are summed in 64 bits, so that the norm is the exact one's to float32's rounding, 2^-24; products are taken in 64
bits and rounded to float32, and a bfloat16 output once more to 2^-8: 2^-23 and 2^-8 plus that, of every single element, hold it
(values below float32's smallest normal number, 2^-126, apart).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BOTH = [torch.float32, torch.bfloat16]
IDS = ["f32", "bf16"]


def exact(grads, max_norm):
    n = math.sqrt(sum(float(g.detach().double().square().sum()) for g in grads))
    return n, min(1.0, max_norm / (n + 1e-6))


def near(out, g, factor):
    want = g.detach().double().cpu() * factor
    tol = 2.0 ** -23 + (2.0 ** -8 if out.dtype == torch.bfloat16 else 0.0)
    return bool(((out.detach().double().cpu() - want).abs() <= tol * want.abs() + 2.0 ** -126).all())


def make(shapes, dtypes, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * 10.0 ** (i % 4 - 2)).to(dtypes[i % len(dtypes)]).cuda() for i, s in enumerate(shapes)]


def check(grads, max_norm, out_dtypes=None):
    from CudaGaussianVoxelizer import clip_grad_norm_
    before = [g.clone() for g in grads]
    norm, factor = exact(before, max_norm)
    outs = None
    if out_dtypes is not None:
        outs = [torch.full(g.shape, float("nan"), dtype=out_dtypes[i % len(out_dtypes)], device="cuda") for i, g in enumerate(grads)]
    got = clip_grad_norm_(grads, max_norm, out=outs)
    assert got.shape == () and got.dtype == torch.float32 and got.is_cuda
    assert abs(float(got) - norm) <= 2.0 ** -23 * norm
    for g, b, o in zip(grads, before, outs or grads):
        assert near(o, b, factor)
        if outs is not None:
            assert torch.equal(g, b)
    if factor == 1.0 and outs is None:
        assert all(torch.equal(g, b) for g, b in zip(grads, before))


SHAPES = [(1,), (3,), (7, 5), (8,), (64, 64), (100, 3), (4097,), (33, 257), (), (1000, 100), (8191,), (8193,), (0, 4)]


@pytest.mark.parametrize("max_norm", [0.0, 0.5, 1e3, 1e9])
@pytest.mark.parametrize("dtypes", [[torch.float32], [torch.bfloat16], BOTH], ids=["f32", "bf16", "mixed"])
def test_in_place(dtypes, max_norm):
    check(make(SHAPES, dtypes), max_norm)


@pytest.mark.parametrize("max_norm", [0.5, 1e9])
@pytest.mark.parametrize("dtypes,outs", [([torch.float32], [torch.float32]), ([torch.bfloat16], [torch.float32]),
                                         ([torch.bfloat16], [torch.bfloat16]), (BOTH, [torch.bfloat16, torch.float32, torch.float32])])
def test_into_others(dtypes, outs, max_norm):
    check(make(SHAPES, dtypes, 1), max_norm, outs)


@pytest.mark.parametrize("count", [1, 2, 119, 120, 121, 240, 241, 700])
def test_many_tensors(count):
    """Counts around those that a launch takes, empty ones among them."""
    shapes = [((i * 37) % 300,) if i % 5 else (i % 7, 50) for i in range(count - 1)] + [(129, 7)]
    check(make(shapes, BOTH, count), 2.0)
    check(make(shapes, BOTH, count), 2.0, [torch.float32])


@pytest.mark.parametrize("n", [40_000_000, 9_000_001])
@pytest.mark.parametrize("dtype", BOTH, ids=IDS)
def test_large(n, dtype):
    """More elements than the workgroups take a chunk each at the smallest chunk."""
    from CudaGaussianVoxelizer import clip_grad_norm_
    gen = torch.Generator(device="cuda").manual_seed(n)
    grads = [torch.randn(n, generator=gen, device="cuda").to(dtype), torch.randn(513, generator=gen, device="cuda").to(dtype)]
    before = [g.clone() for g in grads]
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    got = float(clip_grad_norm_(grads, 1.0))
    assert abs(got - norm) <= 2.0 ** -23 * norm
    tol = 2.0 ** -23 + (2.0 ** -8 if dtype == torch.bfloat16 else 0.0)
    for g, b in zip(grads, before):
        want = b.double() / (norm + 1e-6)
        assert bool(((g.double() - want).abs() <= tol * want.abs() + 2.0 ** -126).all())


def test_elements_beyond_32_bits():
    """A tensor of more than 2^32 bytes and 2^31 elements: all of it counts and is scaled."""
    from CudaGaussianVoxelizer import clip_grad_norm_
    n = (1 << 31) + 77
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 12345, (1 << 31) - 1, 1 << 31, n - 1], device="cuda")
    g[at] = 3.0
    norm = clip_grad_norm_(g, 1.0)
    want = math.sqrt(45.0)
    assert abs(float(norm) - want) <= 2.0 ** -23 * want
    assert bool(((g[at].double() - 3.0 / (want + 1e-6)).abs() <= (2.0 ** -8 + 2.0 ** -23) * 3.0 / want).all())
    assert int(torch.count_nonzero(g[:1 << 30])) + int(torch.count_nonzero(g[1 << 30:])) == 5


def test_float32_range():
    """Squares that float32 does not hold, above and below: the norm is exact all the same, infinite only where float32 is."""
    for size in (1e30, 1e-30, 3e38):
        check([torch.full((1000,), size, device="cuda"), torch.full((3,), -size, device="cuda")], 1e-3 if size < 1 else 2.0) \
            if size < 3e38 else None
    from CudaGaussianVoxelizer import clip_grad_norm_
    g = torch.full((10000,), 3e38, device="cuda")
    assert math.isinf(float(clip_grad_norm_(g, 1.0)))
    assert bool(((g.double() - 0.01).abs() <= 0.01 * 2.0 ** -22).all())      # the factor is that of 64 bits


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_not_finite(bad):
    """As the formula: a NaN makes everything NaN, an infinity itself NaN and the others 0."""
    from CudaGaussianVoxelizer import clip_grad_norm_
    a, b = torch.ones(300, device="cuda"), torch.ones(50, device="cuda").bfloat16()
    a[7] = bad
    norm = float(clip_grad_norm_([a, b], 1.0))
    if math.isnan(bad):
        assert math.isnan(norm) and bool(a.isnan().all()) and bool(b.isnan().all())
    else:
        assert norm == math.inf and bool(a[7].isnan()) and int(torch.count_nonzero(a)) == 1 and int(torch.count_nonzero(b)) == 0


def test_parameters():
    """Parameters stand for their gradients, those without one are skipped; the result is torch's."""
    from CudaGaussianVoxelizer import clip_grad_norm_
    torch.manual_seed(1)
    layers = torch.nn.Sequential(torch.nn.Linear(40, 30), torch.nn.Linear(30, 20), torch.nn.Linear(7, 7)).cuda()
    layers[:2](torch.randn(9, 40, device="cuda")).square().sum().backward()
    params = list(layers.parameters())
    mine = [None if p.grad is None else p.grad.clone() for p in params]
    want = torch.nn.utils.clip_grad_norm_(params, 0.7)
    theirs = [None if p.grad is None else p.grad.clone() for p in params]
    for p, g in zip(params, mine):
        p.grad = g
    assert params[-1].grad is None
    got = clip_grad_norm_(layers.parameters(), 0.7)
    torch.testing.assert_close(got, want, rtol=1e-6, atol=0)
    for p, t in zip(params, theirs):
        assert (p.grad is None) == (t is None)
        if t is not None:
            torch.testing.assert_close(p.grad, t, rtol=2e-6, atol=0)
    out = [torch.zeros_like(p) for p in params]
    clip_grad_norm_(params, 0.1, out=out)
    assert torch.count_nonzero(out[-1]) == 0 and torch.count_nonzero(out[0]) > 0
    assert float(clip_grad_norm_([torch.nn.Parameter(torch.ones(3, device="cuda"))], 1.0)) == 0.0


@pytest.mark.parametrize("dtype", BOTH, ids=IDS)
def test_layouts(dtype):
    """Transposed, sliced, strided and unaligned tensors, in place and into outputs of other layouts; what lies between a strided
    tensor's elements stays."""
    from CudaGaussianVoxelizer import clip_grad_norm_
    base = torch.randn(50, 70, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()

    def views():
        flat = torch.zeros(base.numel() + 1, dtype=dtype, device="cuda")
        flat[1:] = base.flatten()
        wide = torch.full((50, 140), 7.0, dtype=dtype, device="cuda")
        wide[:, ::2] = base
        return [(base.clone(), None), (base.t().contiguous().t(), None), (flat[1:].view(50, 70), None), (wide[:, ::2], wide)]

    norm, factor = exact([base], 1.0)
    for v, whole in views():
        assert abs(float(clip_grad_norm_([v], 1.0)) - norm) <= 2.0 ** -23 * norm
        assert near(v, base, factor)
        if whole is not None:
            assert bool((whole[:, 1::2] == 7.0).all())
    for v, _ in views():
        for o, whole in views():
            clip_grad_norm_([v], 1.0, out=[o])
            assert torch.equal(v, base) and near(o, base, factor)
            if whole is not None:
                assert bool((whole[:, 1::2] == 7.0).all())


def test_versions_and_grad_mode():
    """Gradients that are clipped in place count as modified; a graph through a clipped tensor's old value notices."""
    from CudaGaussianVoxelizer import clip_grad_norm_
    g = torch.ones(10, device="cuda")
    x = torch.ones(10, device="cuda", requires_grad=True)
    y = (x * g).sum()
    v = g._version
    clip_grad_norm_([g], 0.5)
    assert g._version > v
    with pytest.raises(RuntimeError):
        y.backward()


def test_runs_are_equal_and_streams_are_the_callers():
    from CudaGaussianVoxelizer import clip_grad_norm_
    grads = make([(300, 400), (77,), (5000,)] * 50, BOTH, 5)
    outs = [torch.empty(g.shape, device="cuda") for g in grads]
    want = clip_grad_norm_(grads, 1.0, out=outs)
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(3)] * 2:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            o = [torch.empty(g.shape, device="cuda") for g in grads]
            got.append((clip_grad_norm_(grads, 1.0, out=o), o))
    torch.cuda.synchronize()
    for n, o in got:
        assert torch.equal(n, want) and all(torch.equal(a, b) for a, b in zip(o, outs))


@pytest.mark.parametrize("count", [20, 150])
def test_graph_replays(count):
    from CudaGaussianVoxelizer import clip_grad_norm_
    shapes = [(200, 30), (77,)] * (count // 2)
    grads, outs = make(shapes, BOTH), [torch.empty(s, device="cuda") for s in shapes]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        clip_grad_norm_(grads, 1.0, out=outs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm_(grads, 1.0, out=outs)
    for seed in range(4):
        for g, x in zip(grads, make(shapes, BOTH, 10 + seed)):
            g.copy_(x)
        graph.replay()
        got = [norm.clone()] + [o.clone() for o in outs]
        torch.cuda.synchronize()
        eager = [torch.empty(s, device="cuda") for s in shapes]
        n = clip_grad_norm_(grads, 1.0, out=eager)
        for a, b in zip(got, [n] + eager):
            assert torch.equal(a, b)


def test_refusals():
    from CudaGaussianVoxelizer import clip_grad_norm_
    a, b = torch.ones(10, device="cuda"), torch.ones(10, device="cuda")
    same = [a, a]
    overlap = [a[:6], a[4:]]
    for tensors, kw in ((same, {}), (overlap, {}), ([a, b.cpu()], {}), ([a.cpu()], {}), ([a.half()], {}), ([a, 3.0], {}),
                        ([a.to_sparse()], {}), ([a], dict(max_norm=-1.0)), ([a], dict(max_norm=float("nan"))),
                        ([a], dict(out=[b, b])), ([a], dict(out=[b[:9]])), ([a], dict(out=[b.half()])), ([a], dict(out=[b.cpu()])),
                        ([a, b], dict(out=[b, a])), ([a, b], dict(out=[torch.zeros(10, device="cuda")] * 2)),
                        ([a[:5]], dict(out=[a[2:7]]))):
        with pytest.raises(RuntimeError):
            clip_grad_norm_(tensors, **{"max_norm": 1.0, **kw})
    assert bool((a == 1).all()) and bool((b == 1).all())
    # read twice, written apart: both count
    norm = clip_grad_norm_([a, a], 1.0, out=[torch.empty(10, device="cuda"), torch.empty(10, device="cuda")])
    assert abs(float(norm) - math.sqrt(20.0)) < 1e-5
    assert float(clip_grad_norm_([], 1.0)) == 0.0
