"""GPU parity of layer_norm (g2v_layer_norm_*) against a plain float64 statement of the formula, whose gradients come from
autograd, and against differences of that statement.

Tolerances (L2-relative).  float32: means and sums of at most 8192 terms, added in a tree of lanes below a chain of at most 32
(34 x 2^-24), a root and a few products: below 1e-5.  A bfloat16 result is rounded once, to 2^-8 at most: below 4e-3.  Weight
gradients are float32 sums over rows of float32 terms (chains of at most a workgroup's rows, then a tree) in both: 1e-5 of the terms'
magnitudes.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 1e-5, torch.bfloat16: 4e-3}
BOTH = [torch.float32, torch.bfloat16]
IDS = ["f32", "bf16"]


def say(*a):
    print(*a, flush=True)


def rel(x, y):
    x, y = x.detach().double().cpu(), y.detach().double().cpu()
    n = float(y.norm())
    return float((x - y).norm()) / n if n > 0 else float(x.norm())


def plain(x, w, b, eps):
    """float64, of the sum where there is a residual."""
    d = x - x.mean(-1, keepdim=True)
    y = d / (d.square().mean(-1, keepdim=True) + eps).sqrt()
    y = y if w is None else y * w
    return y if b is None else y + b


def make(shape, dtype, seed, wdtype=torch.float32, offset=0.3):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)   # noqa: E731
    C = shape[-1]
    return {"x": (r(*shape) + offset).to(dtype), "residual": (2 * r(*shape) + offset).to(dtype), "w": (1 + 0.2 * r(C)).to(wdtype),
            "b": (0.1 * r(C)).to(wdtype), "gy": r(*shape).to(dtype), "gs": r(*shape).to(dtype)}


def run(d, residual, eps=1e-5, weight=True, bias=True):
    """(y, sum or None, grads of x, w, b, residual) on the GPU."""
    from CudaGaussianVoxelizer import layer_norm
    x, w, b, res = (d[n].detach().cuda().requires_grad_() for n in ("x", "w", "b", "residual"))
    w, b, res = w if weight else None, b if bias else None, res if residual else None
    got = layer_norm(x, w, b, residual=res, eps=eps)
    with torch.no_grad():
        again = layer_norm(x, w, b, residual=res, eps=eps)
    if residual:
        assert all(torch.equal(p, q) for p, q in zip(got, again))
        torch.autograd.backward(got, [d["gy"].cuda(), d["gs"].cuda()])
        y, total = got
    else:
        assert torch.equal(got, again)
        got.backward(d["gy"].cuda())
        y, total = got, None
    return y.detach(), total, [None if t is None else t.grad for t in (x, w, b, res)]


def check(d, residual, eps=1e-5, weight=True, bias=True):
    dtype = d["x"].dtype
    y, total, grads = run(d, residual, eps, weight, bias)
    s = d["x"]
    if residual:
        s = (d["x"].float() + d["residual"].float()).to(dtype)
        assert torch.equal(total.detach().cpu(), s) and total.is_contiguous()
    s = s.double().requires_grad_()
    w, b = (d[n].double().requires_grad_() for n in ("w", "b"))
    want = plain(s, w if weight else None, b if bias else None, eps)
    want.backward(d["gy"].double())
    dx = s.grad + (d["gs"].double() if residual else 0.0)
    errs = [rel(y, want), rel(grads[0], dx)]
    say(" ".join(f"{e:.1e}" for e in errs))
    assert y.dtype == dtype and y.is_contiguous() and max(errs) < TOL[dtype], errs
    if residual:
        assert torch.equal(grads[3], grads[0])
    dims = tuple(range(s.dim() - 1))
    xh = plain(s.detach(), None, None, eps)
    for g, t, terms, on in ((grads[1], w, d["gy"].double() * xh, weight), (grads[2], b, d["gy"].double(), bias)):
        if not on:
            assert g is None
            continue
        size = terms.abs().sum(dims)
        bound = (1e-5 if g.dtype == torch.float32 else 4e-3) * size + 1e-30
        assert g.dtype == d["w"].dtype and ((g.double().cpu() - t.grad).abs() <= bound).all()


@pytest.mark.parametrize("dtype", BOTH, ids=IDS)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("C", [1, 2, 3, 4, 7, 8, 17, 32, 64, 75, 100, 128, 255, 256, 257, 511, 512, 513, 771, 1000, 1024, 1025, 1030, 2048,
                               2050, 4096, 4099, 8192])
def test_widths(C, residual, dtype):
    check(make((2, 37, C), dtype, C), residual)


@pytest.mark.parametrize("dtype", BOTH, ids=IDS)
@pytest.mark.parametrize("shape", [(1, 64), (1, 1, 1024), (64,), (3, 64), (2, 3, 5, 40), (70000, 32), (9001, 256), (5000, 1024), (1500, 4096)])
def test_rows(shape, dtype):
    """From one row (and none but it) to more than the workgroups take in one go."""
    check(make(shape, dtype, shape[0]), True)


@pytest.mark.parametrize("dtype", BOTH, ids=IDS)
@pytest.mark.parametrize("wdtype", BOTH, ids=["wf32", "wbf16"])
@pytest.mark.parametrize("weight,bias", [(True, True), (True, False), (False, True), (False, False)])
def test_weights(weight, bias, wdtype, dtype):
    """Weights of either type with rows of either type, and without one or both."""
    check(make((3, 50, 96), dtype, 7, wdtype), False, weight=weight, bias=bias)


@pytest.mark.parametrize("offset", [1e3, 1e5])
@pytest.mark.parametrize("C", [64, 1000, 4096])
def test_far_from_zero(C, offset):
    """Rows whose mean is far larger than their spread.  The mean is a float32: off by a few 2^-24 of the offset, 0.02 at 1e5 (float32's
    inputs themselves are 0.004 apart there), and so is every difference to it; the variance is that of the differences."""
    d = make((40, C), torch.float32, C, offset=offset)
    y, _, _ = run(d, False)
    assert float((y.double().cpu() - plain(d["x"].double(), d["w"].double(), d["b"].double(), 1e-5)).abs().max()) < 8 * 2.0 ** -24 * offset * 2 + 1e-5


@pytest.mark.parametrize("dtype", BOTH, ids=IDS)
def test_constant_rows_and_extremes(dtype):
    """A constant row gives the bias (its differences are 0), an infinity or NaN its own row's alone."""
    from CudaGaussianVoxelizer import layer_norm
    x = torch.randn(6, 128, generator=torch.Generator().manual_seed(1)).to(dtype)
    x[1] = 2.0
    x[2, 5] = float("inf")
    x[3, 7] = float("nan")
    w, b = torch.full((128,), 1.5), torch.linspace(-1, 1, 128)
    got = layer_norm(x.cuda(), w.cuda(), b.cuda()).cpu()
    assert torch.equal(got[1], b.to(dtype))
    assert torch.isnan(got[2]).all() and torch.isnan(got[3]).all()
    ok = [0, 4, 5]
    assert rel(got[ok], plain(x[ok].double(), w.double(), b.double(), 1e-5)) < TOL[dtype]


def test_eps():
    d = make((30, 64), torch.float32, 3)
    d["x"] = d["x"] * 1e-3
    for eps in (0.0, 1e-12, 1e-6, 0.1):
        check(d, False, eps)


def test_gradient_against_differences():
    """Central differences of the float64 statement along random directions (step 1e-5: error 1e-10 relative)."""
    d = make((2, 9, 20), torch.float32, 3)
    d["residual"] = torch.zeros_like(d["x"])
    _, _, (gx, gw, gb, _) = run(d, True, 1e-3)

    def value(m):
        return float((plain(m["x"], m["w"], m["b"], 1e-3) * d["gy"].double()).sum() + (m["x"] * d["gs"].double()).sum())

    base = {n: d[n].double() for n in ("x", "w", "b")}
    gen = torch.Generator().manual_seed(4)
    for n, g in (("x", gx), ("w", gw), ("b", gb)):
        u = torch.randn(base[n].shape, generator=gen, dtype=torch.float64)
        step = [value(dict(base, **{n: base[n] + s * 1e-5 * u})) for s in (1, -1)]
        want, got = (step[0] - step[1]) / 2e-5, float((g.double().cpu() * u).sum())
        assert abs(got - want) <= 1e-5 * float((g.double().cpu().abs() * u.abs()).sum()), n


@pytest.mark.parametrize("dtype", BOTH, ids=IDS)
@pytest.mark.parametrize("C", [64, 36, 1026])
def test_layouts(C, dtype):
    """Slices of a wider tensor, transposed leading dimensions, rows off 16-byte boundaries, a transposed row and expanded rows, alone
    and mixed, give the contiguous tensors' results bit for bit."""
    B, n = 3, 20
    d = make((B, n, C), dtype, 5)
    want = run(d, True)

    def views(t):
        wide = torch.randn(B, n, 3 * C, device="cuda").to(dtype)
        wide[..., C:2 * C] = t
        yield wide[..., C:2 * C]
        yield t.cuda().transpose(0, 1).contiguous().transpose(0, 1)
        flat = torch.zeros(t.numel() + 1, dtype=dtype, device="cuda")
        flat[1:] = t.cuda().flatten()
        yield flat[1:].view(t.shape)
        yield t.cuda().transpose(1, 2).contiguous().transpose(1, 2)
        yield t.cuda()

    names = ("x", "residual", "gy", "gs")
    all_views = {k: list(views(d[k])) for k in names}
    for i in range(5):
        for shift in (0, 1):
            v = {k: all_views[k][(i + shift * j) % 5] for j, k in enumerate(names)}
            got = run(dict(d, **v), True)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
            for a, b in zip(got[2], want[2]):
                assert torch.equal(a, b)
    from CudaGaussianVoxelizer import layer_norm
    row = d["x"][:1].cuda()
    assert torch.equal(layer_norm(row.expand(B, n, C)), layer_norm(row.expand(B, n, C).contiguous()))
    x = d["x"].cuda().requires_grad_()
    layer_norm(x).sum().backward()      # an expanded gradient
    want = x.grad
    x.grad = None
    layer_norm(x).backward(torch.ones_like(x))
    assert torch.equal(x.grad, want)


def test_partial_gradients():
    from CudaGaussianVoxelizer import layer_norm
    d = make((4, 30, 48), torch.float32, 9)
    want = run(d, True)[2]
    names = ("x", "w", "b", "residual")
    for on in ((0,), (1,), (2,), (3,), (0, 2), (1, 3)):
        t = [d[n].cuda().requires_grad_(i in on) for i, n in enumerate(names)]
        got = layer_norm(t[0], t[1], t[2], residual=t[3])
        live = [o for o in got if o.requires_grad]
        torch.autograd.backward(got, [d["gy"].cuda(), d["gs"].cuda()]) if len(live) == 2 else got[0].backward(d["gy"].cuda())
        for i in range(4):
            assert (t[i].grad is None) == (i not in on)
            assert t[i].grad is None or torch.equal(t[i].grad, want[i])
    # the norm's output alone, the sum's alone
    t = [d[n].cuda().requires_grad_() for n in names]
    layer_norm(t[0], t[1], t[2], residual=t[3])[0].backward(d["gy"].cuda())
    alone = layer_norm((d["x"] + d["residual"]).cuda().requires_grad_(), t[1].detach(), t[2].detach())
    assert alone.shape == t[0].shape and torch.equal(t[0].grad, t[3].grad) and torch.equal(t[1].grad, want[1])
    t = [d[n].cuda().requires_grad_() for n in names]
    layer_norm(t[0], t[1], t[2], residual=t[3])[1].backward(d["gs"].cuda())
    assert torch.equal(t[0].grad.cpu(), d["gs"]) and torch.equal(t[3].grad.cpu(), d["gs"]) and t[1].grad is None


@pytest.mark.parametrize("dtype", BOTH, ids=IDS)
@pytest.mark.parametrize("shape", [(300, 256), (700, 1024), (50, 4100)])
def test_graph_replays(shape, dtype):
    from CudaGaussianVoxelizer import _C
    d = {k: t.cuda() for k, t in make(shape, dtype, 1).items()}

    def step():
        y, s, st = _C.layer_norm_forward(d["x"], d["w"], d["b"], d["residual"], 1e-5, True)
        return (y, s) + _C.layer_norm_backward(d["gy"], s, d["w"], st, d["gs"])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(4):
        for k, t in make(shape, dtype, 50 + seed).items():
            d[k].copy_(t)
        graph.replay()
        got = [t.clone() for t in held]
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_runs_are_equal_and_streams_are_the_callers():
    d = make((9000, 512), torch.bfloat16, 2)
    want = run(d, True)
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(3)] * 2:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(run(d, True))
    torch.cuda.synchronize()
    for y, total, grads in got:
        assert torch.equal(y, want[0]) and torch.equal(total, want[1])
        assert all(torch.equal(a, b) for a, b in zip(grads, want[2]))


@pytest.mark.parametrize("dtype", BOTH, ids=IDS)
def test_empty(dtype):
    from CudaGaussianVoxelizer import layer_norm
    for shape in ((0, 64), (2, 0, 64), (0, 5, 64)):
        x, r = (torch.zeros(shape, device="cuda", dtype=dtype, requires_grad=True) for _ in range(2))
        w, b = (torch.ones(64, device="cuda", requires_grad=True) for _ in range(2))
        y, s = layer_norm(x, w, b, residual=r)
        assert y.shape == shape and s.shape == shape
        y.sum().backward()
        assert torch.count_nonzero(w.grad) == 0 and torch.count_nonzero(b.grad) == 0 and x.grad.shape == shape


def test_offsets_beyond_32_bits():
    """Rows behind 4 GiB, far apart."""
    from CudaGaussianVoxelizer import layer_norm
    n, stride, C = 70000, 40000, 64
    base = torch.zeros((n - 1) * stride + C, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(base, (n, C), (stride, 1))
    v = torch.randn(n, C, device="cuda").bfloat16()
    x.copy_(v)
    assert torch.equal(layer_norm(x), layer_norm(v))


def test_module():
    """PyLayerNorm has torch.nn.LayerNorm's parameters: a state of one loads into the other, and they agree."""
    from CudaGaussianVoxelizer import PyLayerNorm
    torch.manual_seed(0)
    ref = torch.nn.LayerNorm(96, device="cuda")
    with torch.no_grad():
        ref.weight.add_(0.1 * torch.randn(96, device="cuda"))
        ref.bias.add_(0.1 * torch.randn(96, device="cuda"))
    own = PyLayerNorm(96)
    own.load_state_dict(ref.state_dict())
    x, r = torch.randn(5, 40, 96, device="cuda"), torch.randn(5, 40, 96, device="cuda")
    assert rel(own(x), ref(x)) < 2 * TOL[torch.float32]
    y, s = own(x, residual=r)
    assert torch.equal(s, x + r) and rel(y, ref(x + r)) < 2 * TOL[torch.float32]
    own = own.bfloat16()
    y = own(x.bfloat16())
    y.float().square().sum().backward()
    assert y.dtype == torch.bfloat16 and own.weight.grad.dtype == torch.bfloat16
    assert PyLayerNorm(96, bias=False).bias is None


def test_refusals():
    from CudaGaussianVoxelizer import layer_norm
    x, w = torch.randn(4, 32, device="cuda"), torch.ones(32, device="cuda")
    for args, kw in (((x.cpu(),), {}), ((x.half(),), {}), ((x.double(),), {}), ((x[0, 0],), {}), (([1.0],), {}),
                     ((x, w[:31]), {}), ((x, w.half()), {}), ((x, w.cpu()), {}), ((x, w, w.bfloat16()), {}), ((x, None, w[:5]), {}),
                     ((x,), dict(residual=x[:3])), ((x,), dict(residual=x.bfloat16())), ((x,), dict(residual=x.cpu())),
                     ((x,), dict(eps=-1.0)), ((x,), dict(eps=float("nan"))), ((torch.zeros(2, 8193, device="cuda"),), {}),
                     ((torch.zeros(2, 0, device="cuda"),), {})):
        with pytest.raises(RuntimeError):
            layer_norm(*args, **kw)
    leaf = x.requires_grad_()
    g, = torch.autograd.grad(layer_norm(leaf).square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        layer_norm(fwAD.make_dual(x.detach(), torch.ones_like(x)))
