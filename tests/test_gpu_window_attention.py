"""GPU parity of gaussian_attention with a window and sinks (g2v_window_attention_*) against a plain float64 statement of the
formula, whose gradients are the formula's, and against differences of that statement.

Tolerances (L2-relative) are those of the attention over all keys, of which this is the same sum over fewer: float32 keeps 24
bits in products and sums, and scores of up to about 20 carry 20 x 2^-24 into a probability: below 1e-5.  bfloat16 rounds an
output once (2^-9 at most) and its probabilities independently: below 4e-3; a gradient is a product with rounded score
gradients: below 8e-3.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

TOL = {torch.float32: (1e-5, 1e-5), torch.bfloat16: (4e-3, 8e-3)}
BOTH = [torch.float32, torch.bfloat16]
FAR = 1 << 40


def say(*a):
    print(*a, flush=True)


def rel(x, y):
    x, y = x.detach().double().cpu(), y.detach().double().cpu()
    n = float(y.norm())
    return float((x - y).norm()) / n if n > 0 else float(x.norm())


def visible(nq, nk, window, sinks):
    """(nq, nk) bool."""
    left, right = (FAR if w is None else w for w in window)
    p = torch.arange(nq)[:, None] + nk - nq
    j = torch.arange(nk)[None]
    return (j <= p + right) & ((j >= p - left) | (j < sinks))


def plain(q, k, v, window, sinks, mask=None, g=None, scale=None):
    """float64 (on the CPU): output and, with g, the gradients of q, k, v; keys that no query sees are left out."""
    B, nq, hq, D = q.shape
    nk, group = k.shape[1], hq // k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    out, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    for b in range(B):
        see = visible(nq, nk, window, sinks)
        if mask is not None:
            see = see & mask[b].cpu()[None]
        keys = see.any(0).nonzero()[:, 0]
        if not len(keys):
            continue
        see = see[:, keys]
        none = ~see.any(1, keepdim=True)
        for h in range(hq):
            K, V = k[b, keys, h // group], v[b, keys, h // group]
            p = torch.softmax((scale * q[b, :, h] @ K.T).masked_fill(~see & ~none, -torch.inf), -1).masked_fill(none, 0.0)
            out[b, :, h] = p @ V
            if g is not None:
                G = g[b, :, h].detach().double().cpu()
                dp = G @ V.T
                ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
                dq[b, :, h] = ds @ K
                dk[b, keys, h // group] += ds.T @ q[b, :, h]
                dv[b, keys, h // group] += p.T @ G
    return out, dq, dk, dv


def make(B, nq, nk, hq, hk, D, dtype, seed, size=1.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)   # noqa: E731
    q, k, v, go = r(B, nq, hq, D) * size, r(B, nk, hk, D) * size, r(B, nk, hk, D), r(B, nq, hq, D)
    return [t.to(dtype) for t in (q, k, v, go)]


def random_mask(B, nk, keep, seed):
    return torch.rand(B, nk, generator=torch.Generator().manual_seed(seed)) < keep


def run(q, k, v, g, window, sinks, mask=None, scale=None):
    from CudaGaussianVoxelizer import gaussian_attention
    leaves = [t.detach().cuda().requires_grad_() for t in (q, k, v)]
    mask = None if mask is None else mask.cuda()
    out = gaussian_attention(*leaves, key_mask=mask, scale=scale, window=window, sinks=sinks)
    with torch.no_grad():
        assert torch.equal(gaussian_attention(*leaves, key_mask=mask, scale=scale, window=window, sinks=sinks), out)
    out.backward(g.cuda())
    return [out.detach()] + [t.grad for t in leaves]


def check(q, k, v, g, window, sinks, mask=None, scale=None):
    dtype = q.dtype
    say(f"[window] {tuple(q.shape)} {tuple(k.shape)} {dtype} {window} {sinks}")
    got = run(q, k, v, g, window, sinks, mask, scale)
    errs = [rel(a, b) for a, b in zip(got, plain(q, k, v, window, sinks, mask, g, scale))]
    say(" ".join(f"{e:.1e}" for e in errs))
    assert got[0].dtype == dtype and got[0].is_contiguous()
    assert errs[0] < TOL[dtype][0] and max(errs[1:]) < TOL[dtype][1], errs
    if mask is not None:
        for t in got[2:]:
            assert torch.count_nonzero(t.cpu()[~mask]) == 0


IDS = ["f32", "bf16"]


@pytest.mark.parametrize("dtype", BOTH, ids=IDS)
@pytest.mark.parametrize("D", [1, 7, 24, 32, 33, 64, 72, 75, 96, 100, 128])
def test_widths(D, dtype):
    check(*make(2, 300, 300, 4, 2, D, dtype, D), (40, 25), 5)


@pytest.mark.parametrize("dtype", BOTH, ids=IDS)
@pytest.mark.parametrize("window,sinks", [((3, 0), 0), ((0, 5), 0), ((64, 64), 0), ((63, 0), 4), ((31, 32), 64), ((100, 7), 65),
                                          ((10, 10), 33), ((700, 0), 1), ((0, 700), 3), ((None, 0), 0), ((0, None), 2), ((5, 5), 130),
                                          ((None, None), 0), ((1 << 31, 20), 0), ((20, 20), 5000)])
@pytest.mark.parametrize("n", [65, 500])
def test_windows(n, window, sinks, dtype):
    check(*make(1, n, n, 2, 2, 64, dtype, n), window, sinks)


@pytest.mark.parametrize("dtype", BOTH, ids=IDS)
@pytest.mark.parametrize("nq,nk", [(1, 1), (1, 2), (2, 1), (1, 64), (1, 65), (1, 5000), (3, 4999), (33, 1000), (100, 1163),
                                   (300, 100), (300, 1), (64, 64), (257, 300), (1500, 1500)])
@pytest.mark.parametrize("window,sinks", [((100, 0), 4), ((30, 70), 0), ((500, 500), 40)])
def test_lengths(nq, nk, window, sinks, dtype):
    """Queries at the end of the keys, of one length with them, and more of them than keys (whose first stand before all keys and
    see none, or the first)."""
    check(*make(2, nq, nk, 2, 1, 32, dtype, nq * 7 + nk), window, sinks)


@pytest.mark.parametrize("dtype", BOTH, ids=IDS)
@pytest.mark.parametrize("hq,hk,nq,nk", [(8, 1, 1, 700), (6, 2, 40, 300), (12, 4, 365, 365), (5, 5, 333, 400), (7, 1, 200, 200)])
def test_shared_key_heads(hq, hk, nq, nk, dtype):
    check(*make(2, nq, nk, hq, hk, 64, dtype, hq), (50, 50), 6)


def some_masks(nk):
    """An empty scene, a single key, a valid prefix (padding), a valid suffix, shares at random, all."""
    at = torch.arange(nk)
    return torch.stack([torch.zeros(nk, dtype=torch.bool), at == nk // 2, at < nk // 3, at >= nk - nk // 4,
                        random_mask(1, nk, 0.8, 1)[0], random_mask(1, nk, 0.05, 2)[0], torch.ones(nk, dtype=torch.bool)])


@pytest.mark.parametrize("dtype", BOTH, ids=IDS)
@pytest.mark.parametrize("D", [32, 64, 75, 128])
@pytest.mark.parametrize("nq,nk", [(300, 300), (1, 2500), (90, 700)])
def test_masks(nq, nk, D, dtype):
    mask = some_masks(nk)
    q, k, v, g = make(len(mask), nq, nk, 4, 2, D, dtype, D)
    check(q, k, v, g, (60, 40), 5, mask)
    from CudaGaussianVoxelizer import gaussian_attention
    dev = [t.cuda() for t in (q, k, v)]
    got = gaussian_attention(*dev, mask.cuda(), window=(60, 40), sinks=5)
    assert torch.count_nonzero(got[0]) == 0
    assert torch.equal(got[-1], gaussian_attention(*dev, window=(60, 40), sinks=5)[-1])


@pytest.mark.parametrize("dtype", BOTH, ids=IDS)
@pytest.mark.parametrize("nq,nk", [(1, 900), (70, 400), (333, 333)])
def test_hidden_rows_are_not_read(nq, nk, dtype):
    """NaN, infinities and the type's extremes in masked rows, and in rows that no query's window reaches, change no bit."""
    mask = random_mask(2, nk, 0.6, 4)
    window, sinks = (75, 3), 7
    q, k, v, g = make(2, nq, nk, 4, 4, 40, dtype, 3)
    hidden = ~mask | ~visible(nq, nk, window, sinks).any(0)[None]
    results = []
    for bad in (0.0, float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).min, torch.finfo(dtype).max):
        kb, vb = (torch.where(hidden[:, :, None, None], torch.full_like(t, bad), t) for t in (k, v))
        results.append(run(q, kb, vb, g, window, sinks, mask))
        if nk > nq:   # the same without a mask
            unseen = ~visible(nq, nk, window, sinks).any(0)[None, :, None, None]
            kb, vb = (torch.where(unseen, torch.full_like(t, bad), t) for t in (k, v))
            results[-1] += run(q, kb, vb, g, window, sinks)
    for r in results[1:]:
        for a, b in zip(r, results[0]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", BOTH, ids=IDS)
@pytest.mark.parametrize("D", [64, 128])
def test_wide_windows_are_the_attention_over_all_keys(D, dtype):
    """The same sums in another order: both are within the tolerance of 64 bits."""
    from CudaGaussianVoxelizer import gaussian_attention
    q, k, v, g = make(2, 400, 700, 4, 2, D, dtype, 5)
    mask = random_mask(2, 700, 0.7, 6)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    out = gaussian_attention(*leaves, mask.cuda())
    out.backward(g.cuda())
    for window in ((700, 700), (None, None)):
        got = run(q, k, v, g, window, 0, mask)
        for a, b, tol in zip(got, [out] + [t.grad for t in leaves], (TOL[dtype][0],) + (TOL[dtype][1],) * 3):
            assert rel(a, b) < 2 * tol


@pytest.mark.parametrize("dtype", BOTH, ids=IDS)
@pytest.mark.parametrize("slope", [0.5, -0.5, 8.0])
@pytest.mark.parametrize("window,sinks", [((150, 0), 0), ((0, 150), 3), ((90, 90), 2)])
def test_references_far_from_the_maximum(window, sinks, slope, dtype):
    """Scores that climb or fall over the whole row, so that what a row sees first is far from its maximum.  Values are whole numbers
    that bfloat16 holds and the softmax is all but a choice, so that outputs are exact to their rounding."""
    n, d = 700, 64
    q, k = torch.zeros(1, n, 1, d), torch.zeros(1, n, 1, d)
    q[..., 0], q[..., 1] = slope, slope
    k[..., 0] = (torch.arange(n) // 64 * 64)[None, :, None]
    k[..., 1] = (torch.arange(n) % 64)[None, :, None]
    gen = torch.Generator().manual_seed(1)
    v, g = torch.randn(1, n, 1, d, generator=gen), torch.randn(1, n, 1, d, generator=gen)
    q, k, v, g = (t.to(dtype) for t in (q, k, v, g))
    got = run(q, k, v, g, window, sinks, scale=1.0)
    want = plain(q, k, v, window, sinks, None, g, 1.0)
    # float32: a score of 5600 carries 5600 x 2^-24 x log2(e) into the exponent, 4.8e-4 of a probability
    tol = 1e-3 if dtype == torch.float32 else 5e-3
    assert rel(got[0], want[0]) < tol and rel(got[3], want[3]) < 2 * tol
    assert all(torch.isfinite(t).all() for t in got)


@pytest.mark.parametrize("dtype", BOTH, ids=IDS)
def test_alone_in_the_window(dtype):
    """A query whose only key is its own has that key's value, and no gradient of q and k, exactly.  Its probability is 2^(c s - m),
    with the product c s rounded in m but not before the difference: at scores of 40 in base 2 off by 40 x 2^-24 x ln 2, 1.7e-6, and
    so are the output and dV beside their own rounding: the tolerances of both types hold that."""
    q, k, v, g = make(2, 300, 300, 4, 4, 64, dtype, 8)
    out, dq, dk, dv = run(q, k, v, g, (0, 0), 0)
    assert rel(out, v) < TOL[dtype][0] and rel(dv, g) < TOL[dtype][1]
    assert torch.count_nonzero(dq) == 0 and torch.count_nonzero(dk) == 0


@pytest.mark.parametrize("scale", [0.01, 1.0])
@pytest.mark.parametrize("dtype", BOTH, ids=IDS)
def test_scale(scale, dtype):
    check(*make(1, 200, 200, 2, 2, 32, dtype, 9), (33, 12), 2, scale=scale)


def test_gradient_against_differences():
    """Central differences of the float64 statement along random directions (step 1e-5: error 1e-10 relative)."""
    window, sinks = (9, 4), 3
    q, k, v, g = make(1, 60, 80, 4, 2, 16, torch.float32, 21)
    mask = random_mask(1, 80, 0.8, 22)
    _, *grads = run(q, k, v, g, window, sinks, mask)
    base = [t.double() for t in (q, k, v)]
    gen = torch.Generator().manual_seed(4)
    for i, got in enumerate(grads):
        u = torch.randn(base[i].shape, generator=gen, dtype=torch.float64)
        step = [float((plain(*[t + s * 1e-5 * u if n == i else t for n, t in enumerate(base)], window, sinks, mask)[0] * g.double()).sum())
                for s in (1, -1)]
        want, have = (step[0] - step[1]) / 2e-5, float((got.double().cpu() * u).sum())
        assert abs(have - want) <= 1e-5 * float((got.double().cpu().abs() * u.abs()).sum())


@pytest.mark.parametrize("dtype", BOTH, ids=IDS)
@pytest.mark.parametrize("D", [64, 36])
def test_layouts(D, dtype):
    """Views of a fused projection, heads-first storage, rows off 16-byte boundaries and a transposed row give the contiguous
    tensors' results bit for bit; gradients that arrive expanded or transposed do too."""
    B, n, h, window, sinks = 2, 200, 4, (50, 20), 3
    q, k, v, g = (t.cuda() for t in make(B, n, n, h, h, D, dtype, 7))
    mask = random_mask(B, n, 0.8, 3)
    want = run(q, k, v, g, window, sinks, mask)

    def views(t):
        fused = torch.randn(B, n, 3 * h, D, device="cuda").to(dtype)
        fused[:, :, h:2 * h] = t
        yield fused[:, :, h:2 * h]
        yield t.transpose(1, 2).contiguous().transpose(1, 2)
        flat = torch.zeros(t.numel() + 1, dtype=dtype, device="cuda")
        flat[1:] = t.flatten()
        yield flat[1:].view(t.shape)
        yield t.transpose(2, 3).contiguous().transpose(2, 3)

    for qv, kv, vv, gv in zip(views(q), views(k), views(v), views(g)):
        for a, b in zip(run(qv, kv, vv, gv, window, sinks, mask), want):
            assert torch.equal(a, b)
    ones = run(q, k, v, torch.ones_like(g), window, sinks, mask)
    for a, b in zip(run(q, k, v, torch.ones((), dtype=dtype, device="cuda").expand(g.shape), window, sinks, mask), ones):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", BOTH, ids=IDS)
@pytest.mark.parametrize("masked", [False, True])
def test_offsets_beyond_32_bits(masked, dtype):
    """A long cache whose rows lie far apart: keys behind 4 GiB, reached from the sinks over the gap."""
    nk, stride, D = 70000, 40000, 64
    base = torch.zeros((nk - 1) * stride + 2 * D, dtype=dtype, device="cuda")
    assert base.numel() * 2 > 1 << 32
    k = torch.as_strided(base, (1, nk, 1, D), (base.numel(), stride, D, 1))
    v = torch.as_strided(base, (1, nk, 1, D), (base.numel(), stride, D, 1), D)
    q, kc, vc, _ = (t.cuda() for t in make(1, 3, nk, 1, 1, D, dtype, 2))
    k.copy_(kc)
    v.copy_(vc)
    mask = random_mask(1, nk, 0.7, 5).cuda() if masked else None
    from CudaGaussianVoxelizer import gaussian_attention
    got = gaussian_attention(q, k, v, mask, window=(200, 0), sinks=5)
    assert torch.equal(got, gaussian_attention(q, kc, vc, mask, window=(200, 0), sinks=5))
    keys = torch.cat([torch.arange(0, 5), torch.arange(nk - 400, nk)])
    small = [t[:, keys].contiguous() for t in (kc, vc)]
    assert rel(got, plain(q, *small, (200, 0), 5, None if mask is None else mask[:, keys.cuda()])[0]) < TOL[dtype][0]


@pytest.mark.parametrize("dtype", BOTH, ids=IDS)
@pytest.mark.parametrize("nq,nk,masked", [(1, 3000, False), (1, 3000, True), (300, 300, True), (700, 900, False)])
def test_graph_replays(nq, nk, masked, dtype):
    """A captured step, replayed over new inputs with eager work between, gives the eager results bit for bit."""
    from CudaGaussianVoxelizer import _C
    window, sinks = (80, 30), 4
    q, k, v, g = (t.cuda() for t in make(2, nq, nk, 4, 2, 64, dtype, 11))
    mask = random_mask(2, nk, 0.7, 12).cuda() if masked else None

    def step():
        out, rest, lse = _C.window_attention_forward(q, k, v, window, sinks, mask, for_backward=True)
        return (out,) + _C.window_attention_backward(g, q, k, v, out, rest, lse, window, sinks, mask)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(4):
        for t, x in zip((q, k, v, g), make(2, nq, nk, 4, 2, 64, dtype, 100 + seed)):
            t.copy_(x)
        if masked:
            mask.copy_(random_mask(2, nk, 0.3 + 0.2 * seed, seed))
        graph.replay()
        got = [t.clone() for t in held]
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", BOTH, ids=IDS)
@pytest.mark.parametrize("nq,nk", [(1, 9000), (2100, 2100)])
def test_runs_are_equal_and_streams_are_the_callers(nq, nk, dtype):
    q, k, v, g = (t.cuda() for t in make(2, nq, nk, 4, 2, 64, dtype, 13))
    mask = random_mask(2, nk, 0.9, 1)
    want = run(q, k, v, g, (900, 100), 8, mask)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams * 2:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(run(q, k, v, g, (900, 100), 8, mask))
    torch.cuda.synchronize()
    for r in got:
        for a, b in zip(r, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", BOTH, ids=IDS)
def test_empty(dtype):
    from CudaGaussianVoxelizer import gaussian_attention
    for B, nq, nk in ((0, 5, 5), (2, 0, 5), (2, 5, 0), (2, 0, 0), (2, 0, 300), (1, 0, 1)):
        leaves = [torch.randn(B, n, 2, 32, device="cuda", dtype=dtype, requires_grad=True) for n in (nq, nk, nk)]
        for window, sinks in (((3, 3), 1), ((0, 0), 0), ((None, 0), 0)):
            out = gaussian_attention(*leaves, torch.ones(B, nk, dtype=torch.bool, device="cuda"), window=window, sinks=sinks)
            assert out.shape == (B, nq, 2, 32) and torch.count_nonzero(out) == 0
            for g in torch.autograd.grad(out.sum(), leaves):
                assert torch.count_nonzero(g) == 0


def test_partial_gradients():
    from CudaGaussianVoxelizer import gaussian_attention
    q, k, v, g = (t.cuda() for t in make(1, 150, 150, 2, 2, 64, torch.bfloat16, 17))
    want = run(q, k, v, g, (20, 20), 3)
    for wanted in ((0,), (1,), (2,), (0, 2), (1, 2)):
        leaves = [t.detach().requires_grad_(i in wanted) for i, t in enumerate((q, k, v))]
        gaussian_attention(*leaves, window=(20, 20), sinks=3).backward(g)
        for i, t in enumerate(leaves):
            assert (t.grad is None) == (i not in wanted)
            assert t.grad is None or torch.equal(t.grad, want[1 + i])


@pytest.mark.parametrize("n,hq,hk,D,dtype,window,sinks,keep", [
    (9000, 8, 8, 64, torch.bfloat16, (256, 256), 16, 1.0), (9000, 8, 8, 64, torch.bfloat16, (1500, 0), 70, 0.8),
    (6000, 4, 2, 128, torch.bfloat16, (300, 300), 4, 1.0), (5000, 4, 4, 96, torch.bfloat16, (300, 300), 4, 1.0),
    (5000, 4, 4, 64, torch.float32, (128, 128), 4, 0.9), (4000, 2, 2, 128, torch.float32, (400, 0), 33, 1.0)])
def test_rounds_of_workgroups(n, hq, hk, D, dtype, window, sinks, keep):
    """Enough tiles for several rounds of the card's workgroups, sinks' queries in many splits."""
    mask = None if keep == 1.0 else random_mask(1, n, keep, n)
    check(*make(1, n, n, hq, hk, D, dtype, n), window, sinks, mask)


def test_backward_without_the_rounding_lost():
    from CudaGaussianVoxelizer import _C
    q, k, v, g = make(1, 300, 300, 4, 2, 64, torch.bfloat16, 23)
    dev = [t.cuda() for t in (q, k, v)]
    out, rest, lse = _C.window_attention_forward(*dev, (40, 40), 2, for_backward=True)
    assert rest is not None
    got = _C.window_attention_backward(g.cuda(), *dev, out, None, lse, (40, 40), 2)
    for x, y in zip(got, plain(q, k, v, (40, 40), 2, None, g)[1:]):
        assert rel(x, y) < TOL[torch.bfloat16][1]


def test_refusals():
    from CudaGaussianVoxelizer import PyGaussianAttention, gaussian_attention
    q, k, v, g = (t.cuda() for t in make(1, 20, 20, 2, 2, 32, torch.float32, 1))
    for kw in (dict(window=5), dict(window=(1, 2, 3)), dict(window=(-1, 2)), dict(window=(1.5, 2)), dict(window=(True, 2)),
               dict(window=(3, 3), sinks=-1), dict(window=(3, 3), sinks=1.0), dict(sinks=2), dict(window="ab"),
               dict(window=(3, 3), key_mask=torch.ones(1, 20, device="cuda")), dict(window=(3, 3), scale=0.0)):
        with pytest.raises(RuntimeError):
            gaussian_attention(q, k, v, **kw)
    for kw in (dict(window=3), dict(sinks=1), dict(window=(2, -3))):
        with pytest.raises(RuntimeError):
            PyGaussianAttention(64, 2, **kw)
    with pytest.raises(RuntimeError):
        gaussian_attention(q, k.bfloat16(), v, window=(3, 3))
    with pytest.raises(RuntimeError):
        gaussian_attention(q.cpu(), k.cpu(), v.cpu(), window=(3, 3))
    leaf = q.requires_grad_()
    grad, = torch.autograd.grad(gaussian_attention(leaf, k, v, window=(3, 3)).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        gaussian_attention(fwAD.make_dual(q.detach(), g), k, v, window=(3, 3))
