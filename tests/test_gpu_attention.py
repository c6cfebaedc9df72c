"""GPU parity of gaussian_attention (g2v_attention_*) against a plain float64 statement of the formula, whose gradients are
the formula's, and against differences of that statement.

Tolerances (L2-relative).  float32: products keep 24 bits and sum in float32, scores of up to about 20 carry 20 x 2^-24 into
the exponent and so into each probability: a few 1e-6, below 1e-5.  bfloat16: an output is rounded once (2^-9 at most, 2^-10.8
in the mean square), its probabilities too, independently; together below 4e-3.  A gradient is a product with rounded
score gradients, whose delta takes the rounded output: below 8e-3.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

TOL = {torch.float32: (1e-5, 1e-5), torch.bfloat16: (4e-3, 8e-3)}


def say(*a):
    print(*a, flush=True)


def rel(x, y):
    x, y = x.detach().double().cpu(), y.detach().double().cpu()
    n = float(y.norm())
    return float((x - y).norm()) / n if n > 0 else float(x.norm())


def plain(q, k, v, mask, g=None, scale=None):
    """float64 (on the CPU): output and, with g, the gradients of q, k, v.  Masked keys are left out, not weighted with 0."""
    B, nq, hq, D = q.shape
    group = hq // k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    out, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    for b in range(B):
        keys = torch.arange(k.shape[1]) if mask is None else mask[b].cpu().nonzero()[:, 0]
        if not len(keys):
            continue
        for h in range(hq):
            K, V = k[b, keys, h // group], v[b, keys, h // group]
            p = torch.softmax(scale * q[b, :, h] @ K.T, -1)
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


def check(q, k, v, g, mask, dtype, scale=None):
    from CudaGaussianVoxelizer import gaussian_attention
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    cm = None if mask is None else mask.cuda()
    out = gaussian_attention(*leaves, key_mask=cm, scale=scale)
    with torch.no_grad():
        assert torch.equal(gaussian_attention(*leaves, key_mask=cm, scale=scale), out)
    out.backward(g.cuda())
    want = plain(q, k, v, mask, g, scale)
    errs = [rel(a, b) for a, b in zip([out] + [t.grad for t in leaves], want)]
    say(" ".join(f"{e:.1e}" for e in errs))
    assert out.dtype == dtype and out.is_contiguous()
    assert errs[0] < TOL[dtype][0] and max(errs[1:]) < TOL[dtype][1], errs
    if mask is not None:
        off = ~mask
        for t in leaves[1:]:
            assert torch.count_nonzero(t.grad.cpu()[off]) == 0


BOTH = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("dtype", BOTH, ids=["f32", "bf16"])
@pytest.mark.parametrize("D", [1, 7, 8, 24, 32, 33, 64, 72, 75, 96, 100, 128])
def test_widths(D, dtype):
    check(*make(2, 70, 150, 4, 2, D, dtype, D), None, dtype)


@pytest.mark.parametrize("dtype", BOTH, ids=["f32", "bf16"])
@pytest.mark.parametrize("nq,nk", [(1, 1), (1, 2), (2, 1), (31, 33), (32, 32), (33, 31), (64, 64), (63, 65), (65, 127),
                                   (128, 129), (257, 300), (300, 257), (1, 5000), (3, 4999), (5000, 1), (700, 1500)])
def test_lengths(nq, nk, dtype):
    check(*make(1, nq, nk, 2, 2, 64, dtype, nq * 7 + nk), None, dtype)


@pytest.mark.parametrize("dtype", BOTH, ids=["f32", "bf16"])
@pytest.mark.parametrize("hq,hk,nq", [(8, 1, 1), (6, 2, 40), (12, 4, 65), (5, 5, 33), (7, 1, 100)])
def test_shared_key_heads(hq, hk, nq, dtype):
    check(*make(2, nq, 90, hq, hk, 32, dtype, hq), None, dtype)


@pytest.mark.parametrize("dtype", BOTH, ids=["f32", "bf16"])
@pytest.mark.parametrize("D", [32, 64, 75, 128])
@pytest.mark.parametrize("keep", [0.03, 0.5, 0.97])
def test_masks(keep, D, dtype):
    """One scene keeps no key, one a single key, the rest a share; a mask that keeps all equals none."""
    B, nk = 4, 300
    q, k, v, g = make(B, 70, nk, 4, 2, D, dtype, D)
    mask = random_mask(B, nk, keep, D)
    mask[0] = False
    mask[1] = False
    mask[1, 177] = True
    check(q, k, v, g, mask, dtype)
    from CudaGaussianVoxelizer import gaussian_attention
    q, k, v = q.cuda(), k.cuda(), v.cuda()
    assert torch.count_nonzero(gaussian_attention(q, k, v, mask.cuda())[0]) == 0
    assert torch.equal(gaussian_attention(q, k, v, torch.ones_like(mask).cuda()), gaussian_attention(q, k, v))


@pytest.mark.parametrize("dtype", BOTH, ids=["f32", "bf16"])
@pytest.mark.parametrize("nq", [1, 70])
def test_masked_rows_are_not_read(nq, dtype):
    """NaN, infinities and the type's extremes in masked rows change no bit of any result."""
    from CudaGaussianVoxelizer import gaussian_attention
    B, nk = 2, 400
    q, k, v, g = (t.cuda() for t in make(B, nq, nk, 4, 4, 40, dtype, 3))
    mask = random_mask(B, nk, 0.6, 4).cuda()
    results = []
    for bad in (0.0, float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).min, torch.finfo(dtype).max):
        kb, vb = (torch.where(mask[:, :, None, None], t, torch.full_like(t, bad)) for t in (k, v))
        leaves = [t.detach().clone().requires_grad_() for t in (q, kb, vb)]
        out = gaussian_attention(*leaves, key_mask=mask)
        out.backward(g)
        results.append([out.detach()] + [t.grad for t in leaves])
    for r in results[1:]:
        for a, b in zip(r, results[0]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", BOTH, ids=["f32", "bf16"])
def test_large_scores(dtype):
    """Scores of hundreds: the running maximum moves often and most probabilities vanish."""
    q, k, v, g = make(1, 100, 500, 2, 2, 64, dtype, 8, size=1.0)
    q = q * torch.linspace(0.1, 8.0, 100)[None, :, None, None].to(dtype)
    k = k * torch.linspace(0.2, 6.0, 500)[None, :, None, None].to(dtype)
    from CudaGaussianVoxelizer import gaussian_attention
    out = gaussian_attention(q.cuda(), k.cuda(), v.cuda())
    # a score of 200 carries 200 x 2^-24 (float32) into the exponent: 2e-5 of a probability
    assert rel(out, plain(q, k, v, None)[0]) < (5e-5 if dtype == torch.float32 else 4e-3)


@pytest.mark.parametrize("dtype", BOTH, ids=["f32", "bf16"])
@pytest.mark.parametrize("nq,nk", [(70, 1000), (1, 5000), (300, 700)])
@pytest.mark.parametrize("slope", [0.5, -0.5, 8.0])
def test_references_far_from_the_maximum(slope, nq, nk, dtype):
    """Scores that climb (or fall) by `slope` a key over the whole row, up to 40000: the first tile's reference is far off and
    has to be renewed, and nearly all probabilities vanish.  Powers of two only, so the scores are exact in both types."""
    d = 64
    step = torch.arange(nk) // 64 * 64 if dtype == torch.bfloat16 else torch.arange(nk)   # 8 bits hold 64 * 0 .. 64 * 78
    q, k = torch.zeros(1, nq, 1, d), torch.zeros(1, nk, 1, d)
    q[..., 0] = slope
    q[..., 1] = 1.0
    k[..., 0] = step[None, :, None]
    k[..., 1] = (torch.arange(nk) % 64 * abs(slope) / 16)[None, :, None]
    g = torch.Generator().manual_seed(1)
    v, go = torch.randn(1, nk, 1, d, generator=g), torch.randn(1, nq, 1, d, generator=g)
    q, k, v, go = (t.to(dtype) for t in (q, k, v, go))
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    from CudaGaussianVoxelizer import gaussian_attention
    out = gaussian_attention(*leaves, scale=1.0)
    out.backward(go.cuda())
    want = plain(q, k, v, None, go, 1.0)
    # float32 scores of 40000 carry 2^-9 into the exponent at worst: 2^-24 x 40000 x log2(e), 3.4e-3
    tol = 4e-3 if dtype == torch.float32 else 8e-3
    assert rel(out, want[0]) < tol
    for t, w in zip(leaves[1:], want[2:]):
        assert torch.isfinite(t.grad).all()
    assert rel(leaves[2].grad, want[3]) < tol


@pytest.mark.parametrize("D", [32, 64, 100, 128])
@pytest.mark.parametrize("nq,nk", [(70, 1000), (1, 5000), (300, 700)])
def test_first_keys_with_scores_of_minus_infinity(nq, nk, D):
    """bfloat16 keys whose scores are -inf fill the first tiles, and the others' scores are about -200 (2^-288 without a
    reference): the result is that of the other keys alone."""
    q, k, v, _ = make(1, nq, nk, 2, 2, D, torch.bfloat16, 21, size=0.3)
    q[..., 0], q[..., 1] = 1.0, 1.0
    k[:, :150, :, 0] = -float("inf")
    k[:, 150:, :, 0] = 0.0
    k[..., 1] = -200.0
    mask = (torch.arange(nk) >= 150)[None]
    from CudaGaussianVoxelizer import gaussian_attention
    out = gaussian_attention(q.cuda(), k.cuda(), v.cuda(), scale=1.0)
    # scores of 200 carry 200 x 2^-24 into the exponent, far below the rounding of bfloat16 probabilities and outputs
    assert rel(out, plain(q, k, v, mask, scale=1.0)[0]) < TOL[torch.bfloat16][0]


@pytest.mark.parametrize("dtype", BOTH, ids=["f32", "bf16"])
@pytest.mark.parametrize("scale", [0.01, 1.0])
def test_scale(scale, dtype):
    check(*make(1, 50, 200, 2, 2, 64, dtype, 9, size=0.7), None, dtype, scale)


@pytest.mark.parametrize("D", [16, 64])
def test_gradient_against_differences(D):
    """Central differences of the float64 statement along random directions (step 1e-5: error about 1e-9)."""
    from CudaGaussianVoxelizer import gaussian_attention
    q, k, v, g = make(2, 20, 45, 4, 2, D, torch.float32, 11)
    mask = random_mask(2, 45, 0.7, 5)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    gaussian_attention(*leaves, key_mask=mask.cuda()).backward(g.cuda())
    base = [t.double() for t in (q, k, v)]
    gen = torch.Generator().manual_seed(1)
    for i in range(3):
        u = torch.randn(base[i].shape, generator=gen).double()
        vals = []
        for s in (1, -1):
            m = list(base)
            m[i] = base[i] + s * 1e-5 * u
            vals.append(float((plain(*m, mask)[0] * g.double()).sum()))
        got = leaves[i].grad.double().cpu()
        want = (vals[0] - vals[1]) / 2e-5
        assert abs(float((got * u).sum()) - want) <= 1e-5 * float((got.abs() * u.abs()).sum()), i


@pytest.mark.parametrize("dtype", BOTH, ids=["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 36])
def test_layouts(D, dtype):
    """Views of a fused projection, heads-first storage, data off 16-byte boundaries and transposed rows give the
    contiguous tensors' results bit for bit; expanded heads and scenes too."""
    from CudaGaussianVoxelizer import _C
    B, n, h = 2, 130, 2
    q, k, v, g = (t.cuda() for t in make(B, n, n, h, h, D, dtype, 6))
    want = _C.attention_forward(q, k, v, for_backward=True)
    gwant = _C.attention_backward(g, q, k, v, *want[:3])

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
        got = _C.attention_forward(qv, kv, vv, for_backward=True)
        assert all(a is b is None or torch.equal(a, b) for a, b in zip(got, want))
        for a, b in zip(_C.attention_backward(gv, qv, kv, vv, *got[:3]), gwant):
            assert torch.equal(a, b)
    one = k[:1, :, :1].expand(B, n, h, D)
    assert torch.equal(_C.attention_forward(q, one, one)[0], _C.attention_forward(q, one.contiguous(), one.contiguous())[0])


@pytest.mark.parametrize("stride", [40000, 1 << 24])
def test_offsets_beyond_32_bits(stride):
    """Keys whose rows lie further apart than 32 bits reach: views of a 5 GB buffer, read in place, and of wide strides, packed."""
    from CudaGaussianVoxelizer import _C
    n = (5 << 30) // 2 // stride + 2
    buf = torch.empty(n * stride + 256, dtype=torch.bfloat16, device="cuda")
    kv = torch.as_strided(buf, (1, n, 2, 64), (0, stride, 64, 1))
    q, k, v, g = (t.cuda() for t in make(1, 40, n, 2, 2, 64, torch.bfloat16, 7))
    kv.copy_(k)
    want = _C.attention_forward(q, k, v, for_backward=True)
    got = _C.attention_forward(q, kv, v, for_backward=True)
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(got, want))
    for a, b in zip(_C.attention_backward(g, q, kv, v, *got[:3]), _C.attention_backward(g, q, k, v, *want[:3])):
        assert torch.equal(a, b)
    pos, fr = torch.rand(1, n, 3, device="cuda") * 80, torch.rand(3, 30, device="cuda")
    assert torch.equal(_C.qk_norm_rotary_forward(kv, None, pos, fr)[0], _C.qk_norm_rotary_forward(k, None, pos, fr)[0])


@pytest.mark.parametrize("dtype", BOTH, ids=["f32", "bf16"])
@pytest.mark.parametrize("nq,nk,masked", [(1, 3000, False), (300, 300, True), (700, 900, False)])
def test_graph_replays(nq, nk, masked, dtype):
    """A captured step gives the eager step's results on every replay, with eager work and new inputs between the replays."""
    from CudaGaussianVoxelizer import _C
    q, k, v, g = (t.cuda() for t in make(2, nq, nk, 4, 2, 64, dtype, 5))
    mask = random_mask(2, nk, 0.7, 3).cuda() if masked else None

    def step(q, k, v, g):
        out, rest, lse, lst = _C.attention_forward(q, k, v, mask, for_backward=True)
        return (out,) + _C.attention_backward(g, q, k, v, out, rest, lse, lst)

    static = [t.clone() for t in (q, k, v, g)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = step(*static)
    for i in range(4):
        new = [t.cuda() for t in make(2, nq, nk, 4, 2, 64, dtype, 20 + i)]
        for a, b in zip(static, new):
            a.copy_(b)
        graph.replay()
        want = step(*new)
        torch.cuda.synchronize()
        for a, b in zip(results, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", BOTH, ids=["f32", "bf16"])
def test_empty(dtype):
    from CudaGaussianVoxelizer import gaussian_attention
    for B, nq, nk in ((0, 3, 4), (2, 0, 5), (2, 5, 0), (2, 0, 0)):
        q, k, v, g = make(B, nq, nk, 4, 2, 32, dtype, 1)
        leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
        for mask in (None, torch.ones(B, nk, dtype=torch.bool, device="cuda")):
            out = gaussian_attention(*leaves, key_mask=mask)
            assert out.shape == q.shape and torch.count_nonzero(out) == 0
            for t, grad in zip(leaves, torch.autograd.grad(out, leaves, g.cuda())):
                assert grad.shape == t.shape and torch.count_nonzero(grad) == 0


@pytest.mark.parametrize("dtype", BOTH, ids=["f32", "bf16"])
@pytest.mark.parametrize("nq,nk", [(1, 9000), (2100, 2100)])
def test_runs_are_equal_and_streams_are_the_callers(nq, nk, dtype):
    """Three passes without a wait between them, the second on other inputs, on a stream of the caller's."""
    from CudaGaussianVoxelizer import _C
    sets = [[t.cuda() for t in make(1, nq, nk, 4, 4, 64, dtype, s)] for s in (1, 2)]

    def both(q, k, v, g):
        out, rest, lse, _ = _C.attention_forward(q, k, v, for_backward=True)
        return (out,) + _C.attention_backward(g, q, k, v, out, rest, lse)

    want = both(*sets[0])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        first = both(*sets[0])
        both(*sets[1])
        last = both(*sets[0])
    s.synchronize()
    for a, b, c in zip(want, first, last):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_partial_gradients():
    """Only the wanted gradients are computed, and they are the same."""
    from CudaGaussianVoxelizer import gaussian_attention
    q, k, v, g = (t.cuda() for t in make(1, 60, 80, 2, 2, 32, torch.bfloat16, 2))
    full = [t.clone().requires_grad_() for t in (q, k, v)]
    gaussian_attention(*full).backward(g)
    for i in range(3):
        some = [t.clone().requires_grad_(j == i) for j, t in enumerate((q, k, v))]
        gaussian_attention(*some).backward(g)
        assert torch.equal(some[i].grad, full[i].grad)
        assert all(t.grad is None for j, t in enumerate(some) if j != i)


def test_refusals():
    from CudaGaussianVoxelizer import gaussian_attention
    q = torch.ones(1, 4, 4, 16, device="cuda")
    k = torch.ones(1, 6, 2, 16, device="cuda")
    good = dict(q=q, k=k, v=k)
    gaussian_attention(**good)
    wide = torch.ones(1, 4, 4, 129, device="cuda")
    bad = [
        dict(q=q.half()), dict(q=q.double()), dict(q=q.cpu()), dict(q=q[0]), dict(k=k.bfloat16()), dict(v=k[:, :5]),
        dict(v=k[..., :8]), dict(q=q[:, :, :3]), dict(k=k.expand(2, 6, 2, 16), v=k.expand(2, 6, 2, 16)), dict(q=q[:, :, :0]),
        dict(q=wide, k=wide, v=wide), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")),
        dict(key_mask=torch.ones(1, 6, device="cuda")), dict(key_mask=torch.ones(1, 5, dtype=torch.bool, device="cuda")),
        dict(key_mask=torch.ones(1, 6, dtype=torch.bool)), dict(q=None),
    ]
    for b in bad:
        with pytest.raises(RuntimeError):
            gaussian_attention(**dict(good, **b))


@pytest.mark.parametrize("nq,nk,H,D,dtype,keep", [
    (99, 1301, 24, 64, torch.float32, 1.0), (641, 1299, 12, 64, torch.float32, 1.0), (641, 1299, 12, 64, torch.float32, 0.6),
    (300, 201, 88, 64, torch.float32, 1.0), (401, 640, 36, 64, torch.float32, 1.0), (699, 641, 44, 64, torch.float32, 0.9),
    (700, 200, 88, 64, torch.float32, 1.0), (700, 640, 44, 64, torch.float32, 1.0),
    (500, 1300, 48, 128, torch.bfloat16, 1.0), (401, 3000, 68, 128, torch.bfloat16, 1.0)])
def test_rounds_of_workgroups(nq, nk, H, D, dtype, keep):
    """Tiles that fill the card once and a little: the first ones whole or in two splits, the rest in more."""
    check(*make(1, nq, nk, H, H, D, dtype, nq + nk), None if keep == 1.0 else random_mask(1, nk, keep, nk), dtype)


def _largest_keys():
    """Keys of up to the largest float32 in one channel, where queries are 2^-125: scores of a few units."""
    top = torch.finfo(torch.float32).max
    q, k, v, g = make(1, 70, 300, 2, 2, 32, torch.float32, 13)
    sign = torch.where(torch.arange(300) % 3 == 0, -1.0, 1.0)[None, :, None]
    k[..., 0] = sign * top * torch.linspace(0.9975, 1.0, 300)[None, :, None]
    q[..., 0] = 2.0 ** -125
    return q, k, v, g


def test_largest_finite_values():
    """float32 values beyond the largest bfloat16 (3.39e38) are finite like any other.  Products keep 24 bits as ever: 1e-5."""
    from CudaGaussianVoxelizer import gaussian_attention
    q, k, v, _ = _largest_keys()
    assert rel(gaussian_attention(q.cuda(), k.cuda(), v.cuda()), plain(q, k, v, None)[0]) < 1e-5
    v[..., 3] = float("inf")      # infinities stay what they are
    assert not torch.isfinite(gaussian_attention(q.cuda(), k.cuda(), v.cuda())[..., 3]).any()


def test_gradients_of_largest_finite_values():
    """dQ is a sum over the keys times scale: it is finite wherever that product is, also where the sum alone would not be."""
    from CudaGaussianVoxelizer import gaussian_attention
    q, k, v, g = _largest_keys()
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    gaussian_attention(*leaves).backward(g.cuda())
    for t, w in zip(leaves, plain(q, k, v, None, g)[1:]):
        assert torch.isfinite(t.grad).all() and rel(t.grad, w) < 1e-5


@pytest.mark.parametrize("D", [24, 32, 64, 72, 96, 128])
def test_padding_does_not_cost_accuracy(D):
    """Scenes of few valid keys in a batch that is padded to many: dK and dV of each scene are as near to 64 bits as those of its
    valid keys alone.  The number of planes of P and dS is the same in both then, and with it every rounding but those of float32
    sums (2^-24 each) and of the bfloat16 outputs, which are as large in both: the two errors agree within a few percent, where one
    plane instead of two adds a quarter or more.  (dQ takes two planes always.)"""
    from CudaGaussianVoxelizer import _C
    nk, counts = 3663, [440, 2, 1024, 1025, 3663, 90, 0]
    q, k, v, g = (t.cuda() for t in make(len(counts), 150, nk, 4, 2, D, torch.bfloat16, D))
    # keys of a scene share a direction (the mean of the scores' gradients is what delta takes away)
    k = (k + torch.randn(len(counts), 1, 2, D, generator=torch.Generator().manual_seed(1)).cuda()).bfloat16()
    order = torch.rand(len(counts), nk, generator=torch.Generator().manual_seed(2)).argsort(1).argsort(1)
    mask = order < torch.tensor(counts)[:, None]
    out, rest, lse, lst = _C.attention_forward(q, k, v, mask.cuda(), for_backward=True)
    grads = _C.attention_backward(g, q, k, v, out, rest, lse, lst)
    for b, n in enumerate(counts):
        at, keys = slice(b, b + 1), mask[b].nonzero()[:, 0].cuda()
        assert torch.count_nonzero(grads[1][b][~mask[b].cuda()]) == 0 and torch.count_nonzero(grads[2][b][~mask[b].cuda()]) == 0
        if n < 2:
            continue
        alone = q[at], k[at, keys].contiguous(), v[at, keys].contiguous()
        o, r, l, _ = _C.attention_forward(*alone, for_backward=True)
        lone = _C.attention_backward(g[at], *alone, o, r, l)
        want = plain(*alone, None, g[at])[1:]
        errs = [(rel(x[at, keys], w), rel(y, w)) for x, y, w in zip(grads[1:], lone[1:], want[1:])]
        say(D, n, " ".join(f"{e:.2e}/{f:.2e}" for e, f in errs))
        assert all(e <= 1.05 * f for e, f in errs), (n, errs)


@pytest.mark.parametrize("dtype", BOTH, ids=["f32", "bf16"])
@pytest.mark.parametrize("nq", [11, 130])
@pytest.mark.parametrize("nk", [2048, 2049, 5000])
def test_masks_of_many_keys(nk, nq, dtype):
    """Masks on both sides of the number of keys up to which packing makes their list: an empty scene, a single key, a valid prefix
    (padding), a valid suffix, a random share, few keys, all; rows of NaN where nothing is attended to."""
    B = 7
    q, k, v, g = make(B, nq, nk, 4, 2, 64, dtype, nk + nq)
    at = torch.arange(nk)
    mask = torch.stack([torch.zeros(nk, dtype=torch.bool), at == nk - 1, at < 1300, at >= nk - 700, random_mask(1, nk, 0.8, 1)[0],
                        random_mask(1, nk, 0.02, 2)[0], torch.ones(nk, dtype=torch.bool)])
    check(q, k, v, g, mask, dtype)
    from CudaGaussianVoxelizer import gaussian_attention
    results = []
    for bad in (0.0, float("nan")):
        kb, vb = (torch.where(mask[:, :, None, None], t, torch.full_like(t, bad)) for t in (k, v))
        leaves = [t.cuda().requires_grad_() for t in (q, kb, vb)]
        out = gaussian_attention(*leaves, key_mask=mask.cuda())
        out.backward(g.cuda())
        results.append([out.detach()] + [t.grad for t in leaves])
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("nq,nk", [(10, 1500), (200, 300), (200, 1500)])
def test_backward_without_the_rounding_lost(nq, nk):
    """A bfloat16 backward whose caller did not keep what rounding took from the output: delta is off by that rounding, within the
    bound of gradients."""
    from CudaGaussianVoxelizer import _C
    q, k, v, g = make(1, nq, nk, 4, 2, 64, torch.bfloat16, nk)
    dev = [t.cuda() for t in (q, k, v)]
    out, rest, lse, _ = _C.attention_forward(*dev, for_backward=True)
    assert rest is not None
    got = _C.attention_backward(g.cuda(), *dev, out, None, lse)
    for x, y in zip(got, plain(q, k, v, None, g)[1:]):
        assert rel(x, y) < TOL[torch.bfloat16][1]


@pytest.mark.parametrize("dtype", BOTH, ids=["f32", "bf16"])
@pytest.mark.parametrize("nq,nk", [(70, 1000), (1, 5000), (300, 700)])
@pytest.mark.parametrize("slope", [0.5, -0.5])
def test_gradients_far_from_the_maximum(slope, nq, nk, dtype):
    """dQ and dK where scores climb over the whole row.  Their terms cancel (keys lie far from 0, and one or a few of them have all
    the probability), so errors are measured against the sums of the terms' magnitudes: a float32 score of 2500 carries at
    most 2500 x 2^-24 x log2(e) into the exponent, 2.1e-4 of a probability, bfloat16 rounds outputs to 2^-9 (and P and dS, or their
    second planes).  A term takes P twice (its own and delta's): 1e-3 and 8e-3."""
    d = 64
    step = torch.arange(nk) // 64 * 64 if dtype == torch.bfloat16 else torch.arange(nk)
    q, k = torch.zeros(1, nq, 1, d), torch.zeros(1, nk, 1, d)
    q[..., 0] = slope
    q[..., 1] = 1.0
    k[..., 0] = step[None, :, None]
    k[..., 1] = (torch.arange(nk) % 64 * abs(slope) / 16)[None, :, None]
    gen = torch.Generator().manual_seed(1)
    v, go = torch.randn(1, nk, 1, d, generator=gen), torch.randn(1, nq, 1, d, generator=gen)
    q, k, v, go = (t.to(dtype) for t in (q, k, v, go))
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    from CudaGaussianVoxelizer import gaussian_attention
    gaussian_attention(*leaves, scale=1.0).backward(go.cuda())
    _, dq, dk, _ = plain(q, k, v, None, go, 1.0)
    Q, K, V, G = (t[0, :, 0].double() for t in (q, k, v, go))
    p, dp = torch.softmax(Q @ K.T, -1), G @ V.T
    size = p * (dp.abs() + (p * dp.abs()).sum(-1, keepdim=True))
    tol = 1e-3 if dtype == torch.float32 else 8e-3
    for got, want, most in ((leaves[0].grad, dq, size @ K.abs()), (leaves[1].grad, dk, size.T @ Q.abs())):
        err = float((got.double().cpu()[0, :, 0] - want[0, :, 0]).norm() / most.norm())
        say(f"{err:.1e}")
        assert err < tol
