"""GPU parity of the query/key norms with rotary positions (g2v_qk_norm_rotary_*) against a plain float64 statement of
the formula, whose gradients come from autograd, and against differences of that statement.

Tolerances (L2-relative): float32 results are sums of at most 256 products, a root and one sine of an angle that is
itself a float32 sum: 2^-24 times the largest angle (about 300 radians here, a tenth of the pairs near it) plus a few
roundings, below 1e-5.  A bfloat16 result is rounded once: 2^-9 at most, below 4e-3.  Sums over tokens (weights) and heads
(positions) are float32 in both.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 1e-5, torch.bfloat16: 4e-3}


def say(*a):
    print(*a, flush=True)


def rel(x, y):
    x, y = x.double().cpu(), y.double().cpu()
    n = y.norm()
    return float((x - y).norm() / n) if n > 0 else float(x.norm())


def plain(x, w, pos, freqs, eps):
    """One tensor's rows in the arguments' precision (float64 here)."""
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    y = x * r if w is None else x * r * w
    P = freqs.shape[1]
    t = torch.einsum("bna,ap->bnp", pos, freqs)[:, :, None]
    c, s = t.cos(), t.sin()
    y0, y1 = y[..., 0:2 * P:2], y[..., 1:2 * P:2]
    rot = torch.stack([y0 * c - y1 * s, y0 * s + y1 * c], -1).flatten(-2)
    return torch.cat([rot, y[..., 2 * P:]], -1)


def make(B, nq, nk, hq, hk, D, axes, pairs, dtype, seed, shared, weights=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)   # noqa: E731
    d = {"q": r(B, nq, hq, D).to(dtype), "k": None if hk == 0 else r(B, nq if shared else nk, hk, D).to(dtype),
         "pos": torch.rand(B, nq, axes, generator=g) * 80 - 40, "freqs": torch.rand(axes, pairs, generator=g) * 2.0,
         "qw": r(D) * 0.2 + 1 if weights else None, "kw": r(D) * 0.2 + 1 if weights and hk else None,
         "kpos": None if shared or hk == 0 else torch.rand(B, nk, axes, generator=g) * 80 - 40}
    return d, r


CASES = [
    # B, nq, nk, hq, hk, D, axes, pairs, dtype, shared
    (1, 1, 1, 1, 1, 2, 1, 1, torch.float32, True),
    (1, 5, 5, 3, 1, 7, 2, 2, torch.float32, True),
    (2, 300, 300, 8, 8, 32, 3, 15, torch.float32, True),
    (2, 33, 129, 6, 2, 75, 3, 36, torch.float32, False),
    (1, 257, 100, 4, 4, 256, 4, 128, torch.float32, False),
    (1, 300, 300, 8, 8, 64, 3, 30, torch.bfloat16, True),
    (3, 65, 65, 12, 4, 72, 3, 36, torch.bfloat16, True),
    (2, 17, 40, 2, 5, 33, 1, 0, torch.bfloat16, False),
    (1, 4099, 4099, 5, 2, 128, 3, 63, torch.bfloat16, True),
    (2, 50, 1, 4, 0, 64, 8, 8, torch.float32, True),
]


@pytest.mark.parametrize("case", CASES, ids=[str(c[:8]) for c in CASES])
def test_parity(case):
    from CudaGaussianVoxelizer import qk_norm_rotary
    B, nq, nk, hq, hk, D, axes, pairs, dtype, shared = case
    say(f"[qk_norm] {case}")
    eps = 1e-6
    d, r = make(*case[:9], seed=D, shared=shared)
    leaves = {n: (None if t is None else t.cuda().requires_grad_(n != "freqs")) for n, t in d.items()}
    oq, ok = qk_norm_rotary(leaves["q"], leaves["k"], leaves["pos"], leaves["freqs"], leaves["qw"], leaves["kw"],
                            k_positions=leaves["kpos"], eps=eps)
    ref = {n: (None if t is None else t.double().requires_grad_(n != "freqs")) for n, t in d.items()}
    rq = plain(ref["q"], ref["qw"], ref["pos"], ref["freqs"], eps)
    assert oq.dtype == dtype and oq.is_contiguous() and rel(oq, rq.detach()) < TOL[dtype]
    outs, refs, gs = [oq], [rq], [r(*oq.shape).to(dtype)]
    if hk:
        rk = plain(ref["k"], ref["kw"], ref["pos"] if shared else ref["kpos"], ref["freqs"], eps)
        assert rel(ok, rk.detach()) < TOL[dtype]
        outs, refs, gs = outs + [ok], refs + [rk], gs + [r(*ok.shape).to(dtype)]
    else:
        assert ok is None
    torch.autograd.backward(outs, [g.cuda() for g in gs])
    torch.autograd.backward(refs, [g.double() for g in gs])
    for n in ("q", "k", "pos", "qw", "kw", "kpos"):
        if leaves[n] is not None:
            tol = TOL[dtype] if n in ("q", "k") else TOL[torch.float32]
            want = ref[n].grad if ref[n].grad is not None else torch.zeros_like(ref[n])
            assert rel(leaves[n].grad, want) < tol, n


def test_gradient_against_differences():
    """Central differences of the float64 statement along random directions (step 1e-5: error 1e-10 relative)."""
    from CudaGaussianVoxelizer import qk_norm_rotary
    d, r = make(2, 9, 9, 3, 2, 20, 3, 9, torch.float32, 3, True)
    leaves = {n: t.cuda().requires_grad_(n != "freqs") for n, t in d.items() if t is not None}
    gq, gk = r(2, 9, 3, 20), r(2, 9, 2, 20)
    oq, ok = qk_norm_rotary(leaves["q"], leaves["k"], leaves["pos"], leaves["freqs"], leaves["qw"], leaves["kw"], eps=1e-3)
    torch.autograd.backward([oq, ok], [gq.cuda(), gk.cuda()])

    def value(m):
        return float((plain(m["q"], m["qw"], m["pos"], m["freqs"], 1e-3) * gq.double()).sum()
                     + (plain(m["k"], m["kw"], m["pos"], m["freqs"], 1e-3) * gk.double()).sum())

    base = {n: t.double() for n, t in d.items() if t is not None}
    for n in ("q", "k", "pos", "qw", "kw"):
        u = r(*d[n].shape).double()
        step = [value(dict(base, **{n: base[n] + s * 1e-5 * u})) for s in (1, -1)]
        want, got = (step[0] - step[1]) / 2e-5, float((leaves[n].grad.double().cpu() * u).sum())
        size = float((leaves[n].grad.double().cpu().abs() * u.abs()).sum())   # what the sum's roundings scale with
        assert abs(got - want) <= 1e-5 * size, n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 36])
def test_layouts(dtype, D):
    """Views of a fused projection, heads-first storage, rows off 16-byte boundaries, expanded scenes and a transposed row
    give the contiguous tensors' results bit for bit (forward and backward)."""
    from CudaGaussianVoxelizer import _C
    B, n, h = 2, 70, 4
    d, r = make(B, n, n, h, h, D, 3, 9, dtype, 5, True)
    pos, fr, qw = d["pos"].cuda(), d["freqs"].cuda(), d["qw"].cuda()
    q, k = d["q"].cuda(), d["k"].cuda()
    g = r(B, n, h, D).to(dtype).cuda()
    want = _C.qk_norm_rotary_forward(q, k, pos, fr, qw, None)
    gwant = _C.qk_norm_rotary_backward(g, g, q, k, pos, fr, qw, None)

    def views(t):
        fused = torch.randn(B, n, 3 * h, D, device="cuda").to(dtype)
        fused[:, :, h:2 * h] = t
        yield fused[:, :, h:2 * h]
        yield t.transpose(1, 2).contiguous().transpose(1, 2)
        flat = torch.zeros(t.numel() + 1, dtype=dtype, device="cuda")
        flat[1:] = t.flatten()
        yield flat[1:].view(t.shape)
        yield t.transpose(2, 3).contiguous().transpose(2, 3)

    for qv, kv, gv in zip(views(q), views(k), views(g)):
        got = _C.qk_norm_rotary_forward(qv, kv, pos, fr, qw, None)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        ggot = _C.qk_norm_rotary_backward(gv, gv, qv, kv, pos, fr, qw, None)
        for a, b in zip(ggot, gwant):
            assert (a is None and b is None) or torch.equal(a, b)
    one = q[:1].expand(B, n, h, D)
    assert torch.equal(_C.qk_norm_rotary_forward(one, None, pos, fr)[0],
                       _C.qk_norm_rotary_forward(one.contiguous(), None, pos, fr)[0])


def test_empty_and_zero_rows():
    from CudaGaussianVoxelizer import qk_norm_rotary
    dev = torch.device("cuda")
    fr = torch.rand(3, 10, device=dev)
    w = torch.ones(32, device=dev, requires_grad=True)
    q = torch.zeros(2, 0, 4, 32, device=dev, requires_grad=True)
    oq, ok = qk_norm_rotary(q, q, torch.zeros(2, 0, 3, device=dev), fr, w, w)
    assert oq.shape == q.shape and ok.shape == q.shape
    oq.sum().backward()
    assert torch.equal(w.grad, torch.zeros_like(w)) and q.grad.shape == q.shape
    # rows of zeros have a norm of eps alone: outputs 0, gradients finite
    z = torch.zeros(1, 3, 2, 32, device=dev, requires_grad=True)
    o, _ = qk_norm_rotary(z, None, torch.ones(1, 3, 3, device=dev), fr)
    assert torch.equal(o, torch.zeros_like(o))
    o.sum().backward()
    assert torch.isfinite(z.grad).all()


def test_runs_are_equal_and_streams_are_the_callers():
    from CudaGaussianVoxelizer import _C
    d, r = make(1, 3000, 3000, 8, 8, 64, 3, 30, torch.bfloat16, 9, True)
    q, k, pos, fr = (d[n].cuda() for n in ("q", "k", "pos", "freqs"))
    g = r(*q.shape).bfloat16().cuda()
    want = _C.qk_norm_rotary_backward(g, g, q, k, pos, fr)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _C.qk_norm_rotary_backward(g, g, q, k, pos, fr)
    s.synchronize()
    for a, b in zip(got, want):
        assert (a is None and b is None) or torch.equal(a, b)


def test_refusals():
    from CudaGaussianVoxelizer import qk_norm_rotary
    dev = torch.device("cuda")
    q, pos, fr = torch.ones(1, 4, 2, 16, device=dev), torch.ones(1, 4, 3, device=dev), torch.ones(3, 8, device=dev)
    bad = [
        dict(q=q.half()), dict(q=q.cpu()), dict(q=q[0]), dict(k=q.bfloat16()), dict(k=q[:, :3]), dict(k=q[..., :8]),
        dict(positions=pos[:, :3]), dict(positions=pos.double()), dict(positions=None), dict(freqs=torch.ones(2, 8, device=dev)),
        dict(freqs=torch.ones(3, 9, device=dev)), dict(freqs=fr.clone().requires_grad_()), dict(q_weight=torch.ones(8, device=dev)),
        dict(k_positions=pos[:, :2], k=q), dict(eps=-1.0), dict(eps=float("nan")),
        dict(q=torch.ones(1, 4, 2, 257, device=dev), k=None),
    ]
    for b in bad:
        args = dict(dict(q=q, k=None, positions=pos, freqs=fr), **b)
        with pytest.raises(RuntimeError):
            qk_norm_rotary(**args)


@pytest.mark.parametrize("shared", [True, False])
@pytest.mark.parametrize("wanted", ["pos", "qw", "kw", "q", "k"])
def test_single_gradients(wanted, shared):
    """One input alone wants a gradient: it is the one of the call that gives all, bit for bit."""
    from CudaGaussianVoxelizer import qk_norm_rotary
    d, _ = make(2, 70, 130, 6, 3, 24, 3, 12, torch.float32, 5, shared)
    d = {n: None if t is None else t.cuda() for n, t in d.items()}
    g = torch.Generator().manual_seed(9)
    go = [torch.randn(t.shape, generator=g).cuda() for t in (d["q"], d["k"])]
    grads = []
    for names in ([n for n, t in d.items() if t is not None and n != "freqs"], [wanted]):
        leaves = {n: None if t is None else t.detach().clone().requires_grad_(n in names) for n, t in d.items()}
        out = qk_norm_rotary(leaves["q"], leaves["k"], leaves["pos"], leaves["freqs"], leaves["qw"], leaves["kw"],
                             k_positions=leaves["kpos"])
        torch.autograd.backward(out, go)
        grads.append(leaves[wanted].grad)
    assert grads[0] is not None and torch.equal(*grads)


def test_no_query_heads():
    """Keys alone with the queries' positions: their gradient is the keys'."""
    from CudaGaussianVoxelizer import qk_norm_rotary
    d, _ = make(2, 40, 40, 4, 2, 16, 3, 8, torch.float32, 6, False)
    g = torch.Generator().manual_seed(10)
    go = torch.randn(2, 40, 2, 16, generator=g).cuda()
    res = []
    for empty in (True, False):
        k, pos = d["k"].cuda().requires_grad_(), d["kpos"].cuda().requires_grad_()
        fr, kw = d["freqs"].cuda(), d["kw"].cuda()
        if empty:
            q, out = qk_norm_rotary(torch.empty(2, 40, 0, 16, device="cuda"), k, pos, fr, None, kw)
            assert q.shape == (2, 40, 0, 16)
        else:
            out, _ = qk_norm_rotary(k, None, pos, fr, kw)
        out.backward(go)
        res.append((out.detach(), k.grad, pos.grad))
    for x, y in zip(*res):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("hq,hk,shared", [(0, 2, False), (3, 0, False), (0, 0, False), (0, 0, True)])
def test_positions_of_a_side_without_heads(hq, hk, shared, dtype):
    """A side without heads: its positions and weights turn and scale nothing, so their gradients are zeros (and not what their
    memory held), and the other side's are those of the call without it."""
    from CudaGaussianVoxelizer import _C, qk_norm_rotary
    B, nq, nk, D = 2, 700, 700 if shared else 900, 16
    d, r = make(B, nq, nk, max(hq, 1), max(hk, 1), D, 3, 8, dtype, 11, shared)
    fr = d["freqs"].cuda()
    leaf = lambda t: t.cuda().requires_grad_()   # noqa: E731
    q, k = leaf(d["q"][:, :, :hq]), leaf(d["k"][:, :, :hk])
    pos, kpos, qw, kw = leaf(d["pos"]), None if shared else leaf(d["kpos"]), leaf(d["qw"]), leaf(d["kw"])
    go = [r(*t.shape).to(dtype).cuda() for t in (q, k)]
    out = qk_norm_rotary(q, k, pos, fr, qw, kw, k_positions=kpos)
    wrt = [q, k, pos, qw, kw] + ([] if shared else [kpos])
    used = [torch.full_like(t, float("nan")) for t in (pos, pos, qw, kw) + (() if shared else (kpos, kpos))]
    torch.cuda.synchronize()
    del used      # whose memory the gradients may get
    dq, dk, dpos, dqw, dkw, *dkpos = torch.autograd.grad(out, wrt, go)
    assert dq.shape == q.shape and dk.shape == k.shape
    if hq == 0:
        assert torch.count_nonzero(dqw) == 0
        assert hk > 0 and shared or torch.count_nonzero(dpos) == 0
    else:
        want = _C.qk_norm_rotary_backward(go[0], None, q, None, pos, fr, qw)
        assert torch.equal(dq, want[0]) and torch.equal(dqw, want[2]) and torch.equal(dpos, want[4])
    if hk == 0:
        assert torch.count_nonzero(dkw) == 0
        assert all(torch.count_nonzero(t) == 0 for t in dkpos)
    else:
        want = _C.qk_norm_rotary_backward(go[1], None, k, None, kpos, fr, kw)
        assert torch.equal(dk, want[0]) and torch.equal(dkw, want[2]) and torch.equal(dkpos[0], want[4])
