"""GPU tests of PyGaussianAttention: the layer against the same layer written in float64, gradients of every parameter, input
and position included, and the example that trains through it and the voxelizer.

Tolerance: the projections are float32 library products of at most 96 terms (2^-24 each, summed: below 1e-6), the
operators' own bounds are 1e-5; together below 3e-5.
"""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def rel(x, y):
    x, y = x.detach().double().cpu(), y.detach().double().cpu()
    return float((x - y).norm() / y.norm())


def plain_layer(layer, p, x, positions, mask, context, context_positions):
    """The layer in float64 from its parameters p."""
    H, K, D = layer.heads, layer.kv_heads, layer.head_dim
    c, cpos = (x, positions) if context is None else (context, context_positions)
    q = (x @ p["to_q.weight"].T).unflatten(-1, (H, D))
    kv = (c @ p["to_kv.weight"].T).unflatten(-1, (2 * K, D))
    k, v = kv[:, :, :K], kv[:, :, K:]
    F = layer.freqs.double().cpu()

    def turn(t, w, pos):
        t = t * (t.square().mean(-1, keepdim=True) + layer.eps).rsqrt() * w
        a = (pos @ F)[:, :, None]
        n = 2 * F.shape[1]
        z = torch.view_as_complex(t[..., :n].unflatten(-1, (-1, 2)).contiguous()) * torch.polar(torch.ones_like(a), a)
        return torch.cat([torch.view_as_real(z).flatten(-2), t[..., n:]], -1)

    q, k = turn(q, p["q_weight"], positions), turn(k, p["k_weight"], cpos)
    k, v = k.repeat_interleave(H // K, 2), v.repeat_interleave(H // K, 2)
    s = torch.matmul(q.transpose(1, 2), k.permute(0, 2, 3, 1)) * D ** -0.5
    if mask is not None:
        s = s.masked_fill(~mask[:, None, None], -torch.inf)
    y = torch.matmul(s.softmax(-1), v.transpose(1, 2)).transpose(1, 2)
    return y.flatten(2) @ p["to_out.weight"].T


@pytest.mark.parametrize("cross", [False, True])
@pytest.mark.parametrize("masked", [False, True])
def test_layer(masked, cross):
    from CudaGaussianVoxelizer import PyGaussianAttention
    torch.manual_seed(3)
    layer = PyGaussianAttention(96, 6, 2, wavelengths=(0.8, 40.0))
    B, N, M = 2, 130, 77
    g = torch.Generator().manual_seed(5)
    ins = {"x": torch.randn(B, N, 96, generator=g), "positions": torch.rand(B, N, 3, generator=g) * 20 - 10}
    if cross:
        ins["context"] = torch.randn(B, M, 96, generator=g)
        ins["context_positions"] = torch.rand(B, M, 3, generator=g) * 20 - 10
    mask = torch.rand(B, M if cross else N, generator=g) < 0.7 if masked else None
    go = torch.randn(B, N, 96, generator=g)
    with torch.no_grad():   # weights that are not all ones
        layer.q_weight += 0.2 * torch.randn(16, generator=g).cuda()
        layer.k_weight += 0.2 * torch.randn(16, generator=g).cuda()
    dev = {n: t.cuda().requires_grad_() for n, t in ins.items()}
    y = layer(dev["x"], dev["positions"], None if mask is None else mask.cuda(), context=dev.get("context"),
              context_positions=dev.get("context_positions"))
    y.backward(go.cuda())
    ref = {n: t.double().requires_grad_() for n, t in ins.items()}
    p = {n: t.detach().double().cpu().requires_grad_() for n, t in layer.named_parameters()}
    want = plain_layer(layer, p, ref["x"], ref["positions"], mask, ref.get("context"), ref.get("context_positions"))
    want.backward(go.double())
    assert rel(y, want) < 3e-5
    for n, t in layer.named_parameters():
        assert rel(t.grad, p[n].grad) < 3e-5, n
    for n in ins:
        assert rel(dev[n].grad, ref[n].grad) < 3e-5, n


def test_layer_refusals():
    from CudaGaussianVoxelizer import PyGaussianAttention
    with pytest.raises(RuntimeError):
        PyGaussianAttention(96, 7)
    with pytest.raises(RuntimeError):
        PyGaussianAttention(96, 6, 4)
    with pytest.raises(RuntimeError):
        PyGaussianAttention(8, 4)     # two values a head hold no pair for three axes
    layer = PyGaussianAttention(96, 6)
    with pytest.raises(RuntimeError):
        layer(torch.zeros(1, 4, 96, device="cuda"), torch.zeros(1, 4, 3, device="cuda"),
              context=torch.zeros(1, 4, 96, device="cuda"))


@pytest.mark.parametrize("bf16", [False, True])
def test_example_trains(bf16):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import gaussian_features_step as example
    finally:
        sys.path.pop(0)
    losses = example.train(gaussians=600, scenes=2, channels=64, steps=6, bf16=bf16)
    assert len(losses) == 6 and all(l == l for l in losses)
    assert losses[-1] < losses[0] - 0.05


def test_gradients_of_gradients_are_refused():
    from CudaGaussianVoxelizer import gaussian_attention, qk_norm_rotary, rotary_frequencies
    x = torch.randn(1, 9, 2, 8, device="cuda", requires_grad=True)
    y = gaussian_attention(x, x, x)
    (g,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
    pos = torch.rand(1, 9, 3, device="cuda")
    q, k = qk_norm_rotary(x, x, pos, rotary_frequencies(8))
    (g,) = torch.autograd.grad((q * k).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_forward_mode_is_refused():
    """A tangent of any differentiable input is refused instead of being dropped, with or without gradients enabled; inside a dual
    level inputs without tangents give what they give outside."""
    import torch.autograd.forward_ad as fwad
    from CudaGaussianVoxelizer import gaussian_attention, qk_norm_rotary, rotary_frequencies
    q, k, v = (torch.randn(1, 9, 2, 8, device="cuda") for _ in range(3))
    w = torch.ones(8, device="cuda")
    attn = dict(q=q, k=k, v=v)
    norm = dict(q=q, k=k, positions=torch.rand(1, 9, 3, device="cuda"), freqs=rotary_frequencies(8), q_weight=w, k_weight=w,
                k_positions=torch.rand(1, 9, 3, device="cuda"))
    layer = PyGaussianAttentionOf8()
    want = gaussian_attention(**attn), qk_norm_rotary(**norm)[1], layer(q.flatten(2), norm["positions"])
    with fwad.dual_level():
        assert torch.equal(gaussian_attention(**attn), want[0]) and torch.equal(qk_norm_rotary(**norm)[1], want[1])
        for call, args in ((gaussian_attention, attn), (qk_norm_rotary, norm)):
            for name, t in args.items():
                for enabled in (True, False):
                    dual = fwad.make_dual(t, torch.ones_like(t))
                    with torch.set_grad_enabled(enabled), pytest.raises((RuntimeError, NotImplementedError)):
                        call(**dict(args, **{name: dual}))
        x = fwad.make_dual(q.flatten(2), torch.ones_like(q.flatten(2)))
        with torch.no_grad(), pytest.raises((RuntimeError, NotImplementedError)):
            layer(x, norm["positions"])
    assert torch.equal(layer(q.flatten(2), norm["positions"]), want[2])


def PyGaussianAttentionOf8():
    from CudaGaussianVoxelizer import PyGaussianAttention
    return PyGaussianAttention(16, 2)


@pytest.mark.parametrize("where", ["cpu", "cuda"])
def test_converted_layer(where):
    """A layer converted to bfloat16 (and moved) is the one built in bfloat16: outputs and gradients bit for bit."""
    from CudaGaussianVoxelizer import PyGaussianAttention
    torch.manual_seed(4)
    built = PyGaussianAttention(96, 6, 2, wavelengths=(0.8, 40.0), dtype=torch.bfloat16)
    layer = PyGaussianAttention(96, 6, 2, wavelengths=(0.8, 40.0), device=where)
    layer.load_state_dict(built.state_dict())
    layer = layer.bfloat16().cuda()
    g = torch.Generator().manual_seed(6)
    x, go = (torch.randn(2, 70, 96, generator=g).bfloat16().cuda() for _ in range(2))
    pos = (torch.rand(2, 70, 3, generator=g) * 80 - 40).cuda()
    results = []
    for m in (built, layer):
        xi, pi = x.clone().requires_grad_(), pos.clone().requires_grad_()
        y = m(xi, pi)
        y.backward(go)
        results.append([y.detach(), xi.grad, pi.grad, m.to_q.weight.grad, m.q_weight.grad.bfloat16()])
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("masked", [False, True])
def test_bfloat16_layer(masked):
    """The bfloat16 layer against 64 bits.  On its way an output is rounded eight times (q, k, v, the two normed and turned, the
    probabilities, the attention's output, the last projection), by at most 2^-9 each, 2e-3 added up linearly: below 1.6e-2; a
    gradient passes as many roundings again on its way back: below 3.2e-2."""
    from CudaGaussianVoxelizer import PyGaussianAttention
    torch.manual_seed(8)
    layer = PyGaussianAttention(96, 6, 2, wavelengths=(0.8, 40.0), dtype=torch.bfloat16)
    B, N = 2, 130
    g = torch.Generator().manual_seed(9)
    x, go = (torch.randn(B, N, 96, generator=g).bfloat16() for _ in range(2))
    pos = torch.rand(B, N, 3, generator=g) * 20 - 10
    mask = torch.rand(B, N, generator=g) < 0.7 if masked else None
    xd, pd = x.cuda().requires_grad_(), pos.cuda().requires_grad_()
    y = layer(xd, pd, None if mask is None else mask.cuda())
    y.backward(go.cuda())
    xr, pr = x.double().requires_grad_(), pos.double().requires_grad_()
    p = {n: t.detach().double().cpu().requires_grad_() for n, t in layer.named_parameters()}
    want = plain_layer(layer, p, xr, pr, mask, None, None)
    want.backward(go.double())
    assert y.dtype == torch.bfloat16 and rel(y, want) < 1.6e-2
    assert rel(xd.grad, xr.grad) < 3.2e-2 and rel(pd.grad, pr.grad) < 3.2e-2
    for n, t in layer.named_parameters():
        assert rel(t.grad, p[n].grad) < 3.2e-2, n
