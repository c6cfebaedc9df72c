"""GPU tests of what a deep stack of attention layers over a scene runs together: PyGaussianAttention with a window, PyLayerNorm with the
residual sum, clip_grad_norm_, and the example that trains with them.

Tolerance of a layer: the projections are float32 library products of at most 96 terms (2^-24 each, summed: below 1e-6), the
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


def plain_window_layer(layer, p, x, positions, mask):
    """PyGaussianAttention with a window in float64: every query's own keys, by the definition."""
    H, K, D = layer.heads, layer.kv_heads, layer.head_dim
    n = x.shape[1]
    q = (x @ p["to_q.weight"].T).unflatten(-1, (H, D))
    kv = (x @ p["to_kv.weight"].T).unflatten(-1, (2 * K, D))
    k, v = kv[:, :, :K], kv[:, :, K:]
    F = layer.freqs.double().cpu()

    def turn(t, w):
        t = t * (t.square().mean(-1, keepdim=True) + layer.eps).rsqrt() * w
        a = (positions @ F)[:, :, None]
        m = 2 * F.shape[1]
        z = torch.view_as_complex(t[..., :m].unflatten(-1, (-1, 2)).contiguous()) * torch.polar(torch.ones_like(a), a)
        return torch.cat([torch.view_as_real(z).flatten(-2), t[..., m:]], -1)

    q, k = turn(q, p["q_weight"]), turn(k, p["k_weight"]).repeat_interleave(H // K, 2)
    v = v.repeat_interleave(H // K, 2)
    i, j = torch.arange(n)[:, None], torch.arange(n)[None]
    left, right = layer.window
    see = ((j <= i + right) & ((j >= i - left) | (j < layer.sinks)))[None] & mask[:, None]
    s = torch.matmul(q.transpose(1, 2), k.permute(0, 2, 3, 1)) * D ** -0.5
    none = ~see.any(-1)[:, None, :, None]
    s = s.masked_fill(~see[:, None] & ~none, -torch.inf).softmax(-1).masked_fill(none, 0.0)
    return torch.matmul(s, v.transpose(1, 2)).transpose(1, 2).flatten(2) @ p["to_out.weight"].T


def test_window_layer():
    """A layer with a window and sinks, a masked batch, an empty scene: output and all gradients."""
    from CudaGaussianVoxelizer import PyGaussianAttention
    torch.manual_seed(4)
    layer = PyGaussianAttention(96, 6, 2, wavelengths=(0.8, 40.0), window=(20, 9), sinks=3)
    B, N = 3, 150
    g = torch.Generator().manual_seed(6)
    ins = {"x": torch.randn(B, N, 96, generator=g), "positions": torch.rand(B, N, 3, generator=g) * 20 - 10}
    mask = torch.rand(B, N, generator=g) < 0.8
    mask[1] = False
    go = torch.randn(B, N, 96, generator=g)
    dev = {n: t.cuda().requires_grad_() for n, t in ins.items()}
    y = layer(dev["x"], dev["positions"], mask.cuda())
    y.backward(go.cuda())
    ref = {n: t.double().requires_grad_() for n, t in ins.items()}
    p = {n: t.detach().double().cpu().requires_grad_() for n, t in layer.named_parameters()}
    want = plain_window_layer(layer, p, ref["x"], ref["positions"], mask)
    want.backward(go.double())
    assert rel(y, want) < 3e-5
    for n, t in ins.items():
        assert rel(dev[n].grad, ref[n].grad) < 3e-5, n
    for n, t in layer.named_parameters():
        assert rel(t.grad, p[n].grad) < 3e-5, n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_stack_of_layers(dtype):
    """What a training step of a deep stack runs, one after another on one stream: norms with the residual sum, layers with windows,
    the gradients' norm and clipping.  Against the same stack in float64 from the same weights: the norms and windows by their
    definitions, the clipping by its formula.  float32: five operators' bounds of 3e-5 and their propagation through two layers, below
    3e-4.  bfloat16: every one of about ten roundings of a layer's values is at most 2^-8 and they add up independently: below 5e-2
    (gradients taken together: a weight of a norm's sum may cancel to what is below its terms' roundings)."""
    from CudaGaussianVoxelizer import PyGaussianAttention, PyLayerNorm, clip_grad_norm_
    torch.manual_seed(9)
    C, N, B, tol = 64, 200, 2, 3e-4 if dtype == torch.float32 else 5e-2
    layers = [(PyLayerNorm(C, dtype=dtype), PyGaussianAttention(C, 4, 2, window=(30, 30), sinks=4, dtype=dtype)) for _ in range(2)]
    last = PyLayerNorm(C, dtype=dtype)
    g = torch.Generator().manual_seed(3)
    x, pos = torch.randn(B, N, C, generator=g).to(dtype), torch.rand(B, N, 3, generator=g) * 20 - 10
    mask = torch.rand(B, N, generator=g) < 0.9
    go = torch.randn(B, N, C, generator=g).to(dtype)

    def run():
        branch, total = None, x.cuda()
        for norm, attention in layers:
            if branch is None:
                y = norm(total)
            else:
                y, total = norm(branch, residual=total)
            branch = attention(y, pos.cuda(), mask.cuda())
        return last(branch, residual=total)[0]

    params = [p for norm, attention in layers for p in (*norm.parameters(), *attention.parameters())] + list(last.parameters())
    y = run()
    y.backward(go.cuda())
    before = [p.grad.clone() for p in params]
    total_norm = clip_grad_norm_(params, 0.5)

    def ln(t, w, b):
        d = t - t.mean(-1, keepdim=True)
        return d / (d.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w + b

    ref = [{n: p.detach().double().cpu().requires_grad_() for n, p in m.named_parameters()}
           for m in [m for pair in layers for m in pair] + [last]]
    t = x.double()
    for i, (norm, attention) in enumerate(layers):
        t = t + plain_window_layer(attention, ref[2 * i + 1], ln(t, ref[2 * i]["weight"], ref[2 * i]["bias"]), pos.double(), mask)
    want = ln(t, ref[-1]["weight"], ref[-1]["bias"])
    want.backward(go.double())
    assert rel(y, want) < tol
    grads = [p.grad for r in ref for p in r.values()]
    if dtype == torch.float32:
        for a, b in zip(before, grads):
            assert rel(a, b) < tol
    assert rel(torch.cat([a.flatten().float() for a in before]), torch.cat([b.flatten() for b in grads])) < tol
    norm64 = torch.stack([b.double().square().sum() for b in before]).sum().sqrt()
    assert abs(float(total_norm) - float(norm64)) <= 1e-6 * float(norm64)
    for p, b in zip(params, before):
        assert rel(p.grad, b.double() * min(1.0, 0.5 / (float(norm64) + 1e-6))) < (1e-6 if p.dtype == torch.float32 else 4e-3)
    # again, the same bits
    for p in params:
        p.grad = None
    run().backward(go.cuda())
    assert all(torch.equal(p.grad, b) for p, b in zip(params, before))


@pytest.mark.parametrize("bf16", [False, True])
def test_example_trains_with_a_window_and_clipping(bf16):
    """It runs, its losses are finite and gradients reach what is trained; how far a loss falls is not looked at."""
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import gaussian_features_step as example
    finally:
        sys.path.pop(0)
    losses = example.train(gaussians=600, scenes=2, channels=64, steps=3, bf16=bf16, window=100, clip=0.01)
    assert len(losses) == 3 and all(l == l and abs(l) < 1e3 for l in losses)
    assert losses[0] != losses[1]


def test_captured_backward_beside_an_eager_graph():
    """A step is captured while an eager graph of the same leaves lives: each has its own results."""
    from CudaGaussianVoxelizer import gaussian_attention, layer_norm
    torch.manual_seed(2)
    x = torch.randn(1, 300, 64, device="cuda")
    w = torch.ones(64, device="cuda")

    def step(x, w):
        y = layer_norm(x, w).unflatten(-1, (2, 32))
        return gaussian_attention(y, y, y, window=(40, 40), sinks=2).square().sum()

    leaves = [t.clone().requires_grad_() for t in (x, w)]
    eager = step(*leaves)                      # lives on, unused so far
    held = [t.clone().requires_grad_() for t in (x, w)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(step(*held), held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = torch.autograd.grad(step(*held), held)
    want = torch.autograd.grad(eager, leaves)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, want):
            assert torch.equal(a, b)
