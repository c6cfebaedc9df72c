"""Which tensors clip_grad_norm_ takes for gradients, without a GPU: in place of the kernels stands their formula in 64 bits, so that what
the call passes on, and what it writes, is seen."""
import math

import pytest
import torch


@pytest.fixture
def passed(monkeypatch):
    """The lists of gradients and of outputs (None: in place) of the calls that reach the library."""
    from CudaGaussianVoxelizer import _C
    calls = []

    def formula(grads, max_norm, outs=None):
        calls.append((list(grads), None if outs is None else list(outs)))
        norm = math.sqrt(sum(float(g.detach().double().square().sum()) for g in grads))
        for g, o in zip(grads, grads if outs is None else outs):
            o.copy_(g.double() * min(1.0, max_norm / (norm + 1e-6)))
        return torch.tensor(norm)

    monkeypatch.setattr(_C, "clip_gradients", formula)
    return calls


def same(tensors, others):
    return len(tensors) == len(others) and all(a is b for a, b in zip(tensors, others))


def stack(freeze):
    """Three layers after a backward, those of `freeze` frozen before it."""
    torch.manual_seed(3)
    layers = torch.nn.Sequential(torch.nn.Linear(6, 5), torch.nn.Linear(5, 4), torch.nn.Linear(4, 3))
    for i in freeze:
        layers[i].requires_grad_(False)
    layers(torch.randn(7, 6)).square().sum().backward()
    return layers


@pytest.mark.parametrize("freeze", [(0,), (1,), (0, 2), (0, 1)])
def test_frozen_parameters_are_skipped(passed, freeze):
    """Their values neither count nor change; the norm and the others' gradients are those of torch's function."""
    from CudaGaussianVoxelizer import clip_grad_norm_
    layers, other = stack(freeze), stack(freeze)
    before = [p.detach().clone() for p in layers.parameters()]
    norm = clip_grad_norm_(layers.parameters(), 0.01)
    want = torch.nn.utils.clip_grad_norm_(other.parameters(), 0.01)
    assert all(torch.equal(p, b) for p, b in zip(layers.parameters(), before))
    assert same(passed[0][0], [p.grad for p in layers.parameters() if p.requires_grad])
    torch.testing.assert_close(norm, want, rtol=1e-6, atol=0)
    for p, q in zip(layers.parameters(), other.parameters()):
        assert (p.grad is None) == (q.grad is None)
        if p.grad is not None:
            torch.testing.assert_close(p.grad, q.grad, rtol=1e-6, atol=0)


def test_frozen_parameters_leave_their_outputs(passed):
    from CudaGaussianVoxelizer import clip_grad_norm_
    layers = stack((1,))
    params = list(layers.parameters())
    out = [torch.full_like(p, 7.0, requires_grad=False) for p in params]
    clip_grad_norm_(params, 0.01, out=out)
    kept = [i for i, p in enumerate(params) if p.requires_grad]
    assert same(passed[0][0], [params[i].grad for i in kept]) and same(passed[0][1], [out[i] for i in kept])
    assert all(bool((o == 7.0).all()) == (i not in kept) for i, o in enumerate(out))


def test_parameters_frozen_after_a_backward_stand_for_their_gradients(passed):
    """What is left in .grad is clipped, as torch's function does, be the parameter a torch.nn.Parameter or a plain leaf."""
    from CudaGaussianVoxelizer import clip_grad_norm_
    layers = stack(())
    leaf = torch.ones(4, requires_grad=True)
    (3.0 * leaf).sum().backward()
    params = list(layers.parameters()) + [leaf]
    before = [p.detach().clone() for p in params]
    for p in params[::2]:
        p.requires_grad_(False)
    clip_grad_norm_(params, 0.01)
    assert same(passed[0][0], [p.grad for p in params])
    assert all(torch.equal(p, b) for p, b in zip(params, before))


def test_nothing_but_frozen_parameters(passed):
    from CudaGaussianVoxelizer import clip_grad_norm_
    layer = torch.nn.Linear(3, 3).requires_grad_(False)
    before = [p.clone() for p in layer.parameters()]
    norm = clip_grad_norm_(layer.parameters(), 0.1)
    assert not passed and float(norm) == 0.0 and norm.shape == ()
    assert all(torch.equal(p, b) for p, b in zip(layer.parameters(), before))


def test_gradients_themselves(passed):
    from CudaGaussianVoxelizer import clip_grad_norm_
    grads = [torch.randn(5), torch.randn(2, 3)]
    clip_grad_norm_(iter(grads), 0.1)
    clip_grad_norm_(grads[0], 0.1)
    assert same(passed[0][0], grads) and same(passed[1][0], grads[:1])


def test_gradients_with_a_graph_are_refused(passed):
    """A gradient made with create_graph requires grad and is no parameter: it was taken for one without a gradient, and the norm was 0."""
    from CudaGaussianVoxelizer import clip_grad_norm_
    leaf = torch.ones(3, requires_grad=True)
    grad, = torch.autograd.grad(leaf.pow(3).sum(), leaf, create_graph=True)
    before = grad.detach().clone()
    for tensors in ([grad], [torch.ones(2), grad], grad):
        with pytest.raises(RuntimeError, match="detached"):
            clip_grad_norm_(tensors, 1.0)
    assert not passed and torch.equal(grad, before)
    clip_grad_norm_([grad.detach()], 1.0)
    assert torch.equal(passed[0][0][0], grad)


def test_parameters_whose_gradients_have_a_graph(passed):
    """A parameter's .grad is clipped, made with create_graph or not; so is what a graph's inner tensor retains."""
    from CudaGaussianVoxelizer import clip_grad_norm_
    leaf = torch.nn.Parameter(torch.ones(3))
    inner = 2.0 * leaf
    inner.retain_grad()
    inner.pow(3).sum().backward(create_graph=True)
    assert leaf.grad.requires_grad
    clip_grad_norm_([leaf, inner], 1e9)
    assert same(passed[0][0], [leaf.grad, inner.grad])
