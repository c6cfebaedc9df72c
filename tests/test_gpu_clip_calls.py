"""clip_grad_norm_ as training loops call it, on the GPU: models that are trained in part.

Tolerances.  This norm's squares are summed in 64 bits, torch's in float32: a sum of n squares by pairs is off by at most log2(n) 2^-24,
with the root half of that: below 1e-6 for the 2,000 elements here, and so is every product with the factor, rounded to 2^-24 more.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


def model(dtype):
    torch.manual_seed(5)
    layers = torch.nn.Sequential(torch.nn.Linear(40, 30), torch.nn.Linear(30, 20), torch.nn.Linear(20, 6)).to("cuda", dtype)
    layers[1].requires_grad_(False)
    layers[2].weight.requires_grad_(False)
    layers(torch.randn(9, 40, device="cuda", dtype=dtype)).square().sum().backward()
    return layers


@pytest.mark.parametrize("max_norm", [0.05, 1e6], ids=["clipped", "kept"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_a_partly_frozen_model(dtype, max_norm):
    """Frozen weights stay bit for bit and do not count; gradients and norm are torch's (bfloat16: of the same gradients in float32,
    rounded once); outputs of frozen parameters stay."""
    from CudaGaussianVoxelizer import clip_grad_norm_
    layers = model(dtype)
    params = list(layers.parameters())
    before = [p.detach().clone() for p in params]
    twins = [torch.nn.Parameter(p.detach().float()) for p in params]
    for t, p in zip(twins, params):
        t.grad = None if p.grad is None else p.grad.float().clone()
    want = torch.nn.utils.clip_grad_norm_(twins, max_norm)
    out = [torch.full(p.shape, 7.0, device="cuda") for p in params]
    for got in (clip_grad_norm_(params, max_norm, out=out), clip_grad_norm_(layers.parameters(), max_norm)):
        torch.testing.assert_close(got, want, rtol=1e-6, atol=0)
    assert sum(p.grad is None for p in params) == 3
    for p, b, t, o in zip(params, before, twins, out):
        assert torch.equal(p, b)
        if p.grad is None:
            assert bool((o == 7.0).all())
        else:
            torch.testing.assert_close(o, t.grad, rtol=2e-6, atol=0)
            torch.testing.assert_close(p.grad.float(), t.grad, rtol=2e-6 + (2.0 ** -8 if dtype == torch.bfloat16 else 0.0), atol=0)


def test_strided_tensors_that_share_memory_are_refused():
    """Tensors that go through copies: refused before anything is written, as flat ones are."""
    from CudaGaussianVoxelizer import clip_grad_norm_
    w, square = torch.ones(6, 140, device="cuda"), torch.ones(8, 8, device="cuda")
    for tensors, out in (([w[:, ::2], w[:, ::2]], None), ([square], [square.t()]), ([w[:, :50], w[:, 50:100]], [w[:, 50:100], w[:, :50]]),
                         ([torch.ones(4, device="cuda").expand(3, 4)], None)):
        with pytest.raises(RuntimeError, match="share memory"):
            clip_grad_norm_(tensors, 0.1, out=out)
    assert bool((w == 1).all()) and bool((square == 1).all())


def test_columns_beside_one_another():
    """Slices of a fused gradient, whose spans of memory cross but share no element, are clipped in place."""
    from CudaGaussianVoxelizer import clip_grad_norm_
    fused = torch.randn(300, 96, generator=torch.Generator().manual_seed(2)).cuda()
    before = fused.double()
    norm = clip_grad_norm_([fused[:, :32], fused[:, 32:64], fused[:, 64:]], 0.5)
    want = float(before.square().sum().sqrt())
    assert abs(float(norm) - want) <= 2.0 ** -23 * want
    assert bool(((fused.double() - before * 0.5 / (want + 1e-6)).abs() <= 2.0 ** -23 * before.abs()).all())


@pytest.mark.parametrize("size,count", [(3e38, 1), (1.5e38, 5), (1e38, 11)])
def test_norms_just_below_float32s_largest(size, count):
    """Values whose squares float32 does not hold and whose norm it does, 2 % to 12 % below its largest: finite, and off by its rounding."""
    from CudaGaussianVoxelizer import clip_grad_norm_
    big = torch.zeros(5000, device="cuda")
    big[::400][:count] = size
    small = torch.full((300,), 1.0, device="cuda")
    before = [big.double(), small.double()]
    want = float(sum(b.square().sum() for b in before).sqrt())
    assert 0.85 * torch.finfo(torch.float32).max < want < torch.finfo(torch.float32).max
    norm = float(clip_grad_norm_([big, small], 1e30))
    assert abs(norm - want) <= 2.0 ** -23 * want
    for g, b in zip((big, small), before):
        exact = b * 1e30 / want
        assert bool(((g.double() - exact).abs() <= 2.0 ** -23 * exact + 2.0 ** -126).all())
