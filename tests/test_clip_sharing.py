"""Which tensors clip_grad_norm_ refuses for the memory they share, without a GPU: the look at strided tensors, which reach the library as
copies, against an enumeration of every byte; flat ones are the library's to refuse (tests/test_capi_training.py)."""
import itertools
import random

import pytest
import torch


def places(t):
    """Addresses of a tensor's elements, one after another."""
    at = [t.data_ptr()]
    for n, step in zip(t.shape, t.stride()):
        at = [a + step * t.element_size() * i for a in at for i in range(n)]
    return at


def bytes_of(t):
    return {a + e for a in places(t) for e in range(t.element_size())}


def random_view(rng, base):
    """Any view of the base's memory: up to three dimensions, steps of zero and sizes of one among them."""
    dtype = rng.choice([torch.float32, torch.bfloat16])
    flat = base.view(dtype)
    shape = [rng.randint(1, 5) for _ in range(rng.randint(0, 3))]
    stride = [rng.choice([0, 1, 1, 2, 3, 4, 5, 7, 12, 20]) for _ in shape]
    reach = sum(s * (n - 1) for s, n in zip(stride, shape))
    return torch.as_strided(flat, shape, stride, rng.randint(0, flat.numel() - 1 - reach))


@pytest.mark.parametrize("seed", range(8))
def test_against_every_byte(seed):
    from CudaGaussianVoxelizer import _C
    rng, base = random.Random(seed), torch.zeros(300)
    found = [0, 0, 0, 0]
    for _ in range(400):
        a, b = random_view(rng, base), random_view(rng, base)
        shared, twice = bool(bytes_of(a) & bytes_of(b)), len(set(places(a))) < a.numel()
        assert _C._share_memory(a, b) == _C._share_memory(b, a) == shared, (a.shape, a.stride(), b.shape, b.stride())
        assert _C._overlaps_itself(a) == twice, (a.shape, a.stride())
        found[shared] += 1
        found[2 + twice] += 1
    assert min(found) > 0


def test_what_cannot_be_told_counts_as_shared():
    """Steps without order in them, of which no sum is the target (the last one but one of all sums): the look ends, with the safe answer."""
    from CudaGaussianVoxelizer import _C
    rng = random.Random(1)
    steps = [(2 * rng.randint(10 ** 8, 2 * 10 ** 8), 9) for _ in range(20)]
    assert _C._reaches(sum(s * n for s, n in steps) // 4 * 2, steps)


def checked(grads, outs=None):
    from CudaGaussianVoxelizer import _C
    return _C._clip_checked(grads, grads if outs is None else outs, torch.device("cpu"))


def wide():
    return torch.arange(140.0 * 6).view(6, 140)


def test_refusals():
    w, square = wide(), torch.ones(8, 8)
    columns = w[:, ::2]
    for grads, outs in (([columns, columns], None), ([columns, w[:, ::2]], None), ([columns, w[:, 2:9]], None), ([columns, w], None),
                        ([columns, w[2]], None), ([columns, torch.ones(3), w.view(-1)[836:]], None), ([w[:3, ::3], w[2:, ::2]], None),
                        # an output on its gradient in another order, shifted, on another's gradient, twice, of another type
                        ([square], [square.t()]), ([w[:, 0:50:2]], [w[:, 2:52:2]]), ([w[:, :50], w[:, 50:100]], [w[:, 50:100], w[:, :50]]),
                        ([torch.ones(6, 70)] * 2, [columns, columns]), ([columns], [w.view(torch.bfloat16)[:, ::4]]),
                        # elements that share their place
                        ([torch.ones(4).expand(3, 4)], None), ([torch.ones(3, 4)], [torch.ones(4).expand(3, 4)]),
                        ([torch.ones(9).unfold(0, 3, 1)], None)):
        with pytest.raises(RuntimeError, match="share memory"):
            checked(grads, outs)
    assert torch.equal(w, wide()) and bool((square == 1).all())


def test_what_shares_nothing_passes():
    """Columns beside one another, whose spans cross, in place and as outputs; gradients that are read twice; views in place."""
    w, square = wide(), torch.ones(8, 8)
    parts = [w[:, i::4] for i in range(3)] + [w[:, 3:100:4], w[:, 103::4]]
    checked(parts)
    checked([p.clone() for p in parts], parts)
    checked([w[:, :40], w[:, 40:80], w[:, 80:]], [w[:, :40], w[:, 40:80], w[:, 80:]])
    checked([w[:, ::2], w[:, ::2]], [torch.empty(6, 70), torch.empty(6, 70)])
    checked([torch.ones(4).expand(3, 4)], [torch.empty(3, 4)])
    checked([square.t(), w[:, 1::2]])
    checked([w[2:3, 1:9]], [torch.as_strided(w, (1, 8), (7, 1), 2 * 140 + 1)])    # the same places: the step of one row does not count
    src, dst, back = checked([w[:, ::2], torch.empty(0, 3)[:, ::2], torch.tensor(3.0)])
    assert src[0].is_contiguous() and dst[0] is src[0] and back[0][1] is src[0]


def test_a_fused_projections_gradients():
    """Slices of fused gradients of many layers: the look at crossing spans ends at once."""
    fused = [torch.zeros(96, 3 * 64) for _ in range(24)]
    grads = list(itertools.chain.from_iterable(f.split(64, 1) for f in fused))
    src, dst, back = checked(grads)
    assert len(back) == len(grads) == 72
