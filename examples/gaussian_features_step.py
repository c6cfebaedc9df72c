"""Training steps of Gaussian features: an attention layer over the Gaussians of a batch of scenes makes their features, the
voxelizer splats them, and the feature cosine loss against a target grid trains the layer and the Gaussians' means.

    python examples/gaussian_features_step.py [--gaussians 2000] [--scenes 2] [--channels 64] [--steps 5] [--bf16]
                                              [--window 256] [--clip 35]

With --window the Gaussians are sorted along a space-filling curve, and each attends to that many before and behind it and to the
first ones.  The gradients' norm is clipped.  Synthetic scenes, random weights.  Prints the loss of every step.
"""
import argparse
import os
import sys

import torch
import torch.nn as nn

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "shelfgaussian-cudagaussianvoxelizer_amd"))

from CudaGaussianVoxelizer import (PyCudaFeatsCosineLoss, PyCudaGaussianVoxelizer, PyGaussianAttention,  # noqa: E402
                                   PyLayerNorm, clip_grad_norm_)

VOXEL = [0.4, 0.4, 0.4]
RANGE = [-10.0, -10.0, -1.0, 10.0, 10.0, 2.2]


SINKS = 4


def curve_order(means):
    """Order of each scene's Gaussians (B, N) along a Z-order curve: 10 bits of each coordinate, interleaved."""
    lo, hi = torch.tensor(RANGE[:3], device="cuda"), torch.tensor(RANGE[3:], device="cuda")
    cell = ((means - lo) / (hi - lo) * 1024).long().clamp(0, 1023)
    code = torch.zeros_like(cell[..., 0])
    for bit in range(10):
        for axis in range(3):
            code |= (cell[..., axis] >> bit & 1) << (3 * bit + axis)
    return code.argsort(-1)


class GaussianFeatures(nn.Module):
    """Residual attention over the Gaussians of each scene, then a projection to the splatted channels."""

    def __init__(self, channels, heads, dtype, window=None):
        super().__init__()
        near = {} if window is None else dict(window=(window, window), sinks=SINKS)
        self.attention = PyGaussianAttention(channels, heads, wavelengths=(0.8, 40.0), dtype=dtype, **near)
        self.norm = PyLayerNorm(channels, dtype=dtype)
        self.head = nn.Linear(channels, channels, device="cuda", dtype=dtype)

    def forward(self, x, means, valid):
        x = x + self.attention(self.norm(x), means, key_mask=valid)
        return self.head(x)


def train(gaussians=2000, scenes=2, channels=64, steps=5, bf16=False, seed=0, window=None, clip=35.0):
    """The losses of `steps` steps."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    torch.manual_seed(seed)
    dtype = torch.bfloat16 if bf16 else torch.float32

    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    lo, hi = torch.tensor(RANGE[:3], device="cuda"), torch.tensor(RANGE[3:], device="cuda")
    means = lo + (hi - lo) * rand(scenes, gaussians, 3)
    if window is not None:
        means = means.gather(1, curve_order(means)[..., None].expand_as(means))
    means.requires_grad_()
    opacity = rand(scenes, gaussians)
    variance = 0.2 + rand(scenes, gaussians, 3)
    covariances = torch.diag_embed(variance).flatten(2)
    tokens = torch.randn(scenes, gaussians, channels, generator=g, device="cuda").to(dtype)
    # scenes of fewer Gaussians are padded: padding is not attended to, and splats nothing
    count = torch.linspace(0.6, 1.0, scenes, device="cuda") * gaussians
    valid = torch.arange(gaussians, device="cuda") < count[:, None]
    opacity = opacity * valid

    model = GaussianFeatures(channels, max(1, channels // 32), dtype, window)
    voxelizer = PyCudaGaussianVoxelizer(voxel_size=VOXEL, voxel_range=RANGE)
    cosine = PyCudaFeatsCosineLoss(voxel_size=VOXEL, voxel_range=RANGE)
    optimizer = torch.optim.Adam([{"params": model.parameters(), "lr": 1e-2}, {"params": [means], "lr": 1e-2}])

    target = label = seen = None
    losses = []
    for _ in range(steps):
        features = model(tokens, means, valid)
        density, grid, _ = voxelizer(means, opacity, covariances, features)
        if target is None:
            target = torch.randn(channels, generator=g, device="cuda").to(grid.dtype).expand(grid.shape[1:]).contiguous()
            label = torch.ones(grid.shape[1:4], device="cuda")
            seen = density.detach() > 1e-3
        loss = sum(cosine(label, seen[b], grid[b], target)[0] for b in range(scenes)) / scenes
        optimizer.zero_grad()
        with torch.autograd.set_multithreading_enabled(False):   # one GPU: no waiting for the engine's thread
            loss.backward()
        clip_grad_norm_([*model.parameters(), means], clip)
        optimizer.step()
        losses.append(float(loss.detach()))
    return losses


def main():
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--gaussians", type=int, default=2000)
    p.add_argument("--scenes", type=int, default=2)
    p.add_argument("--channels", type=int, default=64)
    p.add_argument("--steps", type=int, default=5)
    p.add_argument("--bf16", action="store_true")
    p.add_argument("--window", type=int)
    p.add_argument("--clip", type=float, default=35.0)
    for i, loss in enumerate(train(**vars(p.parse_args()))):
        print(f"step {i}: loss {loss:.5f}", flush=True)


if __name__ == "__main__":
    main()
