"""The windowed attention in float32 over long windows, on either side of the rule by which its forward splits rows into planes or packs them
before (tests/test_capi_window_plan.py), against the 64-bit statement of tests/test_gpu_window_attention.py with its tolerances."""
import pytest
import torch

from tests.test_gpu_window_attention import check, make, random_mask

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("keep", [1.0, 0.7], ids=["all", "masked"])
@pytest.mark.parametrize("B,nq,nk,hq,hk,D,window,sinks", [
    (1, 1, 6000, 4, 4, 64, (4096, 0), 4), (2, 1, 5000, 4, 1, 128, (None, 0), 0), (1, 1, 4500, 2, 2, 96, (4096, 0), 70),
    (1, 200, 5000, 2, 1, 96, (3500, 0), 3), (1, 130, 2500, 2, 2, 32, (2000, 100), 0), (2, 1500, 1500, 2, 2, 64, (700, 700), 5),
    (1, 2500, 2500, 1, 1, 128, (1100, 1100), 0), (1, 2500, 2500, 4, 1, 64, (600, 600), 2), (1, 2000, 2000, 2, 2, 72, (300, 300), 9),
    (1, 2000, 2000, 2, 2, 72, (500, 500), 0), (1, 2048, 2048, 1, 1, 16, (None, 0), 0)])
def test_long_windows(B, nq, nk, hq, hk, D, window, sinks, keep):
    mask = None if keep == 1.0 else random_mask(B, nk, keep, nq + D)
    check(*make(B, nq, nk, hq, hk, D, torch.float32, nk + D), window, sinks, mask)
