"""How many bits the windowed attention's gradients keep, against the 64-bit statement of tests/test_gpu_window_attention.py."""
import pytest
import torch

from tests.test_gpu_window_attention import make, plain, random_mask, rel, run, say, visible

pytestmark = pytest.mark.gpu


def most_in_one(q, k, window, sinks, mask):
    """The largest sum of squared probabilities of a row that sees a key."""
    worst = 0.0
    group = q.shape[2] // k.shape[2]
    for b in range(q.shape[0]):
        see = visible(q.shape[1], k.shape[1], window, sinks)
        if mask is not None:
            see = see & mask[b][None]
        rows = see.any(1)
        for h in range(q.shape[2]):
            s = q.shape[3] ** -0.5 * q[b, rows, h].double() @ k[b, :, h // group].double().T
            worst = max(worst, float(torch.softmax(s.masked_fill(~see[rows], -torch.inf), -1).square().sum(-1).max()))
    return worst


@pytest.mark.parametrize("nq,nk,hq,hk,D,window,sinks,keep", [
    (300, 300, 4, 2, 32, (150, 150), 0, 1.0), (400, 400, 2, 2, 40, (100, 120), 8, 1.0), (500, 500, 4, 4, 64, (200, 200), 16, 1.0),
    (300, 300, 2, 1, 64, (None, None), 0, 1.0), (300, 500, 4, 2, 72, (150, 100), 8, 0.8), (400, 400, 2, 2, 96, (150, 150), 4, 1.0),
    (400, 400, 2, 2, 128, (150, 150), 33, 1.0), (1500, 1500, 2, 2, 64, (500, 500), 16, 1.0), (64, 3000, 1, 1, 64, (2500, 2500), 0, 1.0),
    (500, 2500, 2, 2, 64, (1500, 0), 8, 0.5)])
def test_the_values_gradients_are_rounded_once(nq, nk, hq, hk, D, window, sinks, keep):
    """Where a query sees few keys (1,024 at most), where there are few rows (64) and where a mask may leave few, P goes into dV with twice
    bfloat16's bits, 2^-16 off, as in the attention over all keys.  What is left beside the result's own rounding, r of its norm, is the
    forward's: lse holds the sum of a row's probabilities as they were rounded, which is r sqrt(sum P^2) off, independently for each
    row.  The two together: r sqrt(1 + sum P^2), with the largest such sum, and 2^-14 for the planes and float32 sums.  (P in one plane
    would be r sqrt(2) off.)"""
    q, k, v, g = make(2, nq, nk, hq, hk, D, torch.bfloat16, nq + D)
    mask = None if keep == 1.0 else random_mask(2, nk, keep, D)
    share = most_in_one(q, k, window, sinks, mask)
    assert share < 0.4
    want = plain(q, k, v, window, sinks, mask, g)[3]
    r = rel(want.bfloat16(), want)
    got = rel(run(q, k, v, g, window, sinks, mask)[3], want)
    say(f"[window dV] {nq} {nk} {hq} {D} {window} {sinks}: rounding {r:.3e}, dV {got:.3e}, share {share:.2f}")
    assert got <= r * (1.0 + share) ** 0.5 + 2.0 ** -14
