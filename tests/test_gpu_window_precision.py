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


def terms(q, k, v, g, window, sinks, mask):
    """float64: for dQ and dK, sums of P (A + sum P A) |k| and of |dS| |k| (dK: |q|) with A = sum_d |dO| |v|, what P (dP - delta) is made of
    before it cancels; and the largest sum of a score's absolute products, in the exponent's base of 2."""
    scale = q.shape[3] ** -0.5
    q, k, v, g = (t.double() for t in (q, k, v, g))
    before = [torch.zeros_like(q), torch.zeros_like(k)]
    after = [torch.zeros_like(q), torch.zeros_like(k)]
    most = 0.0
    for b in range(q.shape[0]):
        see = visible(q.shape[1], k.shape[1], window, sinks)
        if mask is not None:
            see = see & mask[b][None]
        none = ~see.any(1, keepdim=True)
        for h in range(q.shape[2]):
            Q, K, V, G = q[b, :, h], k[b, :, h], v[b, :, h], g[b, :, h]
            p = torch.softmax((scale * Q @ K.T).masked_fill(~see & ~none, -torch.inf), -1).masked_fill(none, 0.0)
            dp, a = G @ V.T, G.abs() @ V.abs().T
            ds = scale * p * (dp - (p * dp).sum(-1, keepdim=True)).abs()
            t = scale * p * (a + (p * a).sum(-1, keepdim=True))
            before[0][b, :, h], before[1][b, :, h] = t @ K.abs(), t.T @ Q.abs()
            after[0][b, :, h], after[1][b, :, h] = ds @ K.abs(), ds.T @ Q.abs()
            most = max(most, float((scale * 1.4427 * Q.abs() @ K.abs().T)[see].max()))
    return before, after, most


@pytest.mark.parametrize("n,D,window,sinks,keep,size", [
    (200, 64, (1, 1), 0, 1.0, 4.0), (200, 64, (3, 0), 1, 1.0, 4.0), (300, 32, (2, 2), 0, 0.6, 4.0), (130, 128, (0, 4), 2, 1.0, 4.0),
    (200, 40, (8, 8), 0, 0.8, 4.0), (5, 64, (1, 1), 0, 1.0, 6.0), (4, 64, (1, 0), 0, 1.0, 8.0), (6, 128, (1, 1), 1, 1.0, 7.0)])
def test_float32_where_gradients_cancel(n, D, window, sinks, keep, size):
    """Short windows of scores in the tens: one key has nearly all of a row's probability, and dS = P (dP - delta) is what is left of terms
    that are much larger.  float32's bits are those of the terms.  dP and delta are sums of at most 128 products in at most 64 steps one after
    another (six products of planes for every 16 channels; delta 8 values of every 16), each 2^-24 off; the products with k and q and
    their sums take as many again: 128 x 2^-24 of the terms.  P is off by its exponent's error, at most 2 x 48 x 2^-24 of the score's absolute
    products (the score's and lse's), and puts that on what is left."""
    q, k, v, g = make(1, n, n, 2, 2, D, torch.float32, n + D, size=size)
    mask = None if keep == 1.0 else random_mask(1, n, keep, D)
    got, want = run(q, k, v, g, window, sinks, mask), plain(q, k, v, window, sinks, mask, g)
    before, after, most = terms(q, k, v, g, window, sinks, mask)
    for name, x, y, b, a in zip(("dQ", "dK"), got[1:3], want[1:3], before, after):
        off = (x.double().cpu() - y).abs()
        say(f"[window cancel] {n} {D} {window} {name}: {rel(x, y):.1e} of its norm, {float(off.norm() / b.norm()):.1e} of the terms'")
        assert bool((off <= 2.0 ** -24 * (128 * b + 96 * most * a) + 1e-30).all())
