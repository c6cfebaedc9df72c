"""C ABI of the windowed attention, the layer norm and the gradients' clipping: workspace queries and argument checks, and the checks
of the Python side that need no GPU.  Nothing here launches a kernel."""
import ctypes

import pytest
import torch

ONE = ctypes.c_void_p(16)
S3 = (ctypes.c_longlong * 3)(64, 64, 8)
S2 = (ctypes.c_longlong * 2)(64, 8)
F32, BF16 = 0, 1


def _lib():
    from CudaGaussianVoxelizer import _lib
    return _lib.load()


# ---- attention within a window ----

def window(lib, B=1, nq=4, nk=4, hq=2, hk=2, D=8, q=ONE, k=ONE, v=ONE, dt=BF16, mask=None, left=2, right=2, sinks=1, scale=1.0, out=ONE,
           ws=ONE, nws=1 << 30, qs=S3):
    return lib.g2v_window_attention_forward(B, nq, nk, hq, hk, D, q, qs, k, S3, v, S3, dt, mask, left, right, sinks, scale, out, None,
                                            None, ws, nws, None)


@pytest.mark.parametrize("bad,code,word", [
    (dict(B=-1), 1, b"negative"), (dict(D=0), 1, b"head_dim"), (dict(D=129), 1, b"head_dim"), (dict(hq=3), 1, b"multiple"),
    (dict(dt=2), 1, b"dtype"), (dict(scale=0.0), 1, b"scale"), (dict(scale=float("nan")), 1, b"scale"), (dict(left=-2), 1, b"left"),
    (dict(right=-2), 1, b"right"), (dict(sinks=-1), 1, b"sinks"), (dict(q=None), 1, b"null"), (dict(k=None), 1, b"null"),
    (dict(v=None), 1, b"null"), (dict(out=None), 1, b"null"), (dict(qs=None), 1, b"null"), (dict(ws=None), 1, b"workspace"),
    (dict(nws=1), 1, b"workspace"), (dict(B=1 << 20), 3, b"limit"), (dict(nk=1 << 25), 3, b"limit"),
])
def test_window_arguments(bad, code, word):
    lib = _lib()
    assert window(lib, **bad) == code and word in lib.g2v_last_error()


def test_window_without_rows_does_nothing():
    lib = _lib()
    assert window(lib, B=0, q=None, k=None, v=None, out=None, ws=None, qs=None) == 0
    assert window(lib, nq=0, q=None, out=None, ws=None, qs=None) == 0


def test_window_backward_arguments():
    lib = _lib()
    need = lib.g2v_window_attention_backward_workspace(1, 4, 4, 2, 2, 8, F32, 2, 2, 1, 0, 0)

    def call(lse=ONE, out=ONE, g=ONE, dk=ONE, dv=ONE, ws=ONE, nws=need, scale=1.0, left=2):
        return lib.g2v_window_attention_backward(1, 4, 4, 2, 2, 8, ONE, S3, ONE, S3, ONE, S3, F32, None, left, 2, 1, scale, out, None,
                                                 lse, g, S3, ONE, dk, dv, ws, nws, None)

    for bad, word in ((dict(lse=None), b"null"), (dict(out=None), b"null"), (dict(g=None), b"null"), (dict(dk=None), b"together"),
                      (dict(ws=None), b"workspace"), (dict(nws=need - 1), b"workspace"), (dict(scale=0.0), b"scale"),
                      (dict(left=-3), b"left")):
        assert call(**bad) == 1 and word in lib.g2v_last_error(), bad


@pytest.mark.parametrize("query", ["g2v_window_attention_forward_workspace", "g2v_window_attention_backward_workspace"])
def test_window_workspaces(query):
    """Refused sizes need nothing, packing only adds (a mask goes with more planes and so another plan), and no extreme of a window's bounds passes 32 bits anywhere."""
    q = getattr(_lib(), query)
    assert q(1, 4, 4, 2, 2, 129, BF16, 1, 1, 0, 1, 0) == 0 and q(1, 4, 4, 2, 2, 64, BF16, -2, 1, 0, 1, 0) == 0
    for n in (1, 300, 5000, 200000):
        for left, right, sinks in ((0, 0, 0), (256, 256, 16), (-1, -1, 4), (2 ** 31 - 1, 0, 2 ** 31 - 1)):
            base = q(1, n, n, 8, 4, 64, BF16, left, right, sinks, 1, 0)
            assert 0 < base < 1 << 40 and 0 < q(1, n, n, 8, 4, 64, BF16, left, right, sinks, 1, 1) < 1 << 40
            assert base < q(1, n, n, 8, 4, 64, BF16, left, right, sinks, 0, 0) and 0 < q(1, n, n, 8, 4, 64, F32, left, right, sinks, 1, 0)
    for B, nq, nk in ((0, 5, 5), (2, 0, 500), (2, 500, 0), (0, 0, 0), (2, 0, 0)):     # nothing to do, with sinks too
        for sinks in (0, 3):
            assert q(B, nq, nk, 8, 4, 64, F32, 2, 0, sinks, 0, 1) > 0 and q(B, nq, nk, 8, 4, 64, BF16, 2, 0, sinks, 1, 0) > 0
    # a single query of a long stream needs room for its window, not for the stream
    lib = _lib()
    assert lib.g2v_window_attention_forward_workspace(1, 1, 200000, 8, 8, 64, F32, 512, 0, 4, 0, 1) < 1 << 23


def test_window_python_refusals():
    from CudaGaussianVoxelizer import PyGaussianAttention, _C, gaussian_attention
    for w in (5, (1, 2, 3), (-1, 2), (1.5, 2), (True, 2), "ab", (None, -1)):
        with pytest.raises(RuntimeError):
            _C._window(w, 0)
    for s in (-1, 1.0, None, True):
        with pytest.raises(RuntimeError):
            _C._window((1, 1), s)
    assert _C._window((None, 0), 3) == (-1, 0, 3) and _C._window([1 << 60, None], 1 << 60) == (1 << 30, -1, 1 << 30)
    t = torch.randn(1, 4, 2, 8)
    with pytest.raises(RuntimeError):
        gaussian_attention(t, t, t, window=(1, 1))
    with pytest.raises(RuntimeError):
        gaussian_attention(t, t, t, sinks=1)
    with pytest.raises(RuntimeError):
        PyGaussianAttention(64, 2, sinks=1, device="cpu")


# ---- layer norm ----

def norm(lib, B=1, n=4, C=8, x=ONE, xs=S2, res=None, rs=S2, dt=F32, w=ONE, b=ONE, wdt=F32, eps=1e-5, y=ONE, total=None):
    return lib.g2v_layer_norm_forward(B, n, C, x, xs, res, rs, dt, w, b, wdt, eps, y, total, None, None)


@pytest.mark.parametrize("bad,word", [
    (dict(B=-1), b"negative"), (dict(n=-1), b"negative"), (dict(C=0), b"channels"), (dict(C=8193), b"channels"), (dict(dt=2), b"dtype"),
    (dict(wdt=3), b"weight_dtype"), (dict(eps=-1.0), b"eps"), (dict(eps=float("nan")), b"eps"), (dict(x=None), b"null"),
    (dict(xs=None), b"null"), (dict(y=None), b"null"), (dict(res=ONE), b"sum"), (dict(res=ONE, rs=None, total=ONE), b"residual"),
])
def test_norm_arguments(bad, word):
    lib = _lib()
    assert norm(lib, **bad) == 1 and word in lib.g2v_last_error()


def test_norm_without_rows_does_nothing():
    lib = _lib()
    assert norm(lib, n=0, x=None, xs=None, y=None) == 0 and norm(lib, B=0, x=None, xs=None, y=None) == 0


def test_norm_backward_arguments():
    lib = _lib()
    need = lib.g2v_layer_norm_backward_workspace(1, 4, 8, F32)
    assert need > 0 and lib.g2v_layer_norm_backward_workspace(1, 4, 8193, F32) == 0

    def call(x=ONE, stats=ONE, gy=ONE, gs=None, gss=None, dx=ONE, ws=ONE, nws=need, wdt=F32):
        return lib.g2v_layer_norm_backward(1, 4, 8, x, S2, F32, ONE, wdt, stats, gy, S2, gs, gss, dx, ONE, ONE, ws, nws, None)

    for bad, word in ((dict(x=None), b"null"), (dict(stats=None), b"null"), (dict(gy=None), b"null"), (dict(dx=None), b"null"),
                      (dict(gs=ONE), b"grad_sum"), (dict(ws=None), b"workspace"), (dict(nws=need - 1), b"workspace"),
                      (dict(wdt=7), b"weight_dtype")):
        assert call(**bad) == 1 and word in lib.g2v_last_error(), bad


def test_norm_python_refusals():
    from CudaGaussianVoxelizer import layer_norm
    for bad in (torch.randn(3, 4), [1.0], None):
        with pytest.raises(RuntimeError):
            layer_norm(bad)


# ---- clipping ----

def clip(lib, grads=(4096, 8192), gd=(F32, F32), outs=None, od=None, numels=(10, 20), max_norm=1.0, norm=ONE, ws=ONE, nws=1 << 20, count=None):
    n = len(grads)
    P, I, L = ctypes.c_void_p * n, ctypes.c_int * n, ctypes.c_longlong * n
    outs, od = grads if outs is None else outs, gd if od is None else od
    return lib.g2v_clip_gradients(n if count is None else count, P(*grads), I(*gd), P(*outs), I(*od), L(*numels), max_norm, norm, ws, nws,
                                  None)


@pytest.mark.parametrize("bad,word", [
    (dict(count=-1), b"negative"), (dict(max_norm=-1.0), b"max_norm"), (dict(max_norm=float("nan")), b"max_norm"), (dict(norm=None), b"norm"),
    (dict(numels=(10, -1)), b"elements"), (dict(numels=(10, 1 << 41)), b"elements"), (dict(gd=(F32, 2)), b"dtype"),
    (dict(od=(5, F32)), b"dtype"), (dict(grads=(4096, 0)), b"null"), (dict(outs=(4096, 0)), b"null"), (dict(ws=None), b"workspace"),
    (dict(nws=8), b"workspace"),
    # memory that is written and shared: one tensor twice, overlapping ones, an output on another's gradient, in place as another type
    (dict(grads=(4096, 4096)), b"share"), (dict(grads=(4096, 4132)), b"share"), (dict(outs=(8192, 4096)), b"share"),
    (dict(outs=(16384, 16384)), b"share"), (dict(od=(BF16, F32)), b"share"), (dict(outs=(4100, 16384)), b"share"),
    (dict(grads=(4096, 4096), outs=(4096, 16384)), b"share"),
])
def test_clip_arguments(bad, word):
    lib = _lib()
    assert clip(lib, **bad) == 1 and word in lib.g2v_last_error()


def test_clip_workspaces():
    q = _lib().g2v_clip_gradients_workspace
    assert q(-1) == 0 and 0 < q(0) <= q(120) < q(121) < q(2000)


def test_clip_python_refusals():
    from CudaGaussianVoxelizer import clip_grad_norm_
    t = torch.ones(4)
    for tensors, kw in (([t], {}), (t, {}), ([t, 1.0], {}), ([t], dict(max_norm=-1.0)), ([t], dict(out=[t, t])), ([t], dict(out=[None]))):
        with pytest.raises(RuntimeError):
            clip_grad_norm_(tensors, **{"max_norm": 1.0, **kw})
