"""C ABI of the operators in front of the splat: workspace queries and argument checks.  No GPU needed: nothing here launches
a kernel."""
import ctypes

import pytest

ONE = ctypes.c_void_p(16)
S = (ctypes.c_longlong * 3)(64, 64, 8)
F32, BF16 = 0, 1


def _lib():
    from CudaGaussianVoxelizer import _lib
    return _lib.load()


def norm_forward(lib, B=1, nq=4, nk=4, hq=2, hk=2, D=8, A=3, P=3, q=ONE, k=ONE, dt=F32, pos=ONE, kpos=None, fr=ONE, eps=1e-6,
                 oq=ONE, ok=ONE, qs=S, ks=S):
    return lib.g2v_qk_norm_rotary_forward(B, nq, nk, hq, hk, D, A, P, q, qs, k, ks, dt, None, None, pos, kpos, fr, eps, oq, ok,
                                          None)


@pytest.mark.parametrize("bad,code,word", [
    (dict(B=-1), 1, b"negative"), (dict(D=0), 1, b"head_dim"), (dict(D=257), 1, b"head_dim"), (dict(A=0), 1, b"num_axes"),
    (dict(A=9), 1, b"num_axes"), (dict(P=5), 1, b"num_pairs"), (dict(P=-1), 1, b"num_pairs"), (dict(dt=2), 1, b"dtype"),
    (dict(nk=5), 1, b"n_k == n_q"), (dict(q=None), 1, b"null"), (dict(k=None), 1, b"null"), (dict(pos=None), 1, b"null"),
    (dict(fr=None), 1, b"freqs"), (dict(qs=None), 1, b"null"), (dict(oq=None), 1, b"null"), (dict(ok=None), 1, b"null"),
    (dict(eps=-1.0), 1, b"eps"), (dict(eps=float("nan")), 1, b"eps"), (dict(B=1 << 20, nq=1 << 20, nk=1 << 20), 3, b"limit"),
    (dict(hq=8193), 3, b"limit"),
])
def test_norm_arguments(bad, code, word):
    lib = _lib()
    assert norm_forward(lib, **bad) == code and word in lib.g2v_last_error()


def test_norm_without_rows_does_nothing():
    lib = _lib()
    assert norm_forward(lib, B=0, q=None, k=None, pos=None, fr=None, oq=None, ok=None, qs=None, ks=None) == 0
    assert norm_forward(lib, nq=0, nk=0, q=None, k=None, pos=None, fr=None, oq=None, ok=None, qs=None, ks=None) == 0


def test_norm_backward_arguments():
    lib = _lib()
    need = lib.g2v_qk_norm_rotary_backward_workspace(1, 4, 4, 2, 2, 8, 3, F32, 1)
    assert need > 0
    assert lib.g2v_qk_norm_rotary_backward_workspace(1, 4, 4, 2, 2, 257, 3, F32, 1) == 0

    def call(gq=ONE, dq=ONE, ws=ONE, nws=need):
        return lib.g2v_qk_norm_rotary_backward(1, 4, 4, 2, 2, 8, 3, 3, ONE, S, ONE, S, F32, None, None, ONE, None, ONE, 1e-6, gq,
                                               S, ONE, S, dq, ONE, None, None, None, None, ws, nws, None)

    for bad, word in ((dict(gq=None), b"null"), (dict(dq=None), b"null"), (dict(ws=None), b"workspace"),
                      (dict(nws=need - 1), b"workspace")):
        assert call(**bad) == 1 and word in lib.g2v_last_error(), bad


def attention(lib, B=1, nq=4, nk=4, hq=2, hk=2, D=8, q=ONE, k=ONE, v=ONE, dt=BF16, mask=None, scale=1.0, out=ONE, lst=None,
              ws=ONE, nws=1 << 30, qs=S):
    return lib.g2v_attention_forward(B, nq, nk, hq, hk, D, q, qs, k, S, v, S, dt, mask, scale, out, None, None, lst, ws, nws,
                                     None)


@pytest.mark.parametrize("bad,code,word", [
    (dict(B=-1), 1, b"negative"), (dict(D=0), 1, b"head_dim"), (dict(D=129), 1, b"head_dim"), (dict(hq=3), 1, b"multiple"),
    (dict(hk=0), 1, b"multiple"), (dict(dt=2), 1, b"dtype"), (dict(scale=0.0), 1, b"scale"), (dict(scale=-1.0), 1, b"scale"),
    (dict(scale=float("inf")), 1, b"scale"), (dict(scale=float("nan")), 1, b"scale"), (dict(scale=3e38), 1, b"scale"),
    (dict(q=None), 1, b"null"), (dict(k=None), 1, b"null"), (dict(v=None), 1, b"null"), (dict(out=None), 1, b"null"),
    (dict(qs=None), 1, b"null"), (dict(mask=ONE), 1, b"key_list"), (dict(ws=None), 1, b"workspace"),
    (dict(nws=1), 1, b"workspace"), (dict(B=1 << 20), 3, b"limit"), (dict(nk=1 << 25), 3, b"limit"), (dict(nq=1 << 30, hq=2, hk=1), 3, b"limit"),
])
def test_attention_arguments(bad, code, word):
    lib = _lib()
    assert attention(lib, **bad) == code and word in lib.g2v_last_error()


def test_attention_without_rows_does_nothing():
    lib = _lib()
    assert attention(lib, B=0, q=None, k=None, v=None, out=None, ws=None, qs=None) == 0
    assert attention(lib, nq=0, q=None, out=None, ws=None, qs=None) == 0


def test_attention_backward_arguments():
    lib = _lib()
    need = lib.g2v_attention_backward_workspace(1, 4, 4, 2, 2, 8, F32, 0, 0)

    def call(lse=ONE, out=ONE, g=ONE, dk=ONE, dv=ONE, ws=ONE, nws=need, scale=1.0):
        return lib.g2v_attention_backward(1, 4, 4, 2, 2, 8, ONE, S, ONE, S, ONE, S, F32, None, scale, out, None, lse, g, S, ONE,
                                          dk, dv, ws, nws, None)

    for bad, word in ((dict(lse=None), b"null"), (dict(out=None), b"null"), (dict(g=None), b"null"), (dict(dk=None), b"together"),
                      (dict(ws=None), b"workspace"), (dict(nws=need - 1), b"workspace"), (dict(scale=0.0), b"scale")):
        assert call(**bad) == 1 and word in lib.g2v_last_error(), bad


@pytest.mark.parametrize("query", ["g2v_attention_forward_workspace", "g2v_attention_backward_workspace"])
def test_attention_workspaces(query):
    """Refused sizes need nothing; packing and masks only add; what a call checks is what its query says (above)."""
    q = getattr(_lib(), query)
    assert q(1, 4, 4, 2, 2, 129, BF16, 1, 0) == 0 and q(1, 4, 4, 3, 2, 64, BF16, 1, 0) == 0
    for n in (1, 300, 5000, 18000):
        base = q(2, n, n, 8, 4, 64, BF16, 1, 0)
        assert 0 < base < q(2, n, n, 8, 4, 64, BF16, 1, 1) < q(2, n, n, 8, 4, 64, BF16, 0, 0)
        assert q(2, n, n, 8, 4, 64, BF16, 0, 1) == q(2, n, n, 8, 4, 64, BF16, 0, 0)
        assert q(2, n, n, 8, 4, 64, F32, 1, 0) == q(2, n, n, 8, 4, 64, F32, 0, 1) > 0
