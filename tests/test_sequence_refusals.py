"""What the token-sequence operators refuse, before anything reaches a GPU: the Python front end's messages and the C
entry points' status codes (workspace sizes, types, limits).  No GPU needed: every call below returns on the host."""
import ctypes as C

import pytest
import torch


def _B():
    from genjax_amd import backend as B

    return B


def test_linear_categorical_front_end_refusals():
    B = _B()
    x, w, b, y = torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(5), torch.zeros(3, dtype=torch.int32)
    bad = [
        ((y, x, torch.zeros(5, 9), b), "must be"),
        ((y, x[0], w, b), "must be"),
        ((y, x, w[:0], b[:0]), "must be"),
        ((y, x, w, torch.zeros(4)), "bias"),
        ((y, x.double(), w.double(), b.double()), "float32 or all bfloat16"),
        ((y, x.half(), w.half(), b.half()), "float32 or all bfloat16"),
        ((y, x.bfloat16(), w, b), "float32 or all bfloat16"),
        ((y, x, w, b), "device tensor"),
    ]
    for args, message in bad:
        with pytest.raises(B.GjxError, match=message):
            B.linear_categorical_logpdf(*args)


def test_linear_categorical_abi_refusals():
    from genjax_amd import _native as N

    L = N.lib()
    p = C.c_void_p(1 << 20)                      # never dereferenced: each call is refused on the host
    size = C.c_int64()

    def code(dtype=0, x=p, x_ld=8, w=p, w_ld=8, n=3, vocab=5, width=8, y=p, lp=p, lse=p, work=p, work_bytes=1 << 30):
        return L.gjx_linear_categorical_logpdf(dtype, y, x, x_ld, w, w_ld, None, n, vocab, width, lp, lse, work, work_bytes, None)

    assert L.gjx_linear_categorical_workspace(0, p, 8, p, 8, 3, 5, 8, 1, C.byref(size)) == 0 and size.value > 0
    assert L.gjx_linear_categorical_workspace(0, p, 8, p, 8, 3, 5, 8, 1, None) == -1
    assert code(dtype=2) == -1 and b"dtype" in L.gjx_last_error()
    assert code(n=-1) == -1 and code(vocab=0) == -1 and code(width=0) == -1
    assert code(x=None) == -1 and code(w=None) == -1 and code(y=None) == -1 and code(lp=None) == -1
    assert code(x_ld=7) == -1 and code(w_ld=7) == -1 and b"stride" in L.gjx_last_error()
    assert code(work=None) == -1 and code(work_bytes=16) == -1 and b"workspace" in L.gjx_last_error()
    assert code(work=C.c_void_p((1 << 20) + 8)) == -1
    assert code(n=(1 << 24) + 1) == -4 and code(vocab=(1 << 24) + 1) == -4
    assert code(width=65537, x_ld=65537, w_ld=65537) == -4
    assert code(n=0, y=None, x=None, w=None, lp=None, lse=None, work=None, work_bytes=0) == 0       # nothing to do
    assert L.gjx_linear_categorical_grad(0, p, p, 8, p, 8, None, 3, 5, 8, None, p, p, p, p, p, 1 << 30, None) == -1
    assert L.gjx_linear_categorical_grad(0, p, p, 8, p, 8, None, 3, 5, 8, p, p, p, p, p, p, 16, None) == -1
    key = (C.c_uint32 * 2)(0, 1)
    assert L.gjx_random_linear_categorical_i32(key, 0, 0, p, 8, p, 8, None, 3, 5, 8, None, p, 1 << 30, None) == -1
