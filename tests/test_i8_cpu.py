"""Refusals of the 8-bit linear path, which need no GPU: the C entry points check their
arguments before they touch the device, and the Python calls check their tensors. The
pointers are never dereferenced."""
import ctypes

import pytest
import torch

ARG, CUDA, UNSUPPORTED, OK = -1, -3, -6, 0
P = 1 << 20  # "pointers", far enough apart not to overlap
X, R, W, Y, S, Q, SC = (P * k for k in range(1, 8))


def call(name, *args):
    import bbh

    return getattr(bbh.lib(), name)(*args)


def message():
    import bbh

    return bbh.lib().bbh_last_error().decode()


def rmsnorm(x=X, ldx=64, r=R, ldr=64, w=W, y=Y, ldy=64, s=S, lds=64, M=4, D=64, eps=1e-6, dtype=0):
    return call("bbh_rmsnorm", x, ldx, r, ldr, w, y, ldy, s, lds, M, D, eps, dtype, None)


def rmsnorm_i8(x=X, ldx=64, r=R, ldr=64, w=W, q=Q, ldq=64, sc=SC, s=S, lds=64, M=4, D=64, eps=1e-6, dtype=0):
    return call("bbh_rmsnorm_i8", x, ldx, r, ldr, w, q, ldq, sc, s, lds, M, D, eps, dtype, None)


def quantize(x=X, ldx=64, q=Q, ldq=64, sc=SC, M=4, D=64, dtype=0):
    return call("bbh_quantize_i8", x, ldx, q, ldq, sc, M, D, dtype, None)


def dequantize(q=Q, ldq=64, sc=SC, y=Y, ldy=64, M=4, D=64, dtype=0):
    return call("bbh_dequantize_i8", q, ldq, sc, y, ldy, M, D, dtype, None)


def linear(A=X, lda=64, sa=S, Wt=W, ldw=64, sw=SC, b=R, C=Y, ldc=32, M=4, N=32, K=64, gelu=0, dtype=0):
    return call("bbh_linear_i8", A, lda, sa, Wt, ldw, sw, b, C, ldc, M, N, K, gelu, dtype, None)


CALLS = {"rmsnorm": rmsnorm, "rmsnorm_i8": rmsnorm_i8, "quantize": quantize, "dequantize": dequantize,
         "linear": linear}


@pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers are not real")
@pytest.mark.parametrize("name", CALLS)
def test_good_arguments_reach_the_device_check(name):
    assert CALLS[name]() in (CUDA, UNSUPPORTED)


@pytest.mark.parametrize("name", CALLS)
def test_no_rows_is_no_work(name):
    assert CALLS[name](M=0) == OK


def test_linear_without_columns_is_no_work():
    assert linear(N=0) == OK


@pytest.mark.parametrize("name,bad", [
    ("rmsnorm", dict(M=-1)), ("rmsnorm", dict(D=0)), ("rmsnorm", dict(D=32769, ldx=40000, ldr=40000, ldy=40000, lds=40000)),
    ("rmsnorm", dict(x=None)), ("rmsnorm", dict(y=None)), ("rmsnorm", dict(r=None)),  # sum without residual
    ("rmsnorm", dict(ldx=63)), ("rmsnorm", dict(ldr=63)), ("rmsnorm", dict(ldy=63)), ("rmsnorm", dict(lds=63)),
    ("rmsnorm", dict(eps=-1e-6)), ("rmsnorm", dict(eps=float("nan"))), ("rmsnorm", dict(eps=float("inf"))),
    ("rmsnorm", dict(dtype=2)), ("rmsnorm", dict(dtype=-1)), ("rmsnorm", dict(x=X + 1)), ("rmsnorm", dict(w=W + 1)),
    ("rmsnorm", dict(y=X + 2)), ("rmsnorm", dict(y=X, ldy=65)), ("rmsnorm", dict(y=W)), ("rmsnorm", dict(s=Y)),
    ("rmsnorm", dict(s=X - 2)),
    ("rmsnorm_i8", dict(q=None)), ("rmsnorm_i8", dict(sc=None)), ("rmsnorm_i8", dict(ldq=60)),
    ("rmsnorm_i8", dict(q=X)), ("rmsnorm_i8", dict(sc=X + 4)), ("rmsnorm_i8", dict(sc=SC + 2)),
    ("rmsnorm_i8", dict(sc=Q)), ("rmsnorm_i8", dict(eps=-1.0)),
    ("quantize", dict(x=None)), ("quantize", dict(q=None)), ("quantize", dict(D=0)), ("quantize", dict(D=32769)),
    ("quantize", dict(ldx=63)), ("quantize", dict(ldq=63)), ("quantize", dict(dtype=7)), ("quantize", dict(q=X)),
    ("dequantize", dict(q=None)), ("dequantize", dict(sc=None)), ("dequantize", dict(y=None)),
    ("dequantize", dict(ldq=63)), ("dequantize", dict(ldy=63)), ("dequantize", dict(y=Q)), ("dequantize", dict(y=SC)),
    ("dequantize", dict(sc=SC + 1)), ("dequantize", dict(M=-2)),
    ("linear", dict(K=0)), ("linear", dict(K=131072, lda=131072, ldw=131072)), ("linear", dict(M=-1)), ("linear", dict(N=-1)),
    ("linear", dict(A=None)), ("linear", dict(sa=None)), ("linear", dict(Wt=None)), ("linear", dict(sw=None)),
    ("linear", dict(C=None)), ("linear", dict(lda=48)), ("linear", dict(ldw=48)), ("linear", dict(ldc=31)),
    ("linear", dict(lda=72)), ("linear", dict(ldw=72)), ("linear", dict(A=X + 8)), ("linear", dict(Wt=W + 8)),
    ("linear", dict(C=Y + 1)), ("linear", dict(b=R + 1)), ("linear", dict(sa=S + 2)), ("linear", dict(dtype=3)),
    ("linear", dict(C=X)), ("linear", dict(C=W)), ("linear", dict(C=S)), ("linear", dict(C=SC)), ("linear", dict(C=R)),
])
def test_refused_arguments(name, bad):
    assert CALLS[name](**bad) == ARG
    assert message().startswith("bbh_" + {"quantize": "quantize_i8", "dequantize": "dequantize_i8",
                                          "linear": "linear_i8"}.get(name, name))


def test_python_calls_refuse_host_tensors():
    import bbh

    x = torch.zeros(2, 16, dtype=torch.float16)
    q = torch.zeros(2, 16, dtype=torch.int8)
    s = torch.ones(2)
    for f in (lambda: bbh.rmsnorm(x), lambda: bbh.rmsnorm_i8(x), lambda: bbh.quantize_i8(x),
              lambda: bbh.dequantize_i8(q, s), lambda: bbh.linear_i8(q, s, q, s)):
        with pytest.raises(ValueError, match="CUDA"):
            f()


def test_entry_points_return_codes_not_exceptions():
    """Null everything: a code and a message, no crash."""
    import bbh

    L = bbh.lib()
    assert L.bbh_rmsnorm(None, 0, None, 0, None, None, 0, None, 0, 1, 1, 0.0, 0, None) == ARG
    assert L.bbh_linear_i8(None, 0, None, None, 0, None, None, None, 0, 1, 1, 1, 0, 0, None) == ARG
    assert isinstance(ctypes.string_at(L.bbh_last_error()), bytes)


COLUMNS = [("rmsnorm", dict(ldx=192, ldr=192, r=X + 128, ldy=192, y=X + 256)),
           ("rmsnorm", dict(ldx=192, x=X + 128, y=X, ldy=192)), ("rmsnorm", dict(ldx=192, s=X + 128, lds=192)),
           ("quantize", dict(ldx=96, q=X + 128, ldq=192)),
           ("dequantize", dict(ldq=256, y=Q + 64, ldy=128)),
           ("linear", dict(lda=128, C=X + 64, ldc=64))]


@pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers are not real")
@pytest.mark.parametrize("name,args", COLUMNS)
def test_columns_of_one_matrix_do_not_overlap(name, args):
    assert CALLS[name](**args) in (CUDA, UNSUPPORTED)


@pytest.mark.parametrize("name,args", [
    ("rmsnorm", dict(ldx=192, y=X + 126, ldy=192)), ("rmsnorm", dict(ldx=192, y=X + 258, ldy=192)),
    ("rmsnorm", dict(ldx=192, x=X + 128, y=X + 2, ldy=192)), ("rmsnorm", dict(ldx=192, y=X + 128, ldy=193)),
    ("quantize", dict(ldx=96, q=X + 127, ldq=192)), ("quantize", dict(ldx=96, q=X + 129, ldq=192)),
    ("linear", dict(lda=128, C=X + 62, ldc=64)), ("linear", dict(lda=128, C=X + 66, ldc=64))])
def test_columns_that_meet_are_refused(name, args):
    assert CALLS[name](**args) == ARG and "overlap" in message()
