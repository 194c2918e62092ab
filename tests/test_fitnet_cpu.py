"""The fitting-network calls refuse bad arguments before any CUDA call, and the torch ops refuse host tensors (no GPU needed)."""
import ctypes as C

import pytest
import torch

from ai2pot_b200 import capi, fitnet

NULL, ONE = C.c_void_p(None), C.c_void_p(256)
F32 = C.c_int(0)


class Dense(C.Structure):
    """ai2b_dense"""
    _fields_ = ([(k, C.c_int) for k in ("dtype", "activation", "groups", "inner", "outer")] + [("rows", C.c_longlong), ("d_offsets", C.c_void_p)] +
                [("d_x", C.c_void_p), ("x_stride", C.c_longlong), ("d_weight", C.c_void_p), ("d_bias", C.c_void_p), ("d_residual", C.c_void_p),
                 ("residual_stride", C.c_longlong), ("d_y", C.c_void_p), ("d_slope", C.c_void_p), ("d_gy", C.c_void_p), ("gy_stride", C.c_longlong)] +
                [(k, C.c_void_p) for k in ("d_gx", "d_gweight", "d_gbias", "d_gresidual", "d_workspace")] + [("workspace_bytes", C.c_size_t)])


def refused(rc, code, text):
    assert rc == code and text in capi.lib().ai2b_last_error_string(), (rc, capi.lib().ai2b_last_error_string())


def test_route_refusals():
    lib = capi.lib()
    lib.ai2b_route_workspace_bytes.restype = C.c_size_t
    call = lambda tokens, k, experts, index=ONE, ws=ONE, nbytes=1 << 20: lib.ai2b_route(index, C.c_int(0), C.c_longlong(tokens), C.c_int(k), C.c_int(experts), ONE, ONE, ONE, ws,
                                                                                       C.c_size_t(nbytes), NULL)
    refused(call(-1, 1, 3), -1, b"tokens -1")
    refused(call(10, 0, 3), -1, b"k 0")
    refused(call(10, 1, 0), -1, b"experts must be positive")
    refused(call(10, 1, 1025), -2, b"at most 1024")
    refused(call(2 ** 30, 2, 3), -2, b"2^31 - 1 slots")
    refused(call(10, 1, 3, index=NULL), -1, b"NULL")
    refused(call(100000, 1, 3, ws=NULL), -4, b"workspace")
    refused(lib.ai2b_route_dispatch(C.c_int(9), ONE, ONE, C.c_longlong(4), ONE, C.c_longlong(2), C.c_int(1), C.c_int(4), NULL), -1, b"element type 9")
    refused(lib.ai2b_route_dispatch(F32, ONE, ONE, C.c_longlong(3), ONE, C.c_longlong(2), C.c_int(1), C.c_int(4), NULL), -1, b"row stride 3")
    refused(lib.ai2b_route_combine(F32, NULL, ONE, C.c_longlong(4), NULL, ONE, C.c_longlong(2), C.c_int(1), C.c_int(4), NULL), -1, b"NULL")
    refused(lib.ai2b_route_combine_backward(F32, ONE, NULL, ONE, C.c_longlong(4), ONE, C.c_longlong(4), ONE, ONE, ONE, C.c_longlong(2), C.c_int(1), C.c_int(2), C.c_int(4), NULL),
            -1, b"NULL")


def test_dense_refusals():
    lib = capi.lib()
    good = dict(dtype=0, activation=1, groups=1, inner=4, outer=4, rows=8, d_x=256, x_stride=4, d_weight=256, d_y=256, d_gy=256, gy_stride=4, d_slope=256)
    for change, code, text in [(dict(dtype=3), -1, b"element type 3"), (dict(activation=7), -1, b"activation 7"), (dict(rows=-1), -1, b"rows -1"), (dict(inner=0), -1, b"inner 0"),
                               (dict(groups=2), -1, b"need offsets"), (dict(groups=2000, d_offsets=256), -2, b"1024 groups"), (dict(d_x=None), -1, b"x is NULL"),
                               (dict(x_stride=3), -1, b"row stride 3"), (dict(d_weight=None), -1, b"weight is NULL"), (dict(d_y=None), -1, b"y is NULL"),
                               (dict(d_residual=256, residual_stride=2), -1, b"residual")]:
        refused(lib.ai2b_dense_forward(C.byref(Dense(**dict(good, **change))), NULL), code, text)
    for change, code, text in [(dict(d_gy=None), -1, b"gy is NULL"), (dict(gy_stride=1), -1, b"row stride 1"), (dict(d_slope=None, d_gx=256), -1, b"slopes"), (dict(), -4, b"workspace"),
                               (dict(d_workspace=264, workspace_bytes=1 << 40), -4, b"aligned")]:
        refused(lib.ai2b_dense_backward(C.byref(Dense(**dict(good, **change))), NULL), code, text)
    refused(lib.ai2b_dense_forward(NULL, NULL), -1, b"NULL description")


def test_orthogonalize_refusals():
    lib = capi.lib()
    call = lambda dtype=0, batch=1, m=4, n=4, steps=5, eps=1e-7, out=ONE, ws=NULL: lib.ai2b_orthogonalize(
        C.c_int(dtype), out, ONE, C.c_int(batch), C.c_int(m), C.c_int(n), C.c_int(steps), C.c_double(3.0), C.c_double(-4.0), C.c_double(2.0), C.c_double(eps), ws,
        C.c_size_t(0), NULL)
    refused(call(dtype=5), -1, b"element type 5")
    refused(call(m=0), -1, b"m 0")
    refused(call(steps=-1), -1, b"steps -1")
    refused(call(eps=-1.0), -1, b"eps")
    refused(call(batch=70000), -2, b"65535")
    refused(call(out=NULL), -1, b"NULL")
    refused(call(), -4, b"workspace")


def test_host_tensors_are_refused():
    x, w = torch.ones(4, 8), torch.ones(3, 8)
    for call in (lambda: fitnet.route(torch.zeros(4, dtype=torch.int32), 2), lambda: fitnet.dense(x, w), lambda: fitnet.orthogonalize(w)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
