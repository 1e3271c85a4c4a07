"""Refusals of the expert and 8-bit integer operators, and the gradient
formulas against differences — no GPU."""
import ctypes

import numpy as np
import pytest

import kebab_b200 as kb

P = ctypes.c_void_p(64)
BAD = ctypes.c_void_p(65)


def f(name):
    from kebab_b200._call import function
    return function(name)


def grouped(dtype=kb.F16, X=P, ldx=64, W=P, ldw=64, stride=4096, Y=P, ldy=64, off=P, E=2, R=4, N=64, K=64, mode=b"RC"):
    return f("kebab_gemm_grouped")(dtype, X, ldx, W, ldw, stride, Y, ldy, off, E, R, N, K, mode, None)


def grouped_dw(dtype=kb.F16, X=P, ldx=64, dY=P, lddy=64, dW=P, off=P, E=2, R=4, N=64, K=64, mode=b"RC"):
    return f("kebab_gemm_grouped_dw")(dtype, X, ldx, dY, lddy, dW, off, E, R, N, K, mode, None)


@pytest.mark.parametrize("args,code,text", [
    (dict(dtype=kb.F32), kb.ENOTSUP, "F16 and BF16"), (dict(E=0), kb.EINVAL, "experts"), (dict(E=1025), kb.EINVAL, "experts"),
    (dict(R=-1), kb.EINVAL, "dimensions"), (dict(N=0), kb.EINVAL, "dimensions"), (dict(K=0), kb.EINVAL, "dimensions"),
    (dict(K=1 << 31, ldx=1 << 31), kb.EINVAL, "2^30"), (dict(ldx=63), kb.EINVAL, "pitch of X"),
    (dict(mode=b"CR"), kb.EINVAL, "opmode"), (dict(mode=b"RCR"), kb.EINVAL, "opmode"), (dict(X=None), kb.EINVAL, "null")])
def test_grouped_refusals(args, code, text):
    assert grouped(**args) == code
    assert text in kb.last_error()
    assert grouped_dw(**args) == code
    assert text in kb.last_error()


def test_grouped_forward_only_refusals():
    for args in (dict(ldw=63), dict(ldy=63), dict(stride=4095), dict(mode=b"RR", K=65, ldx=65), dict(W=None), dict(Y=None), dict(off=None)):
        assert grouped(**args) == kb.EINVAL, args
    assert grouped(R=0, X=None, Y=None) == kb.OK  # nothing to do
    assert grouped_dw(lddy=63) == kb.EINVAL and grouped_dw(dW=None) == kb.EINVAL and grouped_dw(dY=None) == kb.EINVAL


def test_i8_refusals():
    def gemm(out=kb.F16, q=P, ldq=64, s=P, w=P, ldw=64, ws=P, Y=P, ldy=64, M=4, N=64, K=64):
        return f("kebab_gemm_i8")(out, q, ldq, s, w, ldw, ws, None, Y, ldy, M, N, K, None)

    assert gemm(out=kb.F32) == kb.ENOTSUP
    for args in (dict(M=-1), dict(N=0), dict(K=0), dict(ldq=63), dict(ldw=63), dict(ldy=63), dict(q=None), dict(s=None),
                 dict(w=None), dict(ws=None), dict(Y=None)):
        assert gemm(**args) == kb.EINVAL, args
    assert gemm(K=131073, ldq=131073, ldw=131073) == kb.EINVAL and "overflow" in kb.last_error()
    assert gemm(M=0, q=None, s=None, Y=None) == kb.OK

    def linear(dtype=kb.F16, bias=None, off=None, E=1, ws=P, size=1 << 20, M=4):
        return f("kebab_linear_i8")(dtype, P, 64, P, 64, 4096, P, bias, P, 64, off, E, M, 64, 64, ws, size, None)

    assert linear(E=2) == kb.EINVAL and "one weight matrix" in kb.last_error()
    assert linear(off=P, bias=P) == kb.EINVAL and "no bias" in kb.last_error()
    assert linear(ws=None) == kb.EINVAL and linear(ws=BAD) == kb.EINVAL and linear(size=4 * 68 - 1) == kb.EINVAL
    assert linear(M=0, ws=None, size=0) == kb.OK
    L = kb.lib()
    L.kebab_linear_i8_workspace.argtypes = [ctypes.c_int64, ctypes.c_int64]
    L.kebab_linear_i8_workspace.restype = ctypes.c_int64
    assert L.kebab_linear_i8_workspace(4, 64) == 4 * 68 and L.kebab_linear_i8_workspace(3, 65) == 3 * 84
    assert L.kebab_linear_i8_workspace(3, 0) == -kb.EINVAL

    def quantize(dtype=kb.F16, X=P, ldx=8, q=P, ldq=8, s=P, M=2, K=8):
        return f("kebab_quantize_i8")(dtype, X, ldx, q, ldq, s, M, K, None)

    assert quantize(dtype=7) == kb.ENOTSUP and quantize(M=0, X=None) == kb.OK
    for args in (dict(M=-1), dict(K=0), dict(ldx=7), dict(ldq=7), dict(X=None), dict(q=None), dict(s=None)):
        assert quantize(**args) == kb.EINVAL, args


def test_route_and_exchange_refusals():
    def route(dtype=kb.F32, x=P, ld=300, T=200, E=300, k=2, w=P, ws=P, size=148 * 300 * 4):
        return f("kebab_route")(dtype, x, ld, T, E, k, 1, w, P, P, P, ws, size, None)

    assert route(dtype=9) == kb.ENOTSUP
    for args in (dict(E=0), dict(E=1025, ld=2000), dict(k=0), dict(k=33), dict(E=3, k=4), dict(T=-1), dict(T=1 << 30), dict(ld=299),
                 dict(x=None), dict(w=None), dict(ws=None), dict(size=148 * 300 * 4 - 1), dict(ws=BAD)):
        assert route(**args) == kb.EINVAL, args

    def back(x=P, ldd=8, k=2, d=P, T=3):
        return f("kebab_route_backward")(kb.F32, x, 8, T, 8, k, 1, P, P, P, d, ldd, None)

    assert back(x=None) == kb.EINVAL and back(ldd=7) == kb.EINVAL and back(k=9) == kb.EINVAL and back(d=None) == kb.EINVAL
    assert back(T=0, x=None) == kb.OK

    def dispatch(dtype=kb.F16, x=P, ldx=8, ldxs=8, T=2, k=2, R=4, H=8):
        return f("kebab_expert_dispatch")(dtype, x, ldx, P, P, ldxs, T, k, R, H, None)

    def combine(dtype=kb.F16, ys=P, ldys=8, ldy=8, T=2, k=2, R=4, H=8):
        return f("kebab_expert_combine")(dtype, ys, ldys, P, P, P, ldy, T, k, R, H, None)

    def combine_back(dtype=kb.F16, dy=P, lddy=8, ldys=8, T=2, k=2, R=4, H=8):
        return f("kebab_expert_combine_backward")(dtype, dy, lddy, P, ldys, P, P, P, 8, P, T, k, R, H, None)

    for call in (dispatch, combine, combine_back):
        assert call(dtype=kb.F32) == kb.ENOTSUP
        for args in (dict(T=-1), dict(k=0), dict(k=33), dict(H=0), dict(R=-1), dict(T=1 << 30)):
            assert call(**args) == kb.EINVAL, args
        assert call(T=0) == kb.OK
    assert dispatch(x=None) == kb.EINVAL and dispatch(ldx=7) == kb.EINVAL and dispatch(ldxs=7) == kb.EINVAL
    assert combine(ys=None) == kb.EINVAL and combine(ldys=7) == kb.EINVAL and combine(ldy=7) == kb.EINVAL
    assert combine_back(dy=None) == kb.EINVAL and combine_back(lddy=7) == kb.EINVAL and combine_back(ldys=7) == kb.EINVAL


def test_python_refuses_host_tensors():
    import torch
    x, w = torch.zeros((2, 8), dtype=torch.float16), torch.zeros((2, 8, 8), dtype=torch.float16)
    off, q = torch.zeros(3, dtype=torch.int32), torch.zeros((2, 8), dtype=torch.int8)
    s, slots = torch.zeros(2), torch.zeros((2, 1), dtype=torch.int32)
    for call in (lambda: kb.gemm_grouped(x, w, off), lambda: kb.gemm_grouped_dw(x, x, off), lambda: kb.quantize_i8(x),
                 lambda: kb.gemm_i8(q, s, q, s), lambda: kb.linear_i8(x, q, s), lambda: kb.linear_grouped_i8(x, q[None], s[None], off),
                 lambda: kb.route(x, 1), lambda: kb.dispatch(x, slots), lambda: kb.combine(x, slots),
                 lambda: kb.combine_backward(x, x, slots, s[:, None]), lambda: kb.gemm_grouped(None, w, off)):
        with pytest.raises(kb.KebabError) as e:
            call()
        assert e.value.code == kb.EINVAL and "CUDA tensor" in str(e.value)
    with pytest.raises(kb.KebabError):
        kb.gemm_grouped(x, w, off, opmode="CC")
    with pytest.raises(AttributeError):
        kb.no_such_operator


def softmax_weights(x, experts, renormalize):
    e = np.exp(x - x.max(1, keepdims=True))
    top = np.take_along_axis(e, experts, 1)
    return top / (top if renormalize else e).sum(1, keepdims=True)


@pytest.mark.parametrize("renormalize", [True, False])
def test_routing_gradient_formula(renormalize):
    """The formula that the kernel uses, against central differences of the
    weights in float64: h^2 of a third derivative below 6, and 2^-52 / h."""
    rng = np.random.default_rng(1)
    T, E, k, h = 7, 12, 3, 1e-4
    x, dw = rng.standard_normal((T, E)), rng.standard_normal((T, k))
    experts = np.argsort(-x, axis=1, kind="stable")[:, :k]
    w = softmax_weights(x, experts, renormalize)
    d, p = np.zeros_like(x), np.zeros_like(x)
    np.put_along_axis(d, experts, dw, 1)
    if renormalize:
        np.put_along_axis(p, experts, w, 1)
    else:
        p = np.exp(x) / np.exp(x).sum(1, keepdims=True)
    formula = p * (d - (w * dw).sum(1, keepdims=True))
    for e in range(E):
        step = np.zeros_like(x)
        step[:, e] = h
        up, down = (softmax_weights(x + s * step, experts, renormalize) for s in (1, -1))
        slope = ((up - down) / (2 * h) * dw).sum(1)
        assert np.abs(slope - formula[:, e]).max() <= np.abs(dw).sum(1).max() * (h * h + 2.0 ** -50 / h)
