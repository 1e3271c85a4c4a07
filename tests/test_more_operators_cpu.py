"""Refusals of the norm, 4-bit and few-token operators, and the norm's gradient
formula against differences — no GPU."""
import ctypes

import numpy as np
import pytest

import kebab_b200 as kb

P = ctypes.c_void_p(64)
BAD = ctypes.c_void_p(65)


def f(name):
    from kebab_b200._call import function
    return function(name)


def sizes(name, *args):
    L = kb.lib()
    g = getattr(L, name)
    g.restype = ctypes.c_int64
    g.argtypes = [ctypes.c_int64] * len(args)
    return g(*args)


def test_norm_refusals():
    def norm(dtype=kb.F16, wt=kb.F32, x=P, ldx=8, r=P, ldr=8, w=P, eps=1e-6, s=P, lds=8, y=P, ldy=8, T=2, H=8):
        return f("kebab_rms_norm")(dtype, wt, x, ldx, r, ldr, w, eps, s, lds, y, ldy, T, H, None)

    def norm8(dtype=kb.F16, wt=kb.F32, x=P, ldx=8, r=P, ldr=8, w=P, eps=1e-6, s=P, lds=8, y=None, ldy=0, q=P, ldq=8, sc=P, T=2, H=8):
        return f("kebab_rms_norm_i8")(dtype, wt, x, ldx, r, ldr, w, eps, s, lds, y, ldy, q, ldq, sc, T, H, None)

    for call in (norm, norm8):
        assert call(dtype=7) == kb.ENOTSUP and call(dtype=kb.F16, wt=kb.BF16) == kb.ENOTSUP
        for args in (dict(T=-1), dict(H=0), dict(H=1 << 31, ldx=1 << 31), dict(ldx=7), dict(ldr=7), dict(lds=7), dict(x=None), dict(w=None), dict(s=None),
                     dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(T=1 << 31)):
            assert call(**args) == kb.EINVAL, args
        assert call(T=0, x=None) == kb.OK
    assert norm(y=None) == kb.EINVAL and norm(ldy=7) == kb.EINVAL
    assert norm8(q=None) == kb.EINVAL and norm8(sc=None) == kb.EINVAL and norm8(ldq=7) == kb.EINVAL and norm8(y=P, ldy=7) == kb.EINVAL

    def back(dtype=kb.F16, wt=kb.F32, dy=P, lddy=8, s=P, lds=8, w=P, eps=1e-6, ds=P, ldds=8, dx=P, lddx=8, dw=P, ws=P, size=1 << 20, T=2, H=8):
        return f("kebab_rms_norm_backward")(dtype, wt, dy, lddy, s, lds, w, eps, ds, ldds, dx, lddx, dw, ws, size, T, H, None)

    assert back(dtype=7) == kb.ENOTSUP and back(wt=kb.BF16) == kb.ENOTSUP
    need = sizes("kebab_rms_norm_backward_workspace", 2, 8)
    assert need == 16 + 8 * 8 * 4 and sizes("kebab_rms_norm_backward_workspace", 2, 0) == -kb.EINVAL
    for args in (dict(T=-1), dict(H=0), dict(lddy=7), dict(lds=7), dict(ldds=7), dict(lddx=7), dict(dy=None), dict(s=None), dict(w=None), dict(ws=None),
                 dict(ws=BAD), dict(size=need - 1), dict(eps=-1.0), dict(H=(1 << 32) + 8, lddy=1 << 40, lds=1 << 40, ldds=1 << 40, lddx=1 << 40)):
        assert back(**args) == kb.EINVAL, args
    assert back(T=0, dw=None) == kb.OK and back(dx=None, dw=None) == kb.OK


def test_f4_refusals():
    def quantize(dtype=kb.F16, W=P, ld=64, st=0, c=P, s=P, E=1, N=4, K=64):
        return f("kebab_quantize_f4")(dtype, W, ld, st, c, s, E, N, K, None)

    def tokens(dtype=kb.F16, X=P, ld=64, c=P, s=P, R=4, K=64):
        return f("kebab_quantize_f4_tokens")(dtype, X, ld, c, s, R, K, None)

    def dequantize(dtype=kb.F16, c=P, s=P, W=P, E=1, N=4, K=64):
        return f("kebab_dequantize_f4")(dtype, c, s, W, E, N, K, None)

    for call in (quantize, tokens, dequantize):
        assert call(dtype=9) == kb.ENOTSUP
        for args in (dict(K=0), dict(K=1 << 31), dict(c=None), dict(s=None), dict(c=BAD), dict(s=BAD)):
            assert call(**args) == kb.EINVAL, args
    for call in (quantize, dequantize):
        assert call(N=0) == kb.EINVAL and call(E=0) == kb.EINVAL and call(E=1025) == kb.EINVAL and call(W=None) == kb.EINVAL
    assert quantize(ld=63) == kb.EINVAL and tokens(ld=63) == kb.EINVAL and tokens(X=None) == kb.EINVAL and tokens(R=-1) == kb.EINVAL
    assert tokens(R=0, X=None) == kb.OK
    assert sizes("kebab_f4_code_bytes", 3, 65) == 3 * 48 and sizes("kebab_f4_code_bytes", 3, 0) == -kb.EINVAL
    assert sizes("kebab_f4_weight_scale_bytes", 129, 129) == 4 * 512 and sizes("kebab_f4_weight_scale_bytes", 0, 1) == -kb.EINVAL
    assert sizes("kebab_f4_token_scale_bytes", 3, 129) == 2 * 163 * 16 and sizes("kebab_f4_token_scale_bytes", -1, 1) == -kb.EINVAL
    assert sizes("kebab_linear_f4_workspace", 3, 65) == 3 * 48 + 163 * 16 and sizes("kebab_linear_f4_workspace", 3, 0) == -kb.EINVAL

    def gemm(out=kb.F16, xc=P, xs=P, wc=P, ws=P, Y=P, ldy=64, M=4, N=64, K=64):
        return f("kebab_gemm_f4")(out, xc, xs, wc, ws, None, Y, ldy, M, N, K, None)

    def grouped(out=kb.F16, xc=P, xs=P, wc=P, ws=P, Y=P, ldy=64, off=P, E=2, M=4, N=64, K=64):
        return f("kebab_gemm_grouped_f4")(out, xc, xs, wc, ws, Y, ldy, off, E, M, N, K, None)

    for call in (gemm, grouped):
        assert call(out=kb.F32) == kb.ENOTSUP
        for args in (dict(M=-1), dict(N=0), dict(K=0), dict(K=1 << 31), dict(ldy=63), dict(xc=None), dict(xs=None), dict(wc=None), dict(ws=None), dict(Y=None),
                     dict(xc=BAD), dict(xs=BAD), dict(wc=BAD), dict(ws=BAD)):
            assert call(**args) == kb.EINVAL, args
        assert call(M=0, xc=None, xs=None, Y=None) == kb.OK
    assert grouped(off=None) == kb.EINVAL and grouped(E=0) == kb.EINVAL and grouped(E=1025) == kb.EINVAL

    def linear(dtype=kb.F16, X=P, ld=64, bias=None, off=None, E=1, ws=P, size=1 << 20, M=4, N=64, K=64):
        return f("kebab_linear_f4")(dtype, X, ld, P, P, bias, P, 64, off, E, M, N, K, ws, size, None)

    need = sizes("kebab_linear_f4_workspace", 4, 64)
    assert linear(E=2) == kb.EINVAL and "one weight matrix" in kb.last_error()
    assert linear(off=P, bias=P) == kb.EINVAL and "no bias" in kb.last_error()
    assert linear(dtype=kb.F32) == kb.ENOTSUP
    for args in (dict(X=None), dict(ld=63), dict(ws=None), dict(ws=BAD), dict(size=need - 1), dict(M=-1), dict(N=0), dict(K=0)):
        assert linear(**args) == kb.EINVAL, args
    assert linear(M=0, ws=None, size=0) == kb.OK


def test_layer_refusals():
    def layer(dtype=kb.F16, x=P, ldx=8, r=P, wi=P, wo=P, y=P, ldy=8, T=2, E=4, k=2, H=8, D=8, ws=P, size=1 << 24):
        return f("kebab_expert_layer")(dtype, x, ldx, r, wi, wo, y, ldy, T, E, k, 1, H, D, ws, size, None)

    def layer8(dtype=kb.F16, x=P, ldx=8, r=P, wi=P, si=P, wo=P, so=P, y=P, ldy=8, T=2, E=4, k=2, H=8, D=8, ws=P, size=1 << 24):
        return f("kebab_expert_layer_i8")(dtype, x, ldx, r, wi, si, wo, so, y, ldy, T, E, k, 1, H, D, ws, size, None)

    L = kb.lib()
    L.kebab_expert_layer_workspace.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.c_int, ctypes.c_int64, ctypes.c_int64]
    L.kebab_expert_layer_workspace.restype = ctypes.c_int64
    need = L.kebab_expert_layer_workspace(2, 4, 2, 8, 8)
    assert need > 0
    for T, E, k, H, D in ((-1, 4, 2, 8, 8), (17, 4, 2, 8, 8), (2, 0, 2, 8, 8), (2, 1025, 2, 8, 8), (2, 4, 0, 8, 8), (2, 4, 33, 8, 8), (2, 4, 2, 0, 8), (2, 4, 2, 8, 0),
                          (2, 4, 2, 1 << 25, 8), (2, 4, 2, 8, 1 << 25)):
        assert L.kebab_expert_layer_workspace(T, E, k, H, D) == -kb.EINVAL
        for call in (layer, layer8):
            assert call(T=T, E=E, k=k, H=H, D=D, ldx=max(H, 8), ldy=max(H, 8)) == kb.EINVAL, (T, E, k, H, D)
    for call in (layer, layer8):
        assert call(dtype=kb.F32) == kb.ENOTSUP
        for args in (dict(k=5), dict(ldx=7), dict(ldy=7), dict(x=None), dict(r=None), dict(wi=None), dict(wo=None), dict(y=None), dict(ws=None), dict(ws=BAD), dict(size=need - 1)):
            assert call(**args) == kb.EINVAL, args
        assert call(T=0, x=None, ws=None) == kb.OK
    assert layer8(si=None) == kb.EINVAL and layer8(so=None) == kb.EINVAL
    assert layer8(H=131073, ldx=131073, ldy=131073) == kb.EINVAL and layer8(D=131073) == kb.EINVAL


def test_python_refuses_host_tensors():
    import torch
    x, w = torch.zeros((2, 32), dtype=torch.float16), torch.zeros(32)
    q = kb.F4(torch.zeros((8, 16), dtype=torch.uint8), torch.zeros((1, 1, 512), dtype=torch.uint8))
    t = kb.F4Tokens(torch.zeros((2, 16), dtype=torch.uint8), torch.zeros((1, 162, 16), dtype=torch.uint8))
    off, r = torch.zeros(2, dtype=torch.int32), torch.zeros((4, 32))
    wi, wo, i8 = torch.zeros((4, 8, 32), dtype=torch.float16), torch.zeros((4, 32, 4), dtype=torch.float16), torch.zeros((4, 8, 32), dtype=torch.int8)
    for call in (lambda: kb.rms_norm(x, w), lambda: kb.rms_norm_i8(x, w), lambda: kb.rms_norm_backward(x, x, w), lambda: kb.quantize_f4(x), lambda: kb.quantize_f4(None),
                 lambda: kb.quantize_f4_tokens(x), lambda: kb.dequantize_f4(q, 32), lambda: kb.gemm_f4(t, q), lambda: kb.linear_f4(x, q),
                 lambda: kb.gemm_grouped_f4(t, q, off), lambda: kb.linear_grouped_f4(x, q, off), lambda: kb.expert_layer(x, r, wi, wo, 2),
                 lambda: kb.expert_layer_i8(x, r, i8, w, i8, w, 2)):
        with pytest.raises(kb.KebabError) as e:
            call()
        assert e.value.code == kb.EINVAL and "CUDA tensor" in str(e.value)


def test_norm_gradient_formula():
    """The formula that the kernel uses, against central differences in float64: h^2 of a third derivative of
    magnitude below 100 for these inputs, and 2^-50 / h."""
    rng = np.random.default_rng(1)
    T, H, eps, h = 3, 9, 1e-3, 1e-4
    s, w, dy = rng.standard_normal((T, H)), rng.standard_normal(H), rng.standard_normal((T, H))

    def norm(s, w):
        return s / np.sqrt((s * s).mean(1, keepdims=True) + eps) * w

    rstd = 1 / np.sqrt((s * s).mean(1, keepdims=True) + eps)
    g = dy * w
    dx = rstd * (g - s * rstd ** 2 * (g * s).mean(1, keepdims=True))
    dw = (dy * s * rstd).sum(0)
    bound = np.abs(dy).sum() * (100 * h * h + 2.0 ** -50 / h)
    for c in range(H):
        step = np.zeros(H)
        step[c] = h
        slope = ((norm(s + step, w) - norm(s - step, w)) / (2 * h) * dy).sum(1)
        assert np.abs(slope - dx[:, c]).max() <= bound
        slope = ((norm(s, w + step) - norm(s, w - step)) / (2 * h) * dy).sum()
        assert abs(slope - dw[c]) <= bound
