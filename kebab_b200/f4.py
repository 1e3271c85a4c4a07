"""Products in microscaled 4-bit floating point: 32 consecutive values of a row
share a power-of-two scale (C ABI: include/kebab/f4.h).

    e = the least exponent >= -127 with amax <= 6 * 2^e     (of the 32 values)
    code = the nearest of 0, 1/2, 1, 3/2, 2, 3, 4, 6 to x / 2^e, ties to even
    Y[m, n] = sum_k X[m, k] W[n, k]  (+ bias[n])            (of the codes' values)

Tokens are rows: X is [M, K], W [N, K] (experts: [E, N, K]), Y [M, N]. Weights
are quantised once with quantize_f4(W), activations in every call of linear_f4 /
linear_grouped_f4, or once for several products with quantize_f4_tokens(X). K
and N are any numbers. All calls are asynchronous on `stream` (default: torch's
current stream) and raise KebabError on a refusal.
"""
from typing import NamedTuple

import torch

from ._call import CODES, bad, call, dense, elsewhere, on, pitch, stacked, tensor

_FLOATS = (torch.float16, torch.bfloat16)
_ANY = (torch.float16, torch.bfloat16, torch.float32)
_U8, _I32 = (torch.uint8,), (torch.int32,)
_SLACK = 160  # places of token scales past the last row


class F4(NamedTuple):
    """Quantised weights: codes [N, ceil(K / 32) * 16] (experts: [E, ...]), two
    a byte, and scales [ceil(N / 128), ceil(K / 128), 512] in the order that the
    tensor cores read."""
    codes: torch.Tensor
    scales: torch.Tensor


class F4Tokens(NamedTuple):
    """Quantised tokens: codes [M, ceil(K / 32) * 16], scales
    [ceil(K / 128), M + 160, 16]."""
    codes: torch.Tensor
    scales: torch.Tensor


def _up(a, b):
    return (a + b - 1) // b


def quantize_f4(W, stream=None):
    """Quantises the rows of weights [N, K] or of a stack [E, N, K] (F16, BF16 or F32) -> F4."""
    what = "quantize_f4"
    if isinstance(W, torch.Tensor) and W.dim() not in (2, 3):
        raise bad("quantize_f4: W must have 2 or 3 dimensions, got %s" % (tuple(W.shape),))
    dev = tensor(what, "W", W, W.dim() if isinstance(W, torch.Tensor) else 2, _ANY)
    if not W.numel():
        raise bad("quantize_f4: W must not be empty, got %s" % (tuple(W.shape),))
    if elsewhere(dev, stream):
        with on(dev, stream):
            return quantize_f4(W)
    lead, (N, K) = W.shape[:-2], W.shape[-2:]
    codes = W.new_empty((*lead, N, _up(K, 32) * 16), dtype=torch.uint8)
    scales = W.new_empty((*lead, _up(N, 128), _up(K, 128), 512), dtype=torch.uint8)
    ld, stride = stacked(W) if lead else (pitch(W), 0)
    call("kebab_quantize_f4", dev, CODES[W.dtype], W.data_ptr(), ld, stride, codes.data_ptr(), scales.data_ptr(),
         lead[0] if lead else 1, N, K)
    return F4(codes, scales)


def quantize_f4_tokens(X, stream=None):
    """Quantises the rows of tokens X [M, K] (F16, BF16 or F32) -> F4Tokens."""
    what = "quantize_f4_tokens"
    dev = tensor(what, "X", X, 2, _ANY)
    if X.shape[1] == 0:
        raise bad("quantize_f4_tokens: rows of X must not be empty")
    if elsewhere(dev, stream):
        with on(dev, stream):
            return quantize_f4_tokens(X)
    M, K = X.shape
    codes = X.new_empty((M, _up(K, 32) * 16), dtype=torch.uint8)
    scales = X.new_empty((_up(K, 128), M + _SLACK, 16), dtype=torch.uint8)
    call("kebab_quantize_f4_tokens", dev, CODES[X.dtype], X.data_ptr(), pitch(X), codes.data_ptr(), scales.data_ptr(),
         M, K)
    return F4Tokens(codes, scales)


def _check_weights(what, q, blocks, dim, dev):
    """Checks an F4 of `dim` dimensions whose rows have `blocks` blocks; returns (E, N)."""
    if not isinstance(q, F4):
        raise bad("%s: the weights must be what quantize_f4 returns" % what)
    codes, scales = q
    # Everything at once first: a call has a few microseconds.
    if isinstance(codes, torch.Tensor) and isinstance(scales, torch.Tensor) and codes.dim() == dim:
        shape = codes.shape
        N, at = shape[-2], codes.get_device()
        E = 1 if dim == 2 else shape[0]
        tiles = (N + 127) // 128, (blocks + 3) // 4, 512
        if (at >= 0 and at == (at if dev is None else dev) == scales.get_device() and shape[-1] == blocks * 16 and
                scales.shape == (tiles if dim == 2 else (E, *tiles)) and codes.dtype is scales.dtype is torch.uint8 and
                codes.is_contiguous() and scales.is_contiguous()):
            return E, N
    at = tensor(what, "the weights' codes", codes, dim, _U8, dev)
    if codes.shape[-1] != blocks * 16:
        raise bad("%s: inner dimensions differ: X has %d blocks of 32, the weights %d" %
                  (what, blocks, codes.shape[-1] // 16))
    dense(what, "the weights' codes", codes, codes.shape, _U8, at)
    dense(what, "the weights' scales", scales, (*codes.shape[:-2], _up(codes.shape[-2], 128), _up(blocks, 4), 512), _U8, at)
    raise bad("%s: the weights must not be empty" % what)


def dequantize_f4(q, K, dtype=torch.float32, stream=None):
    """The values [.., N, K] that quantised weights stand for, rounded to `dtype`."""
    what = "dequantize_f4"
    if dtype not in _ANY:
        raise bad("dequantize_f4: dtype must be float16, bfloat16 or float32")
    if not isinstance(K, int) or K < 1:
        raise bad("dequantize_f4: K = %s must be a positive integer" % (K,))
    dim = q.codes.dim() if isinstance(q, F4) and isinstance(q.codes, torch.Tensor) else 2
    if dim not in (2, 3):
        raise bad("dequantize_f4: the codes must have 2 or 3 dimensions")
    E, N = _check_weights(what, q, _up(K, 32), dim, None)
    dev = q.codes.get_device()
    if elsewhere(dev, stream):
        with on(dev, stream):
            return dequantize_f4(q, K, dtype)
    W = q.codes.new_empty((*q.codes.shape[:-1], K), dtype=dtype)
    call("kebab_dequantize_f4", dev, CODES[dtype], q.codes.data_ptr(), q.scales.data_ptr(), W.data_ptr(), E, N, K)
    return W


def _check_output(what, Y, bias, M, N, dtype, dev):
    if bias is not None:
        dense(what, "bias", bias, (N,), (dtype,), dev)
    if Y is not None:
        tensor(what, "Y", Y, 2, (dtype,), dev)
        if Y.shape != (M, N):
            raise bad("%s: Y must be [%d, %d], got %s" % (what, M, N, tuple(Y.shape)))


def _product(what, q, W, bias, offsets, dtype, Y, stream):
    if dtype not in _FLOATS:
        raise bad("%s: dtype must be float16 or bfloat16" % what)
    if not isinstance(q, F4Tokens):
        raise bad("%s: the tokens must be what quantize_f4_tokens returns" % what)
    dev = tensor(what, "the tokens' codes", q.codes, 2, _U8)
    M, blocks = q.codes.shape[0], q.codes.shape[1] // 16
    dense(what, "the tokens' codes", q.codes, (M, blocks * 16), _U8, dev)
    dense(what, "the tokens' scales", q.scales, (_up(blocks, 4), M + _SLACK, 16), _U8, dev)
    E, N = _check_weights(what, W, blocks, 2 if offsets is None else 3, dev)
    if offsets is not None:
        dense(what, "offsets", offsets, (E + 1,), _I32, dev)
    _check_output(what, Y, bias, M, N, dtype, dev)
    if elsewhere(dev, stream):
        with on(dev, stream):
            return _product(what, q, W, bias, offsets, dtype, Y, None)
    Y = q.codes.new_empty((M, N), dtype=dtype) if Y is None else Y
    operands = (CODES[dtype], q.codes.data_ptr(), q.scales.data_ptr(), W.codes.data_ptr(), W.scales.data_ptr())
    if offsets is None:
        call("kebab_gemm_f4", dev, *operands, None if bias is None else bias.data_ptr(), Y.data_ptr(), pitch(Y), M, N,
             blocks * 32)
    else:
        call("kebab_gemm_grouped_f4", dev, *operands, Y.data_ptr(), pitch(Y), offsets.data_ptr(), E, M, N, blocks * 32)
    return Y


def gemm_f4(q, W, bias=None, dtype=torch.bfloat16, Y=None, stream=None):
    """Y [M, N] (F16 or BF16) from quantised tokens (F4Tokens) and weights (F4)."""
    return _product("gemm_f4", q, W, bias, None, dtype, Y, stream)


def gemm_grouped_f4(q, W, offsets, dtype=torch.bfloat16, Y=None, stream=None):
    """Y[r] from row r of the tokens and the weights of its expert e: W an F4 of
    [E, N, K], offsets [E + 1] (int32, on the device; see gemm_grouped)."""
    if not isinstance(offsets, torch.Tensor):
        raise bad("gemm_grouped_f4: offsets must be a CUDA tensor")
    return _product("gemm_grouped_f4", q, W, None, offsets, dtype, Y, stream)


def _linear(what, X, W, bias, offsets, Y, stream):
    dev = tensor(what, "X", X, 2, _FLOATS)
    M, K = X.shape
    if K == 0:
        raise bad("%s: rows of X must not be empty" % what)
    E, N = _check_weights(what, W, _up(K, 32), 2 if offsets is None else 3, dev)
    if offsets is not None:
        dense(what, "offsets", offsets, (E + 1,), _I32, dev)
    _check_output(what, Y, bias, M, N, X.dtype, dev)
    if elsewhere(dev, stream):
        with on(dev, stream):
            return _linear(what, X, W, bias, offsets, Y, None)
    Y = X.new_empty((M, N)) if Y is None else Y
    size = M * _up(K, 32) * 16 + _up(K, 128) * (M + _SLACK) * 16  # kebab_linear_f4_workspace
    ws = X.new_empty((size,), dtype=torch.uint8)
    call("kebab_linear_f4", dev, CODES[X.dtype], X.data_ptr(), pitch(X), W.codes.data_ptr(), W.scales.data_ptr(),
         None if bias is None else bias.data_ptr(), Y.data_ptr(), pitch(Y), None if offsets is None else offsets.data_ptr(),
         E, M, N, K, ws.data_ptr(), size)
    return Y


def linear_f4(X, W, bias=None, Y=None, stream=None):
    """Y [M, N] of X's type: X [M, K] is quantised and multiplied with the
    quantised weights W (an F4 of [N, K])."""
    return _linear("linear_f4", X, W, bias, None, Y, stream)


def linear_grouped_f4(X, W, offsets, Y=None, stream=None):
    """linear_f4 grouped by expert: W an F4 of [E, N, K]; the rows offsets[e] ..
    offsets[e + 1] - 1 of X take expert e."""
    if not isinstance(offsets, torch.Tensor):
        raise bad("linear_grouped_f4: offsets must be a CUDA tensor")
    return _linear("linear_grouped_f4", X, W, None, offsets, Y, stream)
