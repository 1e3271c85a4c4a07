"""Root-mean-square norm of tokens with the residual's addition before it, an
output in 8-bit integers, and the gradients (C ABI: include/kebab/norm.h).

    s = x + residual                                  # rounded to x's type
    y[t, h] = s[t, h] * (mean_h s[t, h]^2 + eps)^(-1/2) * weight[h]

Tokens are rows: x is [T, H] (F16, BF16 or F32, rows contiguous), weight [H] of
x's type or float32. All calls are asynchronous on `stream` (default: torch's
current stream) and raise KebabError on a refusal. kebab_b200.moe has rms_norm
as a differentiable function.
"""
from typing import NamedTuple, Optional

import torch

from ._call import CODES, bad, call, dense, elsewhere, on, pitch, tensor

_ANY = (torch.float16, torch.bfloat16, torch.float32)


class Normed8(NamedTuple):
    """codes [T, H] int8 (rows at a pitch of whole 16 bytes) and scale [T] float32,
    operands of gemm_i8; the sum that was normed; y in x's type where it was
    asked for."""
    codes: torch.Tensor
    scale: torch.Tensor
    residual: torch.Tensor
    y: Optional[torch.Tensor]


def _check(what, x, weight, residual, name="x"):
    dev = tensor(what, name, x, 2, _ANY)
    if x.shape[1] == 0:
        raise bad("%s: rows of %s must not be empty" % (what, name))
    dense(what, "weight", weight, (x.shape[1],), (x.dtype, torch.float32), dev)
    _like(what, "residual", residual, x, dev)
    return dev


def _like(what, name, t, x, dev):
    if t is not None:
        tensor(what, name, t, 2, (x.dtype,), dev)
        if t.shape != x.shape:
            raise bad("%s: %s must be %s, got %s" % (what, name, tuple(x.shape), tuple(t.shape)))


def _rows_like(x):
    """A new contiguous tensor as x (empty_like takes 0.6 us less than new_empty)."""
    return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


def _row_pitch(t):
    """(address, row pitch) of a matrix or of None."""
    return (None, 0) if t is None else (t.data_ptr(), pitch(t))


def rms_norm(x, weight, eps=1e-6, residual=None, stream=None):
    """-> (y, s), both [T, H] of x's type: the normed tokens and the sum
    x + residual that was normed (x itself without a residual)."""
    dev = _check("rms_norm", x, weight, residual)
    if elsewhere(dev, stream):
        with on(dev, stream):
            return rms_norm(x, weight, eps, residual)
    T, H = x.shape
    y = _rows_like(x)
    if residual is None:
        s, r, ldr = x, None, 0
    else:
        s, r, ldr = _rows_like(x), residual.data_ptr(), pitch(residual)
    call("kebab_rms_norm", dev, CODES[x.dtype], CODES[weight.dtype], x.data_ptr(), pitch(x), r, ldr, weight.data_ptr(),
         eps, s.data_ptr(), H, y.data_ptr(), H, T, H)
    return y, s


def rms_norm_i8(x, weight, eps=1e-6, residual=None, keep=False, stream=None):
    """rms_norm with y in 8-bit integers, quantised by row from its 32-bit
    values -> Normed8; `keep`: y in x's type too."""
    dev = _check("rms_norm_i8", x, weight, residual)
    if elsewhere(dev, stream):
        with on(dev, stream):
            return rms_norm_i8(x, weight, eps, residual, keep)
    T, H = x.shape
    # Rows of codes on 16 bytes, as the products' copies need them.
    Hp = (H + 15) // 16 * 16
    codes, scale = x.new_empty((T, Hp), dtype=torch.int8), x.new_empty((T,), dtype=torch.float32)
    codes = codes if Hp == H else codes[:, :H]
    y = _rows_like(x) if keep else None
    s = x if residual is None else _rows_like(x)
    call("kebab_rms_norm_i8", dev, CODES[x.dtype], CODES[weight.dtype], x.data_ptr(), pitch(x), *_row_pitch(residual),
         weight.data_ptr(), eps, s.data_ptr(), H, y.data_ptr() if keep else None, H, codes.data_ptr(), Hp, scale.data_ptr(), T, H)
    return Normed8(codes, scale, s, y)


def rms_norm_backward(dy, s, weight, eps=1e-6, dresidual=None, stream=None, need=(True, True)):
    """Gradients of rms_norm from that of y, and `dresidual`, that of s where it
    is used past the norm -> (dx, dweight): dx [T, H] is the gradient of x and
    of the residual; dweight [H] has weight's type. `need`: whether to compute
    each of the two, None in place of one that is not."""
    what = "rms_norm_backward"
    dev = _check(what, s, weight, None, "s")
    if dy is None:
        raise bad("rms_norm_backward: dy must be a CUDA tensor")
    _like(what, "dy", dy, s, dev)
    _like(what, "dresidual", dresidual, s, dev)
    if elsewhere(dev, stream):
        with on(dev, stream):
            return rms_norm_backward(dy, s, weight, eps, dresidual, need=need)
    T, H = s.shape
    dx, dweight = _rows_like(s) if need[0] else None, torch.empty_like(weight) if need[1] else None
    size = (T * 8 + 15) // 16 * 16 + min((T + 7) // 8 * 8, 1024) * H * 4  # kebab_rms_norm_backward_workspace
    ws = s.new_empty((size,), dtype=torch.uint8)
    call("kebab_rms_norm_backward", dev, CODES[s.dtype], CODES[weight.dtype], dy.data_ptr(), pitch(dy), s.data_ptr(),
         pitch(s), weight.data_ptr(), eps, *_row_pitch(dresidual), dx.data_ptr() if need[0] else None, H,
         dweight.data_ptr() if need[1] else None, ws.data_ptr(), size, T, H)
    return dx, dweight
