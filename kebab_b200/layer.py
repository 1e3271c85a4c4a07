"""A whole mixture-of-experts feed-forward layer for a few tokens, from the
router to the sum over the experts (C ABI: include/kebab/layer.h).

    y[t] = sum_j w[t, j] w_out[e] (silu(g) * u),  [g; u] = w_in[e] x[t]

over the k experts e = e[t, j] with the largest logits router x[t]: what route,
dispatch, gemm_grouped and combine compute together, in two launches, for the up
to FEW_TOKENS tokens that a serving step or a draft has. Nothing is copied to
the host. All calls are asynchronous on `stream` (default: torch's current
stream) and raise KebabError on a refusal.
"""
import ctypes as c

import torch

from . import lib
from ._call import CODES, bad, call, dense, elsewhere, on, pitch, tensor

FEW_TOKENS = 16  # KEBAB_FEW_TOKENS
_FLOATS, _F32, _I8 = (torch.float16, torch.bfloat16), (torch.float32,), (torch.int8,)


def _layer(what, x, router, w_in, in_scale, w_out, out_scale, k, renormalize, stream):
    dev = tensor(what, "x", x, 2, _FLOATS)
    i8 = in_scale is not None
    T, H = x.shape
    if T > FEW_TOKENS:
        raise bad("%s: %d tokens are more than %d" % (what, T, FEW_TOKENS))
    tensor(what, "router", router, 2, _F32, dev)
    E = router.shape[0]
    dense(what, "router", router, (E, H), _F32, dev)
    tensor(what, "w_out", w_out, 3, _I8 if i8 else (x.dtype,), dev)
    D = w_out.shape[2]
    dense(what, "w_in", w_in, (E, 2 * D, H), _I8 if i8 else (x.dtype,), dev)
    dense(what, "w_out", w_out, (E, H, D), _I8 if i8 else (x.dtype,), dev)
    if i8:
        dense(what, "in_scale", in_scale, (E, 2 * D), _F32, dev)
        dense(what, "out_scale", out_scale, (E, H), _F32, dev)
    if not isinstance(k, int) or not 1 <= k <= min(E, 32):
        raise bad("%s: k = %s is not in 1..%d" % (what, k, min(E, 32)))
    if elsewhere(dev, stream):
        with on(dev, stream):
            return _layer(what, x, router, w_in, in_scale, w_out, out_scale, k, renormalize, None)
    size = workspace(T, E, k, H, D)
    if size < 0:
        raise bad("%s: invalid dimensions E=%d H=%d D=%d" % (what, E, H, D))
    y = x.new_empty((T, H))
    ws = x.new_empty((size,), dtype=torch.uint8)
    weights = ((w_in.data_ptr(), in_scale.data_ptr(), w_out.data_ptr(), out_scale.data_ptr()) if i8 else
               (w_in.data_ptr(), w_out.data_ptr()))
    call("kebab_expert_layer_i8" if i8 else "kebab_expert_layer", dev, CODES[x.dtype], x.data_ptr(), pitch(x),
         router.data_ptr(), *weights, y.data_ptr(), H, T, E, k, 1 if renormalize else 0, H, D, ws.data_ptr(), size)
    return y


_workspace = None


def workspace(T, E, k, H, D):
    """kebab_expert_layer_workspace: negative for sizes that a call refuses."""
    global _workspace
    if _workspace is None:
        f = lib().kebab_expert_layer_workspace
        f.argtypes, f.restype = [c.c_int64, c.c_int64, c.c_int, c.c_int64, c.c_int64], c.c_int64
        _workspace = f
    return _workspace(T, E, k, H, D)


def expert_layer(x, router, w_in, w_out, k, renormalize=True, stream=None):
    """y [T, H] of x's type (F16 or BF16) from x [T, H], T <= FEW_TOKENS, router
    [E, H] (float32), w_in [E, 2 D, H] (gate rows, then up rows) and w_out [E,
    H, D] of x's type, all contiguous but x. What is between the products stays
    in 32 bits."""
    return _layer("expert_layer", x, router, w_in, None, w_out, None, k, renormalize, stream)


def expert_layer_i8(x, router, w_in, in_scale, w_out, out_scale, k, renormalize=True, stream=None):
    """expert_layer with experts in 8-bit integers, the codes and scales of
    quantize_i8: in_scale [E, 2 D], out_scale [E, H]. x and the hidden values are
    quantised by row in the call."""
    what = "expert_layer_i8"
    for name, t in (("in_scale", in_scale), ("out_scale", out_scale)):
        if not isinstance(t, torch.Tensor):
            raise bad("%s: %s must be a CUDA tensor" % (what, name))
    return _layer(what, x, router, w_in, in_scale, w_out, out_scale, k, renormalize, stream)
