"""What the wrappers of the language-model operators share: the typed C
functions, checks of tensors, the stream and device of a call."""
import ctypes as c

import torch

from . import BF16, EINVAL, F16, F32, KebabError, lib
from . import check as _check

P, I, L = c.c_void_p, c.c_int, c.c_int64
_SIGNATURES = {
    "kebab_quantize_i8": [I, P, L, P, L, P, L, L, P],
    "kebab_gemm_i8": [I, P, L, P, P, L, P, P, P, L, L, L, L, P],
    "kebab_gemm_grouped_i8": [I, P, L, P, P, L, L, P, P, L, P, L, L, L, L, P],
    "kebab_linear_i8": [I, P, L, P, L, L, P, P, P, L, P, L, L, L, L, P, L, P],
    "kebab_route": [I, P, L, L, L, I, I, P, P, P, P, P, L, P],
    "kebab_route_backward": [I, P, L, L, L, I, I, P, P, P, P, L, P],
    "kebab_expert_dispatch": [I, P, L, P, P, L, L, I, L, L, P],
    "kebab_expert_combine": [I, P, L, P, P, P, L, L, I, L, L, P],
    "kebab_expert_combine_backward": [I, P, L, P, L, P, P, P, L, P, L, I, L, L, P],
    "kebab_gemm_grouped": [I, P, L, P, L, L, P, L, P, L, L, L, L, c.c_char_p, P],
    "kebab_gemm_grouped_dw": [I, P, L, P, L, P, P, L, L, L, L, c.c_char_p, P],
}
CODES = {torch.float16: F16, torch.bfloat16: BF16, torch.float32: F32}
_functions = {}


def function(name):
    f = _functions.get(name)
    if f is None:
        f = getattr(lib(), name)
        f.argtypes, f.restype = _SIGNATURES[name], c.c_int
        _functions[name] = f
    return f


def bad(msg):
    return KebabError(EINVAL, msg)


def tensor(what, name, t, dim, dtypes, device=None):
    """Checks that `t` is a CUDA tensor of that rank and type with contiguous
    rows, on `device` if given; returns its device index."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise bad("%s: %s must be a CUDA tensor" % (what, name))
    if t.dim() != dim:
        raise bad("%s: %s must have %d dimension(s), got %s" % (what, name, dim, tuple(t.shape)))
    if t.dtype not in dtypes:
        raise bad("%s: %s has type %s" % (what, name, t.dtype))
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise bad("%s: rows of %s must be contiguous" % (what, name))
    at = t.device.index
    if device is not None and at != device:
        raise bad("%s: %s is on another device" % (what, name))
    return at


def dense(what, name, t, shape, dtypes, device):
    """As tensor(), of that very shape and contiguous throughout."""
    tensor(what, name, t, len(shape), dtypes, device)
    if tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise bad("%s: %s must be a contiguous tensor of shape %s, got %s" % (what, name, tuple(shape), tuple(t.shape)))


def pitch(t):
    """Elements from one row to the next of the last two dimensions."""
    return t.stride(-2) if t.shape[-2] > 1 else t.shape[-1]


def stacked(t):
    """(row pitch, matrix pitch) of a stack of matrices."""
    ld = pitch(t)
    return ld, t.stride(0) if t.shape[0] > 1 else ld * t.shape[1]


class on:
    """Runs a call on a device and, where one is given, a stream: what the call
    allocates belongs to that stream."""

    def __new__(cls, device, stream):
        if stream is not None:
            if stream.device.index != device:
                raise bad("the stream belongs to another device than the tensors")
            return torch.cuda.stream(stream)
        if torch.cuda.current_device() != device:
            return torch.cuda.device(device)
        return _HERE


class _Here:
    def __enter__(self):
        return None

    def __exit__(self, *a):
        return False


_HERE = _Here()


def call(name, *args):
    """Calls a C function with the current stream of the current device last."""
    rc = function(name)(*args, torch.cuda.current_stream().cuda_stream)
    if rc:
        _check(rc)
