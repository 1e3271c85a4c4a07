"""What the wrappers of the language-model operators share: the typed C
functions, checks of tensors, the stream and device of a call."""
import ctypes as c

import torch

from . import BF16, EINVAL, F16, F32, KebabError, lib
from . import check as _check

P, I, L, F = c.c_void_p, c.c_int, c.c_int64, c.c_float
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
    "kebab_rms_norm": [I, I, P, L, P, L, P, F, P, L, P, L, L, L, P],
    "kebab_rms_norm_i8": [I, I, P, L, P, L, P, F, P, L, P, L, P, L, P, L, L, P],
    "kebab_rms_norm_backward": [I, I, P, L, P, L, P, F, P, L, P, L, P, P, L, L, L, P],
    "kebab_quantize_f4": [I, P, L, L, P, P, L, L, L, P],
    "kebab_quantize_f4_tokens": [I, P, L, P, P, L, L, P],
    "kebab_dequantize_f4": [I, P, P, P, L, L, L, P],
    "kebab_gemm_f4": [I, P, P, P, P, P, P, L, L, L, L, P],
    "kebab_gemm_grouped_f4": [I, P, P, P, P, P, L, P, L, L, L, L, P],
    "kebab_linear_f4": [I, P, L, P, P, P, P, L, P, L, L, L, L, P, L, P],
    "kebab_expert_layer": [I, P, L, P, P, P, P, L, L, L, I, I, L, L, P, L, P],
    "kebab_expert_layer_i8": [I, P, L, P, P, P, P, P, P, L, L, L, I, I, L, L, P, L, P],
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
    if isinstance(t, torch.Tensor):
        at = t.get_device()
        if (at >= 0 and t.dim() == dim and t.dtype in dtypes and (device is None or at == device) and
                (t.stride(-1) == 1 or t.shape[-1] <= 1 or not t.numel())):
            return at
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise bad("%s: %s must be a CUDA tensor" % (what, name))
    if t.dim() != dim:
        raise bad("%s: %s must have %d dimension(s), got %s" % (what, name, dim, tuple(t.shape)))
    if t.dtype not in dtypes:
        raise bad("%s: %s has type %s" % (what, name, t.dtype))
    if device is not None and at != device:
        raise bad("%s: %s is on another device" % (what, name))
    raise bad("%s: rows of %s must be contiguous" % (what, name))


def dense(what, name, t, shape, dtypes, device):
    """As tensor(), of that very shape and contiguous throughout."""
    if (isinstance(t, torch.Tensor) and t.shape == shape and t.dtype in dtypes and t.get_device() == device and
            t.is_contiguous()):
        return
    tensor(what, name, t, len(shape), dtypes, device)
    raise bad("%s: %s must be a contiguous tensor of shape %s, got %s" % (what, name, tuple(shape), tuple(t.shape)))


def pitch(t):
    """Elements from one row to the next of the last two dimensions."""
    return t.stride(-2) if t.shape[-2] > 1 else t.shape[-1]


def stacked(t):
    """(row pitch, matrix pitch) of a stack of matrices."""
    ld = pitch(t)
    return ld, t.stride(0) if t.shape[0] > 1 else ld * t.shape[1]


_current_device = torch.cuda.current_device
# A stream's handle without a torch.cuda.Stream object around it: 0.1 us
# against 3.3 us, where a whole call takes about ten.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda device: torch.cuda.current_stream(device).cuda_stream)


def elsewhere(device, stream):
    """Whether a call has to run under on(): on a given stream, or on a device
    that is not the current one."""
    return stream is not None or _current_device() != device


def on(device, stream):
    """The context of a call on that device and stream: what the call
    allocates belongs to the stream."""
    if stream is None:
        return torch.cuda.device(device)
    if stream.device.index != device:
        raise bad("the stream belongs to another device than the tensors")
    return torch.cuda.stream(stream)


def call(name, device, *args):
    """Calls a C function with the current stream of `device`, the current device, last."""
    rc = (_functions.get(name) or function(name))(*args, _raw_stream(device))
    if rc:
        _check(rc)
