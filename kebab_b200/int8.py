"""Products in 8-bit integers with one scale a token and one an output channel
(C ABI: include/kebab/int8.h).

    q[m, k] = rint(X[m, k] * (127 / amax_m)), scale[m] = amax_m / 127
    Y[m, n] = scale[m] * w_scale[n] * sum_k q[m, k] * Wq[n, k]  (+ bias[n])

Tokens are rows: X is [M, K], Wq [N, K] (int8; experts: [E, N, K]), Y [M, N].
Weights are quantised once with quantize_i8(W), activations in every call of
linear_i8 / linear_grouped_i8. All calls are asynchronous on `stream` (default:
torch's current stream) and raise KebabError on a refusal.
"""
import torch

from ._call import CODES, bad, call, dense, on, pitch, stacked, tensor

_FLOATS = (torch.float16, torch.bfloat16)
_ANY = (torch.float16, torch.bfloat16, torch.float32)
_I8, _F32, _I32 = (torch.int8,), (torch.float32,), (torch.int32,)


def quantize_i8(X, stream=None):
    """Quantises the rows of X ([..., K], F16, BF16 or F32) -> (int8 codes of
    X's shape, float32 scales of its leading shape)."""
    what = "quantize_i8"
    if isinstance(X, torch.Tensor) and X.dim() != 2:
        if X.dim() == 0:
            raise bad("quantize_i8: X must have at least one dimension")
        q, scale = quantize_i8(X.reshape(-1, X.shape[-1]), stream)
        return q.view(X.shape), scale.view(X.shape[:-1])
    dev = tensor(what, "X", X, 2, _ANY)
    M, K = X.shape
    with on(dev, stream):
        q = torch.empty((M, K), dtype=torch.int8, device=X.device)
        scale = torch.empty((M,), dtype=torch.float32, device=X.device)
        call("kebab_quantize_i8", CODES[X.dtype], X.data_ptr(), pitch(X), q.data_ptr(), K, scale.data_ptr(), M, K)
    return q, scale


def _output(what, Y, M, N, dtype, device, dev):
    if Y is None:
        return torch.empty((M, N), dtype=dtype, device=device)
    tensor(what, "Y", Y, 2, (dtype,), dev)
    if tuple(Y.shape) != (M, N):
        raise bad("%s: Y must be [%d, %d], got %s" % (what, M, N, tuple(Y.shape)))
    return Y


def _weights(what, Wq, w_scale, K, dim, dev):
    tensor(what, "Wq", Wq, dim, _I8, dev)
    if Wq.shape[-1] != K:
        raise bad("%s: inner dimensions differ: X has %d, Wq %d" % (what, K, Wq.shape[-1]))
    dense(what, "w_scale", w_scale, Wq.shape[:-1], _F32, dev)


def gemm_i8(q, scale, Wq, w_scale, bias=None, dtype=torch.bfloat16, Y=None, stream=None):
    """Y [M, N] (F16 or BF16) from codes q [M, K] and Wq [N, K]."""
    what = "gemm_i8"
    if dtype not in _FLOATS:
        raise bad("gemm_i8: dtype must be float16 or bfloat16")
    dev = tensor(what, "q", q, 2, _I8)
    (M, K), N = q.shape, Wq.shape[0]
    dense(what, "scale", scale, (M,), _F32, dev)
    _weights(what, Wq, w_scale, K, 2, dev)
    if bias is not None:
        dense(what, "bias", bias, (N,), (dtype,), dev)
    with on(dev, stream):
        Y = _output(what, Y, M, N, dtype, q.device, dev)
        call("kebab_gemm_i8", CODES[dtype], q.data_ptr(), pitch(q), scale.data_ptr(), Wq.data_ptr(), pitch(Wq),
             w_scale.data_ptr(), None if bias is None else bias.data_ptr(), Y.data_ptr(), pitch(Y), M, N, K)
    return Y


def gemm_grouped_i8(q, scale, Wq, w_scale, offsets, dtype=torch.bfloat16, Y=None, stream=None):
    """Y[r] from q[r] and the expert e of row r: Wq [E, N, K], w_scale [E, N],
    offsets [E + 1] (int32, on the device; see gemm_grouped)."""
    what = "gemm_grouped_i8"
    if dtype not in _FLOATS:
        raise bad("gemm_grouped_i8: dtype must be float16 or bfloat16")
    dev = tensor(what, "q", q, 2, _I8)
    (R, K), (E, N) = q.shape, Wq.shape[:2]
    dense(what, "scale", scale, (R,), _F32, dev)
    _weights(what, Wq, w_scale, K, 3, dev)
    dense(what, "offsets", offsets, (E + 1,), _I32, dev)
    with on(dev, stream):
        Y = _output(what, Y, R, N, dtype, q.device, dev)
        call("kebab_gemm_grouped_i8", CODES[dtype], q.data_ptr(), pitch(q), scale.data_ptr(), Wq.data_ptr(),
             *stacked(Wq), w_scale.data_ptr(), Y.data_ptr(), pitch(Y), offsets.data_ptr(), E, R, N, K)
    return Y


def _linear(what, X, Wq, w_scale, bias, offsets, Y, stream):
    dev = tensor(what, "X", X, 2, _FLOATS)
    (M, K), N = X.shape, Wq.shape[-2]
    grouped = offsets is not None
    _weights(what, Wq, w_scale, K, 3 if grouped else 2, dev)
    if bias is not None:
        dense(what, "bias", bias, (N,), (X.dtype,), dev)
    if grouped:
        dense(what, "offsets", offsets, (Wq.shape[0] + 1,), _I32, dev)
    ldw, w_stride = stacked(Wq) if grouped else (pitch(Wq), 0)
    with on(dev, stream):
        Y = _output(what, Y, M, N, X.dtype, X.device, dev)
        size = M * ((K + 15) // 16 * 16 + 4)
        ws = torch.empty((size,), dtype=torch.uint8, device=X.device)
        call("kebab_linear_i8", CODES[X.dtype], X.data_ptr(), pitch(X), Wq.data_ptr(), ldw, w_stride,
             w_scale.data_ptr(), None if bias is None else bias.data_ptr(), Y.data_ptr(), pitch(Y),
             offsets.data_ptr() if grouped else None, Wq.shape[0] if grouped else 1, M, N, K, ws.data_ptr(), size)
    return Y


def linear_i8(X, Wq, w_scale, bias=None, Y=None, stream=None):
    """Y [M, N] of X's type: X [M, K] is quantised by row and multiplied with
    the quantised weights Wq [N, K], w_scale [N]."""
    return _linear("linear_i8", X, Wq, w_scale, bias, None, Y, stream)


def linear_grouped_i8(X, Wq, w_scale, offsets, Y=None, stream=None):
    """linear_i8 grouped by expert: Wq [E, N, K], w_scale [E, N]; the rows
    offsets[e] .. offsets[e + 1] - 1 of X take expert e."""
    if not isinstance(offsets, torch.Tensor):
        raise bad("linear_grouped_i8: offsets must be a CUDA tensor")
    return _linear("linear_grouped_i8", X, Wq, w_scale, None, offsets, Y, stream)
