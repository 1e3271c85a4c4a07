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

from ._call import CODES, bad, call, dense, elsewhere, on, pitch, stacked, tensor

_FLOATS = (torch.float16, torch.bfloat16)
_ANY = (torch.float16, torch.bfloat16, torch.float32)
_I8, _F32, _I32 = (torch.int8,), (torch.float32,), (torch.int32,)


def quantize_i8(X, stream=None):
    """Quantises the rows of X ([..., K], F16, BF16 or F32) -> (int8 codes of
    X's shape, float32 scales of its leading shape)."""
    if isinstance(X, torch.Tensor) and X.dim() != 2:
        if X.dim() == 0:
            raise bad("quantize_i8: X must have at least one dimension")
        if X.is_cuda and elsewhere(X.get_device(), stream):
            with on(X.get_device(), stream):  # reshape copies what cannot be viewed as rows: on the call's stream
                return quantize_i8(X)
        if X.shape[-1] == 0:
            raise bad("quantize_i8: rows of X must not be empty")
        q, scale = quantize_i8(X.reshape(-1, X.shape[-1]))
        return q.view(X.shape), scale.view(X.shape[:-1])
    dev = tensor("quantize_i8", "X", X, 2, _ANY)
    if elsewhere(dev, stream):
        with on(dev, stream):
            return quantize_i8(X)
    M, K = X.shape
    q, scale = X.new_empty((M, K), dtype=torch.int8), X.new_empty((M,), dtype=torch.float32)
    call("kebab_quantize_i8", dev, CODES[X.dtype], X.data_ptr(), pitch(X), q.data_ptr(), K, scale.data_ptr(), M, K)
    return q, scale


def _check_output(what, Y, M, N, dtype, dev):
    if Y is not None:
        tensor(what, "Y", Y, 2, (dtype,), dev)
        if Y.shape != (M, N):
            raise bad("%s: Y must be [%d, %d], got %s" % (what, M, N, tuple(Y.shape)))


def _check_weights(what, Wq, w_scale, K, dim, dev):
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
    M, K = q.shape
    dense(what, "scale", scale, (M,), _F32, dev)
    _check_weights(what, Wq, w_scale, K, 2, dev)
    N = Wq.shape[0]
    if bias is not None:
        dense(what, "bias", bias, (N,), (dtype,), dev)
    _check_output(what, Y, M, N, dtype, dev)
    if elsewhere(dev, stream):
        with on(dev, stream):
            return gemm_i8(q, scale, Wq, w_scale, bias, dtype, Y)
    Y = q.new_empty((M, N), dtype=dtype) if Y is None else Y
    call("kebab_gemm_i8", dev, CODES[dtype], q.data_ptr(), pitch(q), scale.data_ptr(), Wq.data_ptr(), pitch(Wq),
         w_scale.data_ptr(), None if bias is None else bias.data_ptr(), Y.data_ptr(), pitch(Y), M, N, K)
    return Y


def gemm_grouped_i8(q, scale, Wq, w_scale, offsets, dtype=torch.bfloat16, Y=None, stream=None):
    """Y[r] from q[r] and the expert e of row r: Wq [E, N, K], w_scale [E, N],
    offsets [E + 1] (int32, on the device; see gemm_grouped)."""
    what = "gemm_grouped_i8"
    if dtype not in _FLOATS:
        raise bad("gemm_grouped_i8: dtype must be float16 or bfloat16")
    dev = tensor(what, "q", q, 2, _I8)
    R, K = q.shape
    dense(what, "scale", scale, (R,), _F32, dev)
    _check_weights(what, Wq, w_scale, K, 3, dev)
    E, N = Wq.shape[:2]
    dense(what, "offsets", offsets, (E + 1,), _I32, dev)
    _check_output(what, Y, R, N, dtype, dev)
    if elsewhere(dev, stream):
        with on(dev, stream):
            return gemm_grouped_i8(q, scale, Wq, w_scale, offsets, dtype, Y)
    Y = q.new_empty((R, N), dtype=dtype) if Y is None else Y
    ldw, w_stride = stacked(Wq)
    call("kebab_gemm_grouped_i8", dev, CODES[dtype], q.data_ptr(), pitch(q), scale.data_ptr(), Wq.data_ptr(), ldw,
         w_stride, w_scale.data_ptr(), Y.data_ptr(), pitch(Y), offsets.data_ptr(), E, R, N, K)
    return Y


def _linear(what, X, Wq, w_scale, bias, offsets, Y, stream):
    dev = tensor(what, "X", X, 2, _FLOATS)
    M, K = X.shape
    if offsets is None:
        _check_weights(what, Wq, w_scale, K, 2, dev)
        N, E, off, ldw, w_stride = Wq.shape[0], 1, None, pitch(Wq), 0
    else:
        _check_weights(what, Wq, w_scale, K, 3, dev)
        E, N = Wq.shape[:2]
        dense(what, "offsets", offsets, (E + 1,), _I32, dev)
        off, (ldw, w_stride) = offsets.data_ptr(), stacked(Wq)
    if bias is not None:
        dense(what, "bias", bias, (N,), (X.dtype,), dev)
    _check_output(what, Y, M, N, X.dtype, dev)
    if elsewhere(dev, stream):
        with on(dev, stream):
            return _linear(what, X, Wq, w_scale, bias, offsets, Y, None)
    Y = X.new_empty((M, N)) if Y is None else Y
    size = M * ((K + 15) // 16 * 16 + 4)  # kebab_linear_i8_workspace
    ws = X.new_empty((size,), dtype=torch.uint8)
    call("kebab_linear_i8", dev, CODES[X.dtype], X.data_ptr(), pitch(X), Wq.data_ptr(), ldw, w_stride,
         w_scale.data_ptr(), None if bias is None else bias.data_ptr(), Y.data_ptr(), pitch(Y), off, E, M, N, K,
         ws.data_ptr(), size)
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
