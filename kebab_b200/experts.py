"""Operators of a mixture-of-experts layer (C ABI: include/kebab/experts.h).

    routing = route(logits, k)                       # weights, experts, plan
    xs = dispatch(x, routing.slots)                  # tokens to expert order
    ys = gemm_grouped(xs, W, routing.offsets)        # ys[r] = xs[r] W_e
    y = combine(ys, routing.slots, routing.weights)  # back to tokens

Tokens are rows and matrices are row-major torch tensors. Nothing is copied to
the host: the ragged sizes stay on the device in `offsets`. All calls are
asynchronous on `stream` (default: torch's current stream) and raise KebabError
on a refusal. kebab_b200.moe has the same as differentiable functions.
"""
from typing import NamedTuple

import torch

from ._call import CODES, bad, call, dense, elsewhere, on, pitch, stacked, tensor

_FLOATS = (torch.float16, torch.bfloat16)
_ANY = (torch.float16, torch.bfloat16, torch.float32)
_F32, _I32 = (torch.float32,), (torch.int32,)
_ONE_BLOCK, _BLOCKS = 128, 148  # kebab_route_workspace


class Routing(NamedTuple):
    """Of T tokens over E experts: weights [T, k] float32, experts [T, k]
    int32, offsets [E + 1] int32 (choices of lower experts), slots [T, k] int32
    (places of the choices sorted by expert)."""
    weights: torch.Tensor
    experts: torch.Tensor
    offsets: torch.Tensor
    slots: torch.Tensor


def route(logits, k, renormalize=True, stream=None):
    """Top-k routing of logits [T, E] (F16, BF16 or F32): the k largest logits
    of each token (equal ones: the lower expert first), with the softmax over
    them (renormalize) or over all E as weights, and the sort by expert."""
    dev = tensor("route", "logits", logits, 2, _ANY)
    if elsewhere(dev, stream):
        with on(dev, stream):
            return route(logits, k, renormalize)
    T, E = logits.shape
    if not 1 <= k <= E:
        raise bad("route: k = %s is not in 1..%d" % (k, E))
    weights = logits.new_empty((T, k), dtype=torch.float32)
    experts, slots = logits.new_empty((2, T, k), dtype=torch.int32).unbind(0)
    offsets = logits.new_empty((E + 1,), dtype=torch.int32)
    size = 0 if T <= _ONE_BLOCK else 4 * _BLOCKS * E
    ws = logits.new_empty((size,), dtype=torch.uint8) if size else None
    call("kebab_route", dev, CODES[logits.dtype], logits.data_ptr(), pitch(logits), T, E, k, 1 if renormalize else 0,
         weights.data_ptr(), experts.data_ptr(), offsets.data_ptr(), slots.data_ptr(), ws.data_ptr() if size else None,
         size)
    return Routing(weights, experts, offsets, slots)


def route_backward(logits, routing, dweights, renormalize=True, stream=None):
    """Gradient of the logits (of their type) from the weights' [T, k]."""
    what = "route_backward"
    dev = tensor(what, "logits", logits, 2, _ANY)
    T, E = logits.shape
    k = routing.experts.shape[-1]
    dense(what, "routing.weights", routing.weights, (T, k), _F32, dev)
    dense(what, "routing.experts", routing.experts, (T, k), _I32, dev)
    dense(what, "dweights", dweights, (T, k), _F32, dev)
    if elsewhere(dev, stream):
        with on(dev, stream):
            return route_backward(logits, routing, dweights, renormalize)
    d = logits.new_empty((T, E))
    call("kebab_route_backward", dev, CODES[logits.dtype], logits.data_ptr(), pitch(logits), T, E, k,
         1 if renormalize else 0, routing.weights.data_ptr(), routing.experts.data_ptr(), dweights.data_ptr(),
         d.data_ptr(), E)
    return d


def _check_slots(what, slots, dev, T=None):
    """(T, k) of slots, whose tokens are T if that is given."""
    tensor(what, "slots", slots, 2, _I32, dev)
    shape = tuple(slots.shape)
    if not slots.is_contiguous() or (T is not None and shape[0] != T):
        raise bad("%s: slots must be a contiguous tensor of [%s, k], got %s" % (what, "T" if T is None else T, shape))
    return shape


def dispatch(x, slots, rows=None, stream=None):
    """xs[slots[t, j]] = x[t]: x [T, H] -> xs [rows, H] (default T * k rows). A
    slot outside [0, rows) is a dropped choice; rows that no slot names are
    not written."""
    what = "dispatch"
    dev = tensor(what, "x", x, 2, _FLOATS)
    T, H = x.shape
    k = _check_slots(what, slots, dev, T)[1]
    if elsewhere(dev, stream):
        with on(dev, stream):
            return dispatch(x, slots, rows)
    rows = T * k if rows is None else rows
    if rows < 0:
        raise bad("dispatch: rows = %s is negative" % rows)
    xs = x.new_empty((rows, H))
    call("kebab_expert_dispatch", dev, CODES[x.dtype], x.data_ptr(), pitch(x), slots.data_ptr(), xs.data_ptr(), H, T, k,
         rows, H)
    return xs


def combine(ys, slots, weights=None, stream=None):
    """y[t] = sum_j weights[t, j] ys[slots[t, j]] -> [T, H]; without weights
    the plain sum, which is the gradient of dispatch."""
    what = "combine"
    dev = tensor(what, "ys", ys, 2, _FLOATS)
    R, H = ys.shape
    T, k = _check_slots(what, slots, dev)
    if weights is not None:
        dense(what, "weights", weights, (T, k), _F32, dev)
    if elsewhere(dev, stream):
        with on(dev, stream):
            return combine(ys, slots, weights)
    y = ys.new_empty((T, H))
    call("kebab_expert_combine", dev, CODES[ys.dtype], ys.data_ptr(), pitch(ys), slots.data_ptr(),
         None if weights is None else weights.data_ptr(), y.data_ptr(), H, T, k, R, H)
    return y


def combine_backward(dy, ys, slots, weights, stream=None):
    """Gradients of combine -> (dys [R, H], dweights [T, k] float32). Rows of
    dys that no slot names are not written."""
    what = "combine_backward"
    dev = tensor(what, "dy", dy, 2, _FLOATS)
    T, H = dy.shape
    tensor(what, "ys", ys, 2, (dy.dtype,), dev)
    R = ys.shape[0]
    if ys.shape[1] != H:
        raise bad("combine_backward: dy has rows of %d, ys of %d" % (H, ys.shape[1]))
    k = _check_slots(what, slots, dev, T)[1]
    dense(what, "weights", weights, (T, k), _F32, dev)
    if elsewhere(dev, stream):
        with on(dev, stream):
            return combine_backward(dy, ys, slots, weights)
    dys, dweights = dy.new_empty((R, H)), dy.new_empty((T, k), dtype=torch.float32)
    call("kebab_expert_combine_backward", dev, CODES[dy.dtype], dy.data_ptr(), pitch(dy), ys.data_ptr(), pitch(ys),
         slots.data_ptr(), weights.data_ptr(), dys.data_ptr(), H, dweights.data_ptr(), T, k, R, H)
    return dys, dweights


def _mode(what, opmode):
    m = opmode.upper() if isinstance(opmode, str) else opmode
    if m not in ("RC", "RR"):
        raise bad("%s: opmode must be RC or RR, got %s" % (what, opmode))
    return m


def gemm_grouped(X, W, offsets, Y=None, opmode="RC", stream=None):
    """Y[r] = X[r] W_e for the rows offsets[e] <= r < offsets[e + 1] of expert
    e: X [R, K], offsets [E + 1] (int32, on the device), W [E, N, K] ("RC": the
    K x N matrices column-major) or [E, K, N] ("RR"); Y [R, N]. Rows of no
    expert are not written. The gradient of X is
    gemm_grouped(dY, W, offsets, opmode=the other)."""
    what = "gemm_grouped"
    m = _mode(what, opmode)
    dev = tensor(what, "X", X, 2, _FLOATS)
    R, K = X.shape
    tensor(what, "W", W, 3, (X.dtype,), dev)
    E, N, Kw = W.shape if m == "RC" else (W.shape[0], W.shape[2], W.shape[1])
    if Kw != K:
        raise bad("gemm_grouped: inner dimensions differ: X has %d, W %d" % (K, Kw))
    dense(what, "offsets", offsets, (E + 1,), _I32, dev)
    if Y is not None:
        tensor(what, "Y", Y, 2, (X.dtype,), dev)
        if Y.shape != (R, N):
            raise bad("gemm_grouped: Y must be [%d, %d], got %s" % (R, N, tuple(Y.shape)))
    if elsewhere(dev, stream):
        with on(dev, stream):
            return gemm_grouped(X, W, offsets, Y, m)
    Y = X.new_empty((R, N)) if Y is None else Y
    ldw, w_stride = stacked(W)
    call("kebab_gemm_grouped", dev, CODES[X.dtype], X.data_ptr(), pitch(X), W.data_ptr(), ldw, w_stride, Y.data_ptr(),
         pitch(Y), offsets.data_ptr(), E, R, N, K, m.encode())
    return Y


def gemm_grouped_dw(X, dY, offsets, dW=None, opmode="RC", stream=None):
    """The gradient of W: dW[e] = the sum over the expert's rows of dY[r, n]
    X[r, k], [E, N, K] ("RC") or [E, K, N] ("RR"); zeros for an expert without
    rows."""
    what = "gemm_grouped_dw"
    m = _mode(what, opmode)
    dev = tensor(what, "X", X, 2, _FLOATS)
    R, K = X.shape
    tensor(what, "dY", dY, 2, (X.dtype,), dev)
    if dY.shape[0] != R:
        raise bad("gemm_grouped_dw: X has %d rows, dY %d" % (R, dY.shape[0]))
    N = dY.shape[1]
    tensor(what, "offsets", offsets, 1, _I32, dev)
    E = offsets.shape[0] - 1
    if E < 1:
        raise bad("gemm_grouped_dw: offsets must have E + 1 values for E >= 1 experts")
    shape = (E, N, K) if m == "RC" else (E, K, N)
    if dW is not None:
        dense(what, "dW", dW, shape, (X.dtype,), dev)
    if elsewhere(dev, stream):
        with on(dev, stream):
            return gemm_grouped_dw(X, dY, offsets, dW, m)
    dW = X.new_empty(shape) if dW is None else dW
    call("kebab_gemm_grouped_dw", dev, CODES[X.dtype], X.data_ptr(), pitch(X), dY.data_ptr(), pitch(dY), dW.data_ptr(),
         offsets.data_ptr(), E, R, N, K, m.encode())
    return dW
