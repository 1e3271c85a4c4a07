"""A mixture-of-experts feed-forward layer on the framework's operators, in
training and in serving.

    layer = MoE(width, hidden, experts, k, dtype)   # trains with autograd
    y, routing = layer(x)
    served = layer.quantize()                       # 8-bit integer experts, forward only
    y = served(x)

The layer is y[t] = sum_j w[t, j] W2_e (silu(Wg_e x[t]) * Wu_e x[t]) over the k
experts e = e[t, j] that its router picks. `route`, `dispatch`, `combine` and
`grouped_linear` below are the operators as functions with a first gradient; a
second one raises (their backwards are calls that autograd does not see).
Nothing is copied to the host in a step: the ragged sizes stay on the device.

`python -m kebab_b200.moe` trains a small layer on a synthetic task and then
serves single tokens with its experts quantised.
"""
import argparse
import sys

import torch
from torch.autograd.function import once_differentiable

import kebab_b200 as kb


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, renormalize):
        logits = _rows(logits)
        r = kb.route(logits, k, renormalize)
        ctx.save_for_backward(logits, *r)
        ctx.renormalize = renormalize
        ctx.mark_non_differentiable(r.experts, r.offsets, r.slots)
        return tuple(r)

    @staticmethod
    @once_differentiable
    def backward(ctx, dweights, *_):
        logits, *r = ctx.saved_tensors
        return kb.route_backward(logits, kb.Routing(*r), dweights.contiguous(), ctx.renormalize), None, None


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, slots):
        ctx.save_for_backward(slots)
        return kb.dispatch(_rows(x), slots)

    @staticmethod
    @once_differentiable
    def backward(ctx, dxs):
        (slots,) = ctx.saved_tensors
        return kb.combine(_rows(dxs), slots), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ys, slots, weights):
        ys = _rows(ys)
        ctx.save_for_backward(ys, slots, weights)
        return kb.combine(ys, slots, weights)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        dys, dweights = kb.combine_backward(_rows(dy), *ctx.saved_tensors)
        return dys, None, dweights


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, offsets):
        x = _rows(x)
        ctx.save_for_backward(x, w, offsets)
        return kb.gemm_grouped(x, w, offsets)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, offsets = ctx.saved_tensors
        dy = _rows(dy)
        dx = kb.gemm_grouped(dy, w, offsets, opmode="RR") if ctx.needs_input_grad[0] else None
        dw = kb.gemm_grouped_dw(x, dy, offsets) if ctx.needs_input_grad[1] else None
        return dx, dw, None


def _rows(t):
    """`t` with contiguous rows that do not overlap (gradients of a sum are
    expanded: rows of stride 0)."""
    return t if t.stride(-1) == 1 and (t.stride(0) >= t.shape[-1] or t.shape[0] == 1) else t.contiguous()


def route(logits, k, renormalize=True):
    """kb.route, differentiable in the logits through the weights."""
    return kb.Routing(*_Route.apply(logits, k, renormalize))


def dispatch(x, slots):
    """kb.dispatch for slots that are a permutation (as route gives), differentiable in x."""
    return _Dispatch.apply(x, slots)


def combine(ys, slots, weights):
    """kb.combine, differentiable in ys (for slots that name every row of it) and weights."""
    return _Combine.apply(ys, slots, weights)


def grouped_linear(x, w, offsets):
    """kb.gemm_grouped with w [E, N, K], differentiable in x and w (for offsets
    that cover every row of x)."""
    return _GroupedLinear.apply(x, w, offsets)


def _gated(h):
    gate, up = h.chunk(2, dim=-1)
    return torch.nn.functional.silu(gate) * up


class MoE(torch.nn.Module):
    """width -> width through `experts` feed-forward networks of `hidden`, `k` a token."""

    def __init__(self, width, hidden, experts, k, dtype=torch.bfloat16, renormalize=True, device="cuda"):
        super().__init__()
        self.k, self.renormalize = k, renormalize
        make = lambda *shape: torch.nn.Parameter(  # noqa: E731
            torch.randn(shape, device=device, dtype=torch.float32).mul_(shape[-1] ** -0.5).to(dtype))
        self.router = torch.nn.Parameter(torch.randn((experts, width), device=device) * width ** -0.5)
        self.w_in = make(experts, 2 * hidden, width)  # gate rows, then up rows
        self.w_out = make(experts, width, hidden)

    def forward(self, x):
        r = route(x.float() @ self.router.T, self.k, self.renormalize)
        h = _gated(grouped_linear(dispatch(x, r.slots), self.w_in, r.offsets))
        return combine(grouped_linear(h, self.w_out, r.offsets), r.slots, r.weights), r

    def quantize(self):
        return QuantizedMoE(self)


class QuantizedMoE:
    """A trained MoE for serving, its experts' weights in 8-bit integers with a
    scale for each output channel; activations are quantised in each call."""

    def __init__(self, layer):
        self.k, self.renormalize = layer.k, layer.renormalize
        self.router = layer.router.detach()
        self.w_in, self.w_out = kb.quantize_i8(layer.w_in.detach()), kb.quantize_i8(layer.w_out.detach())

    def __call__(self, x):
        r = kb.route(x.float() @ self.router.T, self.k, self.renormalize)
        h = _gated(kb.linear_grouped_i8(kb.dispatch(x, r.slots), *self.w_in, r.offsets))
        return kb.combine(kb.linear_grouped_i8(h, *self.w_out, r.offsets), r.slots, r.weights)


def demo(width=64, hidden=128, experts=8, k=2, tokens=2048, steps=60, lr=1e-2, seed=0):
    """Trains a layer to imitate a fixed random one; returns the losses and the
    relative distance of the quantised layer's output for single tokens."""
    torch.manual_seed(seed)
    target = MoE(width, hidden, experts, k)
    layer = MoE(width, hidden, experts, k)
    with torch.no_grad():
        layer.router.copy_(target.router)
    master = [p.detach().float().clone() for p in layer.parameters()]  # 32-bit copies for the optimiser
    opt = torch.optim.Adam(master, lr=lr)
    losses = []
    for _ in range(steps):
        x = torch.randn((tokens, width), device="cuda").bfloat16()
        with torch.no_grad():
            want = target(x)[0].float()
        loss = (layer(x)[0].float() - want).square().mean() / want.square().mean()
        loss.backward()
        for m, p in zip(master, layer.parameters()):
            m.grad, p.grad = p.grad.float(), None
        opt.step()
        with torch.no_grad():
            for m, p in zip(master, layer.parameters()):
                p.copy_(m)
        losses.append(loss.detach())
    served = layer.quantize()
    off = []
    with torch.no_grad():
        for _ in range(16):
            x = torch.randn((1, width), device="cuda").bfloat16()
            a, b = layer(x)[0].float(), served(x).float()
            off.append((a - b).norm() / a.norm())
    return [float(v) for v in losses], float(torch.stack(off).mean())


def main(argv=None):
    ap = argparse.ArgumentParser(description="Trains a small mixture-of-experts layer, then serves it quantised.")
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--tokens", type=int, default=2048)
    a = ap.parse_args(argv)
    losses, off = demo(steps=a.steps, tokens=a.tokens)
    for i in range(0, len(losses), max(1, len(losses) // 6)):
        print("step %3d  loss %.4f" % (i, losses[i]))
    print("step %3d  loss %.4f" % (len(losses) - 1, losses[-1]))
    print("single tokens, 8-bit experts against 16-bit: relative distance %.4f" % off)
    return 0


if __name__ == "__main__":
    sys.exit(main())
