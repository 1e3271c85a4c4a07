"""A mixture-of-experts feed-forward layer on the framework's operators, in
training and in serving.

    layer = MoE(width, hidden, experts, k, dtype)   # trains with autograd
    y, routing = layer(x)
    served = layer.quantize()                       # 8-bit integer experts, forward only
    y = served(x)
    served = layer.serve(bits)                      # 16, 8 or 4 bits; in 16 and 8 a few tokens take two launches

    block = Block(width, hidden, experts, k)        # the norm before the layer, on a residual stream
    y, stream, routing = block(x, stream)           # stream: the sum x + stream that was normed
    y, stream = block.serve(bits)(x, stream)

The layer is y[t] = sum_j w[t, j] W2_e (silu(Wg_e x[t]) * Wu_e x[t]) over the k
experts e = e[t, j] that its router picks. `route`, `dispatch`, `combine` and
`grouped_linear` below are the operators as functions with a first gradient; a
second one raises (their backwards are calls that autograd does not see).
Nothing is copied to the host in a step: the ragged sizes stay on the device.
To capture a training step into a CUDA graph, warm up on a side stream and let go
of every eager output and loss of the same parameters first: their accumulation
nodes belong to the eager stream, and a captured backward pass that reaches them
ends the process.

`python -m kebab_b200.moe` trains a small layer on a synthetic task and then
serves single tokens with its experts quantised; then two blocks, served in 16,
8 and 4 bits.
"""
import argparse
import sys

import torch
from torch.autograd.function import once_differentiable

import kebab_b200 as kb
from kebab_b200.layer import workspace


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


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        x = _rows(x)
        y, s = kb.rms_norm(x, weight, eps, residual=None if residual is None else _rows(residual))
        ctx.save_for_backward(s, weight)
        ctx.eps, ctx.added = eps, residual is not None
        ctx.set_materialize_grads(False)  # a stream that ends here has no gradient
        return (y, s) if ctx.added else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, ds=None):
        s, weight = ctx.saved_tensors
        if dy is None:
            dx, dweight = ds, None
        else:
            x, w, residual = ctx.needs_input_grad[:3]
            dx, dweight = kb.rms_norm_backward(_rows(dy), s, weight, ctx.eps, dresidual=None if ds is None else _rows(ds),
                                               need=(x or residual, w))
        return dx, dweight, dx if ctx.added else None, None


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


def rms_norm(x, weight, residual=None, eps=1e-6):
    """kb.rms_norm -> (y, s), differentiable in x, weight and the residual; s is x without a residual."""
    out = _RmsNorm.apply(x, weight, residual, eps)
    return (out, x) if residual is None else out


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

    def serve(self, bits=8):
        return ServedMoE(self, bits)


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


class ServedMoE:
    """A trained MoE for serving, its experts in 16 bits, in 8-bit integers or in
    4-bit floating point. Up to kb.FEW_TOKENS tokens through experts of 16 or 8
    bits take kb.expert_layer; more of them, 4 bits, what that does not take and
    large weights that it copies value by value take the separate operators."""

    # Values of the chosen experts' second matrices, at most, whose rows do not start on 16 bytes. us, the layer against
    # the separate operators: 8 bits, 2.1 million 53 and 58, 3.2 million 87 and 57, 131 million (D = 1000) 4654 and 165;
    # 16 bits, 8.4 million 73 and 129, 12.6 million 429 and 318, 134 million 4210 and 2548.
    _UNALIGNED = {16: 10_000_000, 8: 3_000_000}

    def __init__(self, layer, bits=8):
        self.k, self.renormalize, self.bits = layer.k, layer.renormalize, bits
        self.router = layer.router.detach()
        make = {16: lambda w: (w,), 8: kb.quantize_i8, 4: lambda w: (kb.quantize_f4(w),)}.get(bits)
        if make is None:
            raise kb.KebabError(kb.EINVAL, "ServedMoE: bits = %s is not 16, 8 or 4" % (bits,))
        self.w_in, self.w_out = make(layer.w_in.detach()), make(layer.w_out.detach())
        self.linear = {16: kb.gemm_grouped, 8: kb.linear_grouped_i8, 4: kb.linear_grouped_f4}[bits]
        if bits != 4:
            weights = self.w_in[0], self.w_out[0]
            E, H, D = weights[1].shape
            self.takes = all(t.is_contiguous() for t in weights) and workspace(1, E, self.k, H, D) > 0
            aligned = all(t.data_ptr() % 16 == 0 and t.shape[2] * t.element_size() % 16 == 0 for t in weights)
            self.unaligned = 0 if aligned else H * D  # values an expert

    def _few(self, tokens):
        """Whether kb.expert_layer takes a step of so many tokens."""
        return (self.bits != 4 and tokens <= kb.FEW_TOKENS and self.takes and
                min(tokens * self.k, len(self.router)) * self.unaligned <= self._UNALIGNED[self.bits])

    def __call__(self, x):
        if self._few(len(x)):
            few = kb.expert_layer if self.bits == 16 else kb.expert_layer_i8
            return few(x, self.router, *self.w_in, *self.w_out, self.k, self.renormalize)
        r = kb.route(x.float() @ self.router.T, self.k, self.renormalize)
        h = _gated(self.linear(kb.dispatch(x, r.slots), *self.w_in, r.offsets))
        return kb.combine(self.linear(h, *self.w_out, r.offsets), r.slots, r.weights)


class Block(torch.nn.Module):
    """The residual stream's addition and norm, and an MoE on the result."""

    def __init__(self, width, hidden, experts, k, dtype=torch.bfloat16, renormalize=True, device="cuda", eps=1e-6):
        super().__init__()
        self.eps = eps
        self.norm = torch.nn.Parameter(torch.ones(width, device=device))
        self.moe = MoE(width, hidden, experts, k, dtype, renormalize, device)

    def forward(self, x, stream=None):
        y, stream = rms_norm(x, self.norm, stream, self.eps)
        y, r = self.moe(y)
        return y, stream, r

    def serve(self, bits=8):
        return ServedBlock(self, bits)


class ServedBlock:
    """A trained Block for serving; see ServedMoE."""

    def __init__(self, block, bits=8):
        self.norm, self.eps, self.moe = block.norm.detach(), block.eps, block.moe.serve(bits)

    def __call__(self, x, stream=None):
        y, stream = kb.rms_norm(x, self.norm, self.eps, residual=stream)
        return self.moe(y), stream


def _through(blocks, x):
    """The residual stream after the blocks."""
    stream = None
    for b in blocks:
        x, stream = b(x, stream)[:2]
    return x + stream


def demo_blocks(width=64, hidden=128, experts=8, k=2, tokens=2048, steps=40, lr=1e-2, seed=0):
    """Trains two blocks to imitate two fixed random ones; returns the losses and,
    by bits, the relative distance of the served blocks' output for single tokens."""
    torch.manual_seed(seed)
    target = [Block(width, hidden, experts, k) for _ in range(2)]
    blocks = [Block(width, hidden, experts, k) for _ in range(2)]
    with torch.no_grad():
        for a, b in zip(blocks, target):
            a.moe.router.copy_(b.moe.router)
    params = [p for b in blocks for p in b.parameters()]
    master = [p.detach().float().clone() for p in params]  # 32-bit copies for the optimiser
    opt = torch.optim.Adam(master, lr=lr)
    losses = []
    for _ in range(steps):
        x = torch.randn((tokens, width), device="cuda").bfloat16()
        with torch.no_grad():
            want = _through(target, x).float()
        loss = (_through(blocks, x).float() - want).square().mean() / want.square().mean()
        loss.backward()
        for m, p in zip(master, params):
            m.grad, p.grad = p.grad.float(), None
        opt.step()
        with torch.no_grad():
            for m, p in zip(master, params):
                p.copy_(m)
        losses.append(loss.detach())
    off = {}
    with torch.no_grad():
        for bits in (16, 8, 4):
            served, d = [b.serve(bits) for b in blocks], []
            for _ in range(16):
                x = torch.randn((1, width), device="cuda").bfloat16()
                a, b = _through(blocks, x).float(), _through(served, x).float()
                d.append((a - b).norm() / a.norm())
            off[bits] = float(torch.stack(d).mean())
    return [float(v) for v in losses], off


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
    losses, off = demo_blocks(steps=a.steps, tokens=a.tokens)
    print("two blocks: loss %.4f -> %.4f" % (losses[0], losses[-1]))
    for bits, d in off.items():
        print("single tokens through the blocks, served in %d bits: relative distance %.4f" % (bits, d))
    return 0


if __name__ == "__main__":
    sys.exit(main())
