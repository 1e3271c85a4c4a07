"""The norm and the expert layer together, trained and served."""
import pytest

from operator_util import randn
from test_moe_gpu import plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,width,hidden,experts,k", [(1, 64, 128, 4, 2), (37, 128, 64, 5, 1), (300, 256, 192, 9, 4)])
@pytest.mark.parametrize("stream", [False, True])
def test_block_gradients(cuda, tokens, width, hidden, experts, k, stream):
    """As the layer's own gradients: at most 16 roundings of 2^-11 on the way (the
    stream's sum, the normed tokens and their gradients are four more), with a
    factor of 2 for the cancellation in sums of signed terms."""
    import torch
    from kebab_b200.moe import Block
    torch.manual_seed(tokens)
    block = Block(width, hidden, experts, k, torch.float16)
    with torch.no_grad():
        block.norm.copy_(1 + 0.1 * torch.randn(width, device="cuda"))
    x = randn((tokens, width), torch.float16, 1).requires_grad_()
    res = randn((tokens, width), torch.float16, 3).requires_grad_() if stream else None
    dy, ds = randn((tokens, width), torch.float16, 2), randn((tokens, width), torch.float16, 4)
    y, s, _ = block(x, res)
    torch.autograd.backward([y, s], [dy, ds])
    params = [x] + ([res] if stream else []) + [block.norm, block.moe.router, block.moe.w_in, block.moe.w_out]
    exact = [p.detach().double().requires_grad_() for p in params]
    total = exact[0] + exact[1] if stream else exact[0]
    # The values are those of the stored sum, as the block takes them.
    total = total + (s.detach().double() - total.detach())
    n = total * (total.square().mean(1, keepdim=True) + block.eps).rsqrt() * exact[-4]
    want = plain(n, *exact[-3:], k, True)
    torch.autograd.backward([want, total], [dy.double(), ds.double()])
    for i, (got, ref) in enumerate(zip([y] + [p.grad for p in params], [want] + [p.grad for p in exact])):
        assert got.shape == ref.shape and (ref.norm() > 0 or got.norm() == 0), i
        if ref.norm() > 0:
            assert float((got.double() - ref).norm() / ref.norm()) < 32 * 2.0 ** -11, i


def test_norm_function(cuda):
    import torch
    import kebab_b200 as kb
    from kebab_b200 import moe
    x, r = (randn((9, 128), torch.bfloat16, i).requires_grad_() for i in (1, 2))
    w = randn((128,), torch.float32, 3).requires_grad_()
    y, s = moe.rms_norm(x, w, r)
    y.sum().backward()  # rows that share their memory; no gradient of s
    assert torch.equal(x.grad, r.grad)
    dx, dw = kb.rms_norm_backward(torch.ones_like(y), s.detach(), w.detach())
    assert torch.equal(x.grad, dx) and torch.equal(w.grad, dw)
    x.grad = r.grad = w.grad = None
    y, s = moe.rms_norm(x, w, r)
    s.sum().backward()  # the stream alone
    assert torch.equal(x.grad, torch.ones_like(x)) and torch.equal(r.grad, torch.ones_like(r)) and w.grad is None
    x.grad = None
    y, s = moe.rms_norm(x, w)
    assert s is x
    (y.sum() + s.sum()).backward()
    dx, _ = kb.rms_norm_backward(torch.ones_like(y), x.detach(), w.detach())
    assert torch.equal(x.grad, dx + 1)
    x.grad = None
    (g,) = torch.autograd.grad(moe.rms_norm(x, w)[0].sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.float().square().sum(), x)


@pytest.mark.parametrize("bits,near", [(16, 2.0 ** -6), (8, 0.05), (4, 0.5)])
@pytest.mark.parametrize("tokens", [0, 1, 16, 17, 100])
def test_served_blocks(cuda, bits, near, tokens):
    """A stack of blocks, served: 16 bits within a few roundings of 2^-8, 8 bits of 1/254, 4 bits of 1/4 of a value each."""
    import torch
    from kebab_b200.moe import Block
    torch.manual_seed(1)
    blocks = [Block(256, 128, 8, 2) for _ in range(2)]
    served = [b.serve(bits) for b in blocks]
    x = randn((tokens, 256), torch.bfloat16, 5)
    with torch.no_grad():
        a, b, sa, sb = x, x, None, None
        for p, q in zip(blocks, served):
            (a, sa, _), (b, sb) = p(a, sa), q(b, sb)
    assert b.shape == a.shape and sb.dtype == sa.dtype
    if tokens:
        total = (a + sa).float()
        assert float(((b + sb).float() - total).norm() / total.norm()) < near


def test_served_steps_captured(cuda):
    """A decode step of two blocks in a graph, replayed on new tokens; the 8-bit one beside it."""
    import torch
    from kebab_b200.moe import Block
    torch.manual_seed(2)
    served = [[Block(256, 128, 8, 2).serve(bits) for _ in range(2)] for bits in (16, 8, 4)]
    x = randn((3, 256), torch.bfloat16, 1)

    def step():
        out = []
        for blocks in served:
            y, s = x, None
            for b in blocks:
                y, s = b(y, s)
            out.append(y + s)
        return out

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (2, 3):
        x.copy_(randn((3, 256), torch.bfloat16, seed))
        graph.replay()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


def test_training_step_captured(cuda):
    """Forward and backward of a block in a graph, replayed."""
    import torch
    from kebab_b200.moe import Block
    torch.manual_seed(3)
    block = Block(128, 64, 4, 2)
    x, r = (randn((33, 128), torch.bfloat16, i) for i in (1, 2))
    dy = randn((33, 128), torch.bfloat16, 3)
    params = list(block.parameters())

    def step():
        y, s, _ = block(x, r)
        return torch.autograd.grad([y, s], params, [dy, dy])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (4, 5):
        x.copy_(randn((33, 128), torch.bfloat16, seed))
        graph.replay()
        want = step()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_demo(cuda):
    """The example runs, and its blocks' gradients are finite."""
    import math
    from kebab_b200.moe import demo_blocks
    losses, off = demo_blocks(steps=3, tokens=256)
    assert len(losses) == 3 and all(math.isfinite(v) for v in losses)
    assert set(off) == {16, 8, 4} and all(math.isfinite(v) for v in off.values())


def test_refusals(cuda):
    import kebab_b200 as kb
    from kebab_b200.moe import MoE
    with pytest.raises(kb.KebabError):
        MoE(64, 64, 4, 2).serve(5)
