"""The mixture-of-experts layer: its gradients against 64-bit autograd of the
same layer in elementary operations, and the train-then-serve example."""
import pytest

from operator_util import randn

pytestmark = pytest.mark.gpu


def plain(x, router, w_in, w_out, k, renormalize):
    import torch
    logits = x @ router.T
    order = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
    p = torch.softmax(torch.gather(logits, 1, order), 1) if renormalize else torch.gather(torch.softmax(logits, 1), 1, order)
    y = torch.zeros_like(x)
    for e in range(router.shape[0]):
        t, j = torch.nonzero(order == e, as_tuple=True)
        gate, up = (x[t] @ w_in[e].T).chunk(2, -1)
        y = y.index_add(0, t, p[t, j, None] * ((torch.nn.functional.silu(gate) * up) @ w_out[e].T))
    return y


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("tokens,width,hidden,experts,k", [(1, 64, 128, 4, 2), (37, 128, 64, 5, 1), (300, 256, 192, 9, 4)])
def test_gradients(cuda, tokens, width, hidden, experts, k, renormalize):
    """Each 16-bit rounding on the way (xs, h, the product's inputs and outputs
    and their gradients: at most 12 of 2^-11) moves a result by its own size;
    against the norm of the whole gradient 24 * 2^-11 bounds their sum, with
    a factor of 2 for the cancellation in sums of signed terms."""
    import torch
    from kebab_b200.moe import MoE
    torch.manual_seed(tokens)
    layer = MoE(width, hidden, experts, k, torch.float16, renormalize)
    x = randn((tokens, width), torch.float16, 1).requires_grad_()
    y, r = layer(x)
    dy = randn((tokens, width), torch.float16, 2)
    y.backward(dy)
    params = [x, layer.router, layer.w_in, layer.w_out]
    exact = [p.detach().double().requires_grad_() for p in params]
    want = plain(*exact, k, renormalize)
    want.backward(dy.double())
    for name, got, ref in zip(("y", "x", "router", "w_in", "w_out"), [y] + [p.grad for p in params], [want] + [p.grad for p in exact]):
        assert got.shape == ref.shape
        if ref.norm() == 0:
            assert got.norm() == 0, name
        else:
            assert float((got.double() - ref).norm() / ref.norm()) < 24 * 2.0 ** -11, name
    assert int(r.offsets[-1]) == tokens * k


def test_expanded_gradients(cuda):
    """y.sum() sends a gradient whose rows all share their memory."""
    import torch
    from kebab_b200.moe import MoE
    layer = MoE(64, 64, 4, 2)
    x = randn((50, 64), torch.bfloat16, 1).requires_grad_()
    layer(x)[0].sum().backward()
    a = [p.grad.clone() for p in (x, layer.w_in, layer.w_out, layer.router)]
    for p in (x, layer.w_in, layer.w_out, layer.router):
        p.grad = None
    layer(x)[0].backward(torch.ones((50, 64), dtype=torch.bfloat16, device="cuda"))
    for u, p in zip(a, (x, layer.w_in, layer.w_out, layer.router)):
        assert torch.equal(u, p.grad)


def test_no_tokens(cuda):
    import torch
    from kebab_b200.moe import MoE
    layer = MoE(64, 64, 4, 2)
    x = torch.zeros((0, 64), dtype=torch.bfloat16, device="cuda", requires_grad=True)
    y, _ = layer(x)
    y.sum().backward()
    assert y.shape == (0, 64) and x.grad.shape == (0, 64) and (layer.w_in.grad == 0).all()
    assert layer.quantize()(x.detach()).shape == (0, 64)


def test_train_then_serve(cuda):
    """The loss falls well below its start, and 8-bit experts stay within a few
    roundings of 1/254 a value of the 16-bit ones."""
    from kebab_b200.moe import demo
    losses, off = demo(steps=40)
    assert losses[-1] < 0.5 * losses[0]
    assert off < 0.05
