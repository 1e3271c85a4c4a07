"""The expert layer's autograd functions with the products in plain torch on
the CPU — no GPU."""
import pytest

import kebab_b200 as kb


@pytest.fixture
def stand_ins(monkeypatch):
    """kb's operators for one expert and one choice a token."""
    import torch

    def gemm_grouped(x, w, offsets, opmode="RC"):
        return x @ (w[0].T if opmode == "RC" else w[0])

    def route(logits, k, renormalize=True):
        T = logits.shape[0]
        at = torch.arange(T, dtype=torch.int32)[:, None]
        return kb.Routing(logits * logits, at * 0, torch.tensor([0, T], dtype=torch.int32), at)

    for name, f in (("gemm_grouped", gemm_grouped), ("gemm_grouped_dw", lambda x, dy, offsets: (dy.T @ x)[None]),
                    ("route", route), ("route_backward", lambda logits, r, dw, renormalize: 2 * logits * dw),
                    ("dispatch", lambda x, slots: x.clone()),
                    ("combine", lambda ys, slots, weights=None: ys * (1 if weights is None else weights)),
                    ("combine_backward", lambda dy, ys, slots, weights: (dy * weights, (dy * ys).sum(1, keepdim=True)))):
        monkeypatch.setattr(kb, name, f, raising=False)


def test_first_gradients_and_no_second_ones(stand_ins):
    """The backwards are calls that autograd does not see: a second gradient
    has to raise, and not to come back without its terms."""
    import torch
    from kebab_b200 import moe
    T, H = 5, 4
    x, w = torch.randn(T, H, requires_grad=True), torch.randn(1, H, H, requires_grad=True)
    logits = torch.randn(T, 1, requires_grad=True)
    r = moe.route(logits.detach(), 1)
    outs = {"route": (moe.route(logits, 1).weights, logits, 2 * logits),
            "dispatch": (moe.dispatch(x, r.slots), x, torch.ones(T, H)),
            "combine": (moe.combine(x, r.slots, r.weights), x, r.weights.expand(T, H)),
            "grouped_linear": (moe.grouped_linear(x, w, r.offsets), x, w[0].sum(0).expand(T, H))}
    for name, (y, at, want) in outs.items():
        (g,) = torch.autograd.grad(y.sum(), at, create_graph=True)
        assert torch.allclose(g, want), name
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.square().sum(), at)
            pytest.fail("a second gradient of %s came back" % name)
