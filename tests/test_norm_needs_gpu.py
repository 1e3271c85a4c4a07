"""The norm's gradients one without the other: those of the full call, and what autograd asks for."""
import pytest

from operator_util import assert_within, dtype_of, pitched, randn
from test_norm_gpu import f32_error

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,H", [(0, 64), (1, 8192), (5, 64), (70, 1001), (300, 8191), (300, 10240), (9, 20000), (2000, 256)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("residual", [False, True])
def test_one_gradient_alone(cuda, T, H, dtype, residual):
    import torch
    import kebab_b200 as kb
    dt = dtype_of(dtype)
    s, dy, w = randn((T, H), dt, 1), randn((T, H), dt, 2), randn((H,), torch.float32, 3)
    ds = randn((T, H), dt, 4) if residual else None
    pitch = lambda t: pitched(t, 3, 1)  # noqa: E731
    for form in (torch.clone, pitch) if T else (torch.clone,):
        args = form(dy), form(s), w, 1e-6, None if ds is None else form(ds)
        dx, dw = kb.rms_norm_backward(*args)
        a, none = kb.rms_norm_backward(*args, need=(True, False))
        assert none is None and torch.equal(a, dx)
        none, b = kb.rms_norm_backward(*args, need=(False, True))
        if form is pitch:
            # Without dx, which is contiguous, all rows start alike and another kernel takes them, whose sums have another
            # order: both are within the norm's error of each term and T additions of the exact sum.
            assert none is None
            off = 2 * (f32_error(H) + T * 2.0 ** -24)
            rstd = (s.double().square().mean(1, keepdim=True) + 1e-6).rsqrt()
            assert_within(b, dw, off * (dy.double() * s.double() * rstd).abs().sum(0))
        else:
            assert none is None and torch.equal(b, dw)
        assert kb.rms_norm_backward(*args, need=(False, False)) == (None, None)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("frozen", ["weight", "rows"])
def test_frozen(cuda, monkeypatch, frozen, residual):
    """A frozen weight, or frozen rows: the others' gradients are those of all, and nothing else is asked for."""
    import torch
    import kebab_b200 as kb
    from kebab_b200.moe import rms_norm
    x, r, w = randn((30, 128), torch.bfloat16, 1), randn((30, 128), torch.bfloat16, 2), randn((128,), torch.float32, 3)
    asked, whole = [], kb.rms_norm_backward
    monkeypatch.setattr(kb, "rms_norm_backward", lambda *a, **k: asked.append(k.get("need")) or whole(*a, **k))

    def grads(rows, weight):
        a, b, c = x.clone().requires_grad_(rows), r.clone().requires_grad_(rows), w.clone().requires_grad_(weight)
        y, s = rms_norm(a, c, b if residual else None)
        (y.float().square().sum() + (s.float().sum() if residual else 0)).backward()
        return a.grad, b.grad, c.grad

    full, part = grads(True, True), grads(frozen != "rows", frozen != "weight")
    assert [tuple(n) for n in asked] == [(True, True), (frozen != "rows", frozen != "weight")]
    for i, (a, b) in enumerate(zip(full, part)):
        if (i == 2) == (frozen == "weight") or a is None:
            assert b is None
        else:
            assert torch.equal(a, b)
