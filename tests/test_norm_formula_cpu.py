"""The norm's gradients as the benchmark's plain and 64-bit forms have them, against differences of its values — no GPU."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def forms():
    spec = importlib.util.spec_from_file_location("more_operators", os.path.join(ROOT, "perf", "more_operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("residual", [False, True])
def test_gradients(residual):
    """Central differences in 64 bits: h^2 / 6 of third derivatives, below 100 for these inputs, and 2^-50 / h. The
    plain form is in 32 bits: H / 32 + 64 roundings of the magnitudes that it adds."""
    import torch
    m = forms()
    g = torch.Generator().manual_seed(1)
    T, H, h = 3, 9, 1e-4
    rand = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)  # noqa: E731
    s = {"x": rand(T, H), "w": rand(H), "dy": rand(T, H), "train": True, "out": "same"}
    if residual:
        s["r"], s["ds"] = rand(T, H), rand(T, H)
    out = m._exact_norm(s)

    def loss(**changed):
        o = m._exact_norm({**s, **changed})
        return (o["y"] * s["dy"]).sum(1) + ((o["s"] * s["ds"]).sum(1) if residual else 0)

    size = float(s["dy"].abs().sum() + (s["ds"].abs().sum() if residual else 0))
    bound = size * (100 * h * h + 2.0 ** -50 / h)
    for c in range(H):
        step = torch.zeros(H, dtype=torch.float64)
        step[c] = h
        for name in ("x", "r") if residual else ("x",):
            slope = (loss(**{name: s[name] + step}) - loss(**{name: s[name] - step})) / (2 * h)
            assert float((slope - out["dx"][:, c]).abs().max()) <= bound
        slope = (loss(w=s["w"] + step) - loss(w=s["w"] - step)).sum() / (2 * h)
        assert abs(float(slope - out["dw"][c])) <= bound
    plain = m._norm(s)
    for name in ("y", "dx", "dw"):
        assert float((plain[name].double() - out[name]).abs().max()) <= (H / 32 + 64) * 2.0 ** -24 * size * float(s["w"].abs().max() + 1) * 4
