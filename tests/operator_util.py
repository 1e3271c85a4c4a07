"""Shared by the tests of the expert and 8-bit integer operators: seeded
inputs, ragged offsets, and the error bounds of a product summed in FP32."""
import numpy as np

# Unit roundoff of the output types.
UNIT = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float32": 2.0 ** -24}
# Half the spacing of the smallest numbers.
TINY = {"float16": 2.0 ** -25, "bfloat16": 2.0 ** -134, "float32": 2.0 ** -150}


def dtype_of(name):
    import torch
    return getattr(torch, name)


def randn(shape, dtype, seed, device="cuda"):
    import torch
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device=device, dtype=torch.float32).to(dtype)


def pitched(t, extra, shift=0):
    """`t` (rows contiguous) inside a wider buffer: row pitch larger by `extra`
    elements, first element moved by `shift`; the rest of the buffer is NaN (a
    type's extreme value for integers)."""
    import torch
    rows, cols = t.shape[-2:]
    n = int(np.prod(t.shape[:-2], dtype=np.int64)) if t.dim() > 2 else 1
    ld = cols + extra
    fill = float("nan") if t.is_floating_point() else -128
    buf = torch.full((shift + n * rows * ld,), fill, dtype=t.dtype, device=t.device)
    view = buf[shift:].view(*t.shape[:-2], rows, ld)[..., :cols]
    view.copy_(t)
    return view


def counts_of(kind, R, E, seed=0):
    """Row counts of E groups over R rows: even, one (all rows in one group),
    ragged (random, some empty) or ends (the first and last empty)."""
    rng = np.random.default_rng(seed)
    if kind == "even":
        c = np.full(E, R // E)
        c[: R % E] += 1
    elif kind == "one":
        c = np.zeros(E, np.int64)
        c[E // 2] = R
    elif kind == "ragged":
        p = rng.dirichlet(np.full(E, 0.5))
        c = rng.multinomial(R, p)
    else:
        c = np.zeros(E, np.int64)
        inner = max(E - 2, 1)
        c[1 if E > 2 else 0:][:inner] = rng.multinomial(R, np.full(inner, 1.0 / inner))
    assert c.sum() == R
    return c.tolist()


def offsets_of(counts, device="cuda", first=0):
    import torch
    return torch.tensor(np.concatenate([[0], np.cumsum(counts)]) + first, dtype=torch.int32, device=device)


def assert_within(got, want, bound, what=""):
    """|got - want| <= bound in every place; NaN and infinities have to agree."""
    import torch
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if got.numel() == 0:
        return
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "%s: NaN in other places" % what
    assert torch.equal(torch.isfinite(got), finite), "%s: infinities in other places" % what
    excess = ((got - want).abs() - bound)[finite]
    if excess.numel():
        worst = float(excess.max())
        assert worst <= 0, "%s: %.3e over the bound in %d places" % (what, worst, int((excess > 0).sum()))


def product_bound(y, magnitude, terms, dtype):
    """Bound of a product's error: `terms` FP32 additions of exact products
    whose magnitudes sum to `magnitude` (each addition loses at most 2^-23 of
    what has been summed, truncation included), then one rounding."""
    name = str(dtype).replace("torch.", "")
    acc = terms * 2.0 ** -23 * magnitude
    return UNIT[name] * (y.abs() + acc) + acc + TINY[name]
