"""Root-mean-square norm, its 8-bit form and its gradients against 64 bits."""
import pytest

from operator_util import TINY, UNIT, assert_within, dtype_of, pitched, randn

pytestmark = pytest.mark.gpu
EPS = 1e-6


def f32_error(H):
    """Relative error of s rstd w in FP32: at most H / 32 + 16 additions in a row for the mean of squares (half of it
    after the root), 2^-22 of the root, and eight roundings."""
    return (H / 64 + 8 + 4 + 8) * 2.0 ** -24


def reference(x, w, r=None, eps=EPS):
    s = x if r is None else (x.double() + r.double()).to(x.dtype)
    d = s.double()
    rstd = (d.square().mean(1, keepdim=True) + eps).rsqrt()
    return s, rstd, d * rstd * w.double()


def check_norm(x, w, r, y, s):
    want_s, _, want = reference(x, w, r)
    if r is None:
        assert s is x
    else:
        assert s.dtype == x.dtype
        assert_within(s, want_s, 0.0 if x.dtype.itemsize == 2 else UNIT["float32"] * 2 * want_s.double().abs(), "s")
        _, _, want = reference(s, w)  # of the sum as it is stored
    name = str(x.dtype).replace("torch.", "")
    rel = f32_error(x.shape[1])
    assert y.dtype == x.dtype and y.shape == x.shape
    assert_within(y, want, want.abs() * (rel + UNIT[name] * (1 + rel)) + TINY[name], "y")


SHAPES = [(1, 1), (1, 8192), (3, 7), (5, 64), (2, 4097), (300, 8192), (2000, 256), (1500, 1000), (1030, 1024), (700, 2048), (2, 20000),
          (400, 16384), (400, 9000), (1100, 129), (301, 257), (300, 8193), (300, 8200), (310, 8191), (300, 10239), (300, 10248)]


@pytest.mark.parametrize("T,H", SHAPES)
@pytest.mark.parametrize("dtype,weight", [("float16", "float16"), ("bfloat16", "float32"), ("bfloat16", "bfloat16"), ("float32", "float32")])
@pytest.mark.parametrize("residual", [False, True])
def test_norm(cuda, T, H, dtype, weight, residual):
    import kebab_b200 as kb
    x, w = randn((T, H), dtype_of(dtype), 1), randn((H,), dtype_of(weight), 2)
    r = randn((T, H), dtype_of(dtype), 3) if residual else None
    y, s = kb.rms_norm(x, w, EPS, residual=r)
    check_norm(x, w, r, y, s)


@pytest.mark.parametrize("T,H", [(1, 8192), (5, 64), (2, 4097), (300, 8192), (2000, 256), (1500, 1000), (2, 20000), (1100, 129),
                                 (300, 8200), (300, 8191), (300, 10240), (300, 10248), (300, 2501)])
@pytest.mark.parametrize("dtype,weight", [("float16", "float32"), ("bfloat16", "bfloat16"), ("float32", "float32")])
@pytest.mark.parametrize("residual,keep", [(False, False), (True, True)])
def test_norm_i8(cuda, T, H, dtype, weight, residual, keep):
    import torch
    import kebab_b200 as kb
    x, w = randn((T, H), dtype_of(dtype), 4), randn((H,), dtype_of(weight), 5)
    r = randn((T, H), dtype_of(dtype), 6) if residual else None
    n = kb.rms_norm_i8(x, w, EPS, residual=r, keep=keep)
    if keep:
        check_norm(x, w, r, n.y, n.residual)
    else:
        assert n.y is None
    _, _, want = reference(n.residual, w)
    rel = f32_error(H)
    top = want.abs().amax(1)
    assert n.codes.dtype == torch.int8 and int(n.codes.abs().max()) <= 127
    assert_within(n.scale, top / 127, top / 127 * (rel + 2.0 ** -23))
    # Half a step, the value's own error, and that of the step over at most 127 of them.
    got = n.codes.double() * (top / 127)[:, None]
    assert_within(got, want, (top / 127)[:, None] * (0.5 + 127 * (3 * rel + 2.0 ** -22)), "codes")
    codes = kb.rms_norm_i8(x, w, EPS, residual=r).codes
    assert torch.equal(codes, n.codes)


def test_norm_i8_feeds_the_product(cuda):
    """What a serving step does: norm with 8-bit output, then an 8-bit projection."""
    import kebab_b200 as kb
    x, w, W = randn((33, 1024), dtype_of("bfloat16"), 1), randn((1024,), dtype_of("float32"), 2), randn((256, 1024), dtype_of("bfloat16"), 3)
    q, ws = kb.quantize_i8(W)
    n = kb.rms_norm_i8(x, w, residual=x)
    y = kb.gemm_i8(n.codes, n.scale, q, ws)
    want = (n.codes.double() @ q.double().T) * n.scale.double()[:, None] * ws.double()
    assert_within(y, want, want.abs() * (UNIT["bfloat16"] + 2.0 ** -21) + TINY["bfloat16"])


def check_backward(T, H, dtype, weight, with_ds, make=lambda t: t, seed=7):
    import kebab_b200 as kb
    s, dy, w = randn((T, H), dtype_of(dtype), seed), randn((T, H), dtype_of(dtype), seed + 1), randn((H,), dtype_of(weight), seed + 2)
    ds = randn((T, H), dtype_of(dtype), seed + 3) if with_ds else None
    dx, dw = kb.rms_norm_backward(make(dy), make(s), w, EPS, dresidual=None if ds is None else make(ds))
    _, rstd, _ = reference(s, w)
    g, d = dy.double() * w.double(), s.double()
    mean, mean_abs = (g * d).mean(1, keepdim=True), (g * d).abs().mean(1, keepdim=True)
    want = rstd * (g - d * rstd * rstd * mean)
    size = rstd * (g.abs() + d.abs() * rstd * rstd * mean_abs)  # of the terms
    if with_ds:
        want, size = want + ds.double(), size + ds.double().abs()
    name, rel = dtype, 3 * f32_error(H) + H / 32 * 2.0 ** -24
    assert_within(dx, want, size * rel + UNIT[name] * (want.abs() + size * rel) + TINY[name], "dx")
    terms = dy.double() * d * rstd
    # At most T additions of terms with the error of s rstd.
    bound = terms.abs().sum(0) * (f32_error(H) + T * 2.0 ** -24)
    want = terms.sum(0)
    assert dw.dtype == w.dtype
    assert_within(dw, want, bound + UNIT[weight] * (want.abs() + bound) + TINY[weight], "dw")
    return dx, dw


@pytest.mark.parametrize("T,H", [(1, 1), (1, 4096), (3, 7), (700, 1024), (1300, 2048), (200, 4096), (200, 8192), (40, 16384), (37, 20000),
                                 (5, 40000), (200, 1001), (30, 4097), (9, 2049), (200, 8200), (200, 8191), (50, 12288), (50, 12281), (50, 12289)])
@pytest.mark.parametrize("dtype,weight", [("float16", "float16"), ("bfloat16", "float32"), ("float32", "float32")])
@pytest.mark.parametrize("with_ds", [False, True])
def test_backward(cuda, T, H, dtype, weight, with_ds):
    import torch
    first = check_backward(T, H, dtype, weight, with_ds)
    for a, b in zip(first, check_backward(T, H, dtype, weight, with_ds)):
        assert torch.equal(a, b)  # the sums have a fixed order


@pytest.mark.parametrize("extra,shift", [(8, 0), (8, 1), (3, 0)])
def test_pitched_rows(cuda, extra, shift):
    import kebab_b200 as kb
    make = lambda t: pitched(t, extra, shift)  # noqa: E731
    for T, H in ((5, 1024), (301, 8192), (3, 77)):
        x, r, w = randn((T, H), dtype_of("bfloat16"), 1), randn((T, H), dtype_of("bfloat16"), 2), randn((H,), dtype_of("float32"), 3)
        y, s = kb.rms_norm(make(x), w, EPS, residual=make(r))
        check_norm(x, w, r, y, s)
        n = kb.rms_norm_i8(make(x), w, EPS, residual=make(r), keep=True)
        check_norm(x, w, r, n.y, n.residual)
        check_backward(T, H, "bfloat16", "float32", True, make)


def test_empty_and_zero_rows(cuda):
    import torch
    import kebab_b200 as kb
    w = torch.ones(64, device="cuda")
    x = torch.zeros((0, 64), dtype=torch.bfloat16, device="cuda")
    y, s = kb.rms_norm(x, w, residual=x)
    assert y.shape == s.shape == (0, 64)
    n = kb.rms_norm_i8(x, w)
    assert n.codes.shape == (0, 64) and n.scale.shape == (0,)
    dx, dw = kb.rms_norm_backward(x, x, w)
    assert dx.shape == (0, 64) and torch.equal(dw, torch.zeros(64, device="cuda"))
    x = torch.zeros((3, 64), dtype=torch.bfloat16, device="cuda")
    assert torch.equal(kb.rms_norm(x, w)[0], x)  # eps keeps the root finite
    n = kb.rms_norm_i8(x, w)
    assert not n.codes.any() and not n.scale.any()


def test_non_finite_rows_stay_to_themselves(cuda):
    import torch
    import kebab_b200 as kb
    x, w = randn((4, 1024), torch.bfloat16, 1), randn((1024,), torch.float32, 2)
    clean = kb.rms_norm(x, w)[0]
    x[1, 5], x[2, 7] = float("inf"), float("nan")
    y, n = kb.rms_norm(x, w)[0], kb.rms_norm_i8(x, w)
    assert torch.equal(y[[0, 3]], clean[[0, 3]])
    assert torch.isnan(y[1, 5]) and torch.isnan(y[2]).all()  # inf * 0, and NaN throughout
    assert torch.isnan(n.scale[1:3]).all() and torch.isfinite(n.scale[[0, 3]]).all() and not n.codes[1:3].any()


def test_captured(cuda):
    """A training step's norm in a graph, replayed on new inputs."""
    import torch
    import kebab_b200 as kb
    x, r, dy = (randn((65, 2048), torch.bfloat16, i) for i in (1, 2, 3))
    w = randn((2048,), torch.float32, 4)

    def step():
        y, s = kb.rms_norm(x, w, residual=r)
        return (y, s, *kb.rms_norm_backward(dy, s, w, dresidual=dy), *kb.rms_norm_i8(x, w, residual=r)[:2])

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (5, 6):
        for t, k in ((x, 0), (r, 10), (dy, 20)):
            t.copy_(randn((65, 2048), torch.bfloat16, seed + k))
        graph.replay()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


def test_other_stream(cuda):
    import torch
    import kebab_b200 as kb
    x, w = randn((64, 4096), torch.float16, 1), randn((4096,), torch.float16, 2)
    want = kb.rms_norm(x, w, residual=x)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    got = kb.rms_norm(x, w, residual=x, stream=stream)
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(cuda):
    import torch
    import kebab_b200 as kb
    x, w = randn((4, 64), torch.bfloat16, 1), randn((64,), torch.float32, 2)
    for call in (lambda: kb.rms_norm(x, w[:63].contiguous()), lambda: kb.rms_norm(x, w.half()), lambda: kb.rms_norm(x, w, residual=x[:3]),
                 lambda: kb.rms_norm(x, w, residual=x.float()), lambda: kb.rms_norm(x, w, eps=-1.0), lambda: kb.rms_norm(x, w, eps=float("nan")),
                 lambda: kb.rms_norm(x.T, w), lambda: kb.rms_norm(x[0], w), lambda: kb.rms_norm(x[:, :0], w[:0]),
                 lambda: kb.rms_norm_i8(x, w, residual=x[:3]), lambda: kb.rms_norm_backward(x, x[:3], w), lambda: kb.rms_norm_backward(None, x, w),
                 lambda: kb.rms_norm_backward(x, x, w, dresidual=x.half()), lambda: kb.rms_norm(x.double(), w.double())):
        with pytest.raises(kb.KebabError):
            call()
