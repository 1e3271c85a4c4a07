"""The persistent grouped kernel where only larger products reach it: panels
of 512 rows, outputs on odd pitches, reads past a group's end, many groups.
Each test checks that its sizes take that kernel."""
import pytest

from operator_util import assert_within, counts_of, dtype_of, offsets_of, pitched, product_bound, randn
from test_experts_gpu import grouped_plain, weights_of
from test_int8_gpu import codes, i8_bound, i8_plain, scales

pytestmark = pytest.mark.gpu


def persistent(call):
    """call()'s result, after a check of the kernel that it ran."""
    import torch
    from torch.profiler import ProfilerActivity, profile
    call()
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        out = call()
        torch.cuda.synchronize()
    names = [e.name for e in p.events()]
    if names:  # else the machine records none
        names = [n for n in names if "grouped_" in n]
        assert names and all("grouped_umma_kernel" in n for n in names), names
    return out


def status():
    import kebab_b200 as kb
    rc, code = kb.device_status()
    assert rc == kb.OK, hex(code)


def spans(counts, first=0):
    at = first
    for e, c in enumerate(counts):
        yield e, slice(at, at + c)
        at += c


# At least 8 tiles of 256 x 256 a pair (592): panels of 512 rows, the last of
# them a half; tiles of one K-block, a few, and enough for stores by TMA.
WIDE = [900, 0, 257, 1, 1500, 255, 1024, 33, 512, 130]


@pytest.mark.parametrize("opmode", ["RC", "RR"])
@pytest.mark.parametrize("N,K,dtype", [(7688, 40, "bfloat16"), (7688, 264, "float16"), (7944, 1000, "bfloat16"),
                                       (8200, 2048, "float16")])
def test_wide_panels(cuda, N, K, dtype, opmode):
    import torch
    import kebab_b200 as kb
    dt, R = dtype_of(dtype), sum(WIDE)
    assert sum((c + 255) // 256 for c in WIDE) * ((N + 255) // 256) >= 592
    X, W = randn((R, K), dt, 1), weights_of(len(WIDE), N, K, dt, opmode, 2)
    Y = torch.full((R, N), float("nan"), dtype=dt, device="cuda")
    persistent(lambda: kb.gemm_grouped(X, W, offsets_of(WIDE), Y=Y.fill_(float("nan")), opmode=opmode))
    want, size = grouped_plain(X, W, WIDE, opmode)
    assert_within(Y, want, product_bound(want, size, K, dt), "Y")
    status()


@pytest.mark.parametrize("opmode", ["RC", "RR"])
@pytest.mark.parametrize("N,extra,shift", [(7687, 0, 0), (7687, 2, 1), (7688, 3, 0), (7688, 0, 4), (2049, 0, 0), (2056, 1, 5)])
def test_odd_outputs(cuda, N, extra, shift, opmode):
    """Rows of Y that are not on 16-byte boundaries, with panels of 512 rows
    and (about 2050 columns) of 256."""
    import torch
    import kebab_b200 as kb
    dt, K, R = torch.bfloat16, 520, sum(WIDE)
    X, W = randn((R, K), dt, 1), pitched(weights_of(len(WIDE), N, K, dt, opmode, 2), -(N if opmode == "RR" else K) % 8, 0)
    buf = pitched(torch.zeros((R, N), dtype=dt, device="cuda"), extra, shift)
    whole = buf._base if buf._base is not None else buf
    outside = torch.ones_like(whole, dtype=torch.bool)
    outside.as_strided(buf.shape, buf.stride(), buf.storage_offset()).fill_(False)
    before = whole[outside].view(torch.int16).clone()
    persistent(lambda: kb.gemm_grouped(X, W, offsets_of(WIDE), Y=buf, opmode=opmode))
    want, size = grouped_plain(X, W, WIDE, opmode)
    assert_within(buf, want, product_bound(want, size, K, dt), "Y")
    assert torch.equal(whole[outside].view(torch.int16), before)
    status()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("M,N,K", [(1501, 2049, 272), (1280, 2307, 1040), (257, 9999, 4112), (4097, 7689, 144)])
def test_i8_odd_outputs(cuda, M, N, K, dtype):
    import torch
    import kebab_b200 as kb
    dt = dtype_of(dtype)
    q, s, wq, ws = codes((M, K), M), scales((M,), 1), codes((N, K), N), scales((N,), 2)
    bias = randn((N,), dt, 3)
    want, size = i8_plain(q, s, wq, ws, bias)
    for extra in (0, 1, -N % 8):
        Y = pitched(torch.full((M, N), float("nan"), dtype=dt, device="cuda"), extra, 0)
        persistent(lambda: kb.gemm_i8(q, s, wq, ws, bias=bias, dtype=dt, Y=Y))
        assert_within(Y, want, i8_bound(want, size, dt), "Y")
    status()


@pytest.mark.parametrize("R,E,N,K,kind", [(2500, 9, 2049, 272, "ragged"), (6001, 14, 4099, 528, "ragged"), (3000, 4, 4096, 144, "ends")])
def test_grouped_i8(cuda, R, E, N, K, kind):
    import torch
    import kebab_b200 as kb
    dt, counts = torch.float16, counts_of(kind, R, E, R)
    q, s, wq, ws = codes((R, K), 1), scales((R,), 2), codes((E, N, K), 3), scales((E, N), 4)
    Y = torch.full((R, N), float("nan"), dtype=dt, device="cuda")
    persistent(lambda: kb.gemm_grouped_i8(q, s, wq, ws, offsets_of(counts), dtype=dt, Y=Y.fill_(float("nan"))))
    for e, r in spans(counts):
        want, size = i8_plain(q[r], s[r], wq[e], ws[e])
        assert_within(Y[r], want, i8_bound(want, size, dt), "group %d" % e)
    status()


@pytest.mark.parametrize("opmode", ["RC", "RR"])
@pytest.mark.parametrize("N", [1032, 8200])
def test_neighbours_and_rows_of_no_group(cuda, N, opmode):
    """Tiles read past their group's end: rows of NaN there, of other groups
    and of none, stay out; rows of no group are not written."""
    import torch
    import kebab_b200 as kb
    dt, K, first = torch.float16, 264, 77
    counts = [37, 283, 5, 1, 530, 0, 1200, 255, 900, 1030]
    R = first + sum(counts) + 50
    X, W = randn((R, K), dt, 1), weights_of(len(counts), N, K, dt, opmode, 2)
    offsets = offsets_of(counts, first=first)
    clean = persistent(lambda: kb.gemm_grouped(X, W, offsets, opmode=opmode))
    end = first + sum(counts)
    X[:first], X[end:] = float("nan"), float("inf")
    for e, r in spans(counts, first):
        if e % 2:
            X[r], W[e] = float("nan"), float("inf")
    Y = torch.full((R, N), 7.0, dtype=dt, device="cuda")
    persistent(lambda: kb.gemm_grouped(X, W, offsets, Y=Y, opmode=opmode))
    assert (Y[:first] == 7).all() and (Y[end:] == 7).all()
    for e, r in spans(counts, first):
        assert torch.isnan(Y[r]).all() if e % 2 else torch.equal(Y[r], clean[r]), e
    status()


@pytest.mark.parametrize("opmode", ["RC", "RR"])
@pytest.mark.parametrize("R,E", [(2048, 513), (5000, 1024), (70001, 700)])
def test_more_groups_than_are_sorted(cuda, R, E, opmode):
    import torch
    import kebab_b200 as kb
    dt, N, K = torch.bfloat16, 264, 72
    counts = counts_of("ragged", R, E, 1)
    assert E > 512 and 0 in counts
    X, W, dY = randn((R, K), dt, 1), weights_of(E, N, K, dt, opmode, 2), randn((R, N), dt, 3)
    Y = torch.full((R, N), float("nan"), dtype=dt, device="cuda")
    persistent(lambda: kb.gemm_grouped(X, W, offsets_of(counts), Y=Y.fill_(float("nan")), opmode=opmode))
    want, size = grouped_plain(X, W, counts, opmode)
    assert_within(Y, want, product_bound(want, size, K, dt), "Y")
    dW = persistent(lambda: kb.gemm_grouped_dw(X, dY, offsets_of(counts), opmode=opmode))
    for e, r in spans(counts):
        a, b = (dY[r], X[r]) if opmode == "RC" else (X[r], dY[r])
        want, size = a.double().T @ b.double(), a.double().abs().T @ b.double().abs()
        assert_within(dW[e], want, product_bound(want, size, counts[e], dt), "dW of %d" % e)
    status()


@pytest.mark.parametrize("N", [2056, 8200])
def test_streams_and_repeats(cuda, N):
    """Bit for bit the same on repeats, on other streams and in a CUDA graph."""
    import torch
    import kebab_b200 as kb
    dt, K, R = torch.bfloat16, 512, sum(WIDE)
    X, W, offsets = randn((R, K), dt, 1), weights_of(len(WIDE), N, K, dt, "RC", 2), offsets_of(WIDE)
    want = persistent(lambda: kb.gemm_grouped(X, W, offsets))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = [kb.gemm_grouped(X, W, offsets, stream=side if i % 2 else None) for i in range(4)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = kb.gemm_grouped(X, W, offsets)
    for _ in range(2):
        captured.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        outs.append(captured.clone())
    assert all(torch.equal(o, want) for o in outs)
    status()


def test_gradients_against_differences(cuda):
    """The products are linear in X and in W, so differences are exact up to
    rounding: <dY, Y(X + D) - Y(X)> = <dX, D>, and the same for W."""
    import torch
    import kebab_b200 as kb
    E, N, K, dt, R = 5, 2056, 1032, torch.float16, 3000
    offsets = offsets_of(counts_of("ragged", R, E, 4))
    # Multiples of 1/4 and small: every sum below is exact in FP32, and the
    # rounding to FP16 is the only error.
    q = lambda shape, seed: (randn(shape, torch.float32, seed) * 2).round().clamp(-4, 4).to(dt) / 4  # noqa: E731
    X, DX, W, DW, dY = q((R, K), 1), q((R, K), 2), q((E, N, K), 3), q((E, N, K), 4), q((R, N), 5)
    f = lambda a, b, m="RC": persistent(lambda: kb.gemm_grouped(a, b, offsets, opmode=m))  # noqa: E731
    y, u, d = f(X, W).double(), 2.0 ** -11, dY.double()
    for moved, grad, D in ((f(X + DX, W), f(dY, W, "RR"), DX),
                           (f(X, W + DW), kb.gemm_grouped_dw(X, dY, offsets), DW)):
        moved, term = moved.double(), grad.double() * D.double()
        slope = (d * (moved - y)).sum()
        bound = u * ((d * moved).abs().sum() + (d * y).abs().sum() + term.abs().sum()) * 1.01
        assert abs(float(term.sum() - slope)) <= float(bound)
