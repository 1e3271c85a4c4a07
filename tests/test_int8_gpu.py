"""Row quantisation and the 8-bit integer products against plain
implementations: codes bit for bit, products from their exact integer sums."""
import numpy as np
import pytest

from operator_util import TINY, UNIT, assert_within, counts_of, dtype_of, offsets_of, pitched, randn

pytestmark = pytest.mark.gpu


def quantize_plain(x):
    """The definition in IEEE float32: codes and scales of a float32 array."""
    x = np.asarray(x, np.float32)
    top = np.abs(x).max(1)
    live = ~(top < np.float32(1e-30))
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        inv = np.where(live, np.float32(127) / top, np.float32(0))
        scale = np.where(live, top / np.float32(127), np.float32(0))
        v = np.rint(x * inv[:, None])
    return np.nan_to_num(v, nan=0.0).astype(np.int8), scale


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("M,K", [(0, 64), (1, 1), (1, 8192), (3, 17), (5, 2048), (7, 2056), (2, 4104), (33, 1000), (2, 20000),
                                 (2, 9001)])
def test_quantize(cuda, M, K, dtype):
    import kebab_b200 as kb
    x = randn((M, K), dtype_of(dtype), M + K)
    q, scale = kb.quantize_i8(x)
    assert q.shape == (M, K) and scale.shape == (M,)
    if M == 0:
        return
    wq, ws = quantize_plain(x.float().cpu().numpy())
    np.testing.assert_array_equal(q.cpu().numpy(), wq)
    np.testing.assert_array_equal(scale.cpu().numpy(), ws)


def test_quantize_special_rows(cuda):
    import torch
    import kebab_b200 as kb
    for K in (256, 37):
        x = torch.zeros((9, K), device="cuda", dtype=torch.bfloat16)
        x[1] = -float("inf")
        x[2, 3] = float("inf")
        x[3, 5] = float("nan")
        x[4] = 1e-38                      # 127 / amax would overflow
        x[5] = 3.3e38                     # near the type's largest
        x[6] = torch.finfo(torch.bfloat16).min
        x[7] = 2e-30
        x[8] = torch.arange(K, device="cuda") % 255 / 2.0 - 63.5  # many ties
        q, s = kb.quantize_i8(x)
        wq, ws = quantize_plain(x.float().cpu().numpy())
        np.testing.assert_array_equal(q.cpu().numpy(), wq)
        np.testing.assert_array_equal(s.cpu().numpy(), ws)
        assert s[0] == 0 and s[4] == 0 and torch.isinf(s[1:3]).all() and torch.isnan(s[3])
        w, wsc = kb.quantize_i8(randn((64, K), torch.float32, 1))
        y = kb.gemm_i8(q, s, w, wsc)
        assert torch.isnan(y[1:4]).all() and torch.isfinite(y[[0, 4, 7, 8]]).all()
        assert torch.isnan(kb.linear_i8(x, w, wsc)[1:4]).all()


def test_quantize_pitched_and_stacked(cuda):
    import torch
    import kebab_b200 as kb
    x = randn((13, 264), torch.float16, 1)
    want = kb.quantize_i8(x)
    for extra, shift in ((8, 8), (3, 1)):
        got = kb.quantize_i8(pitched(x, extra, shift))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    w = randn((3, 5, 40), torch.bfloat16, 2)
    q, s = kb.quantize_i8(w)
    assert q.shape == (3, 5, 40) and s.shape == (3, 5)
    one = kb.quantize_i8(w[1])
    assert torch.equal(q[1], one[0]) and torch.equal(s[1], one[1])


def codes(shape, seed):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8)


def scales(shape, seed):
    import torch
    return torch.rand(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * 0.02 + 1e-3


def i8_plain(q, s, wq, ws, bias=None):
    """Float64 from the exact sums (below 2^31, so exact in 64 bits), and the
    size that the FP32 steps round."""
    y = (q.double() @ wq.double().T) * s.double()[:, None] * ws.double()
    size = y.abs()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    return y, size


def i8_bound(y, size, dtype):
    """The sum's conversion to FP32, two products and the bias: four roundings
    of 2^-24 of at most `size`; then the output's."""
    name = str(dtype).replace("torch.", "")
    return UNIT[name] * (y.abs() + size * 2.0 ** -21) + size * 2.0 ** -21 + TINY[name]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("M,K", [(1024, 8), (1025, 250), (1030, 256), (1100, 520), (2000, 1024), (1027, 2048), (1500, 2056)])
def test_quantize_many_rows(cuda, M, K, dtype):
    import kebab_b200 as kb
    x = randn((M, K), dtype_of(dtype), M + K)
    q, scale = kb.quantize_i8(x)
    wq, ws = quantize_plain(x.float().cpu().numpy())
    np.testing.assert_array_equal(q.cpu().numpy(), wq)
    np.testing.assert_array_equal(scale.cpu().numpy(), ws)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("M,N,K", [(1, 8, 16), (1, 513, 1024), (2, 256, 8192), (4, 1000, 2064), (7, 129, 160), (8, 512, 512),
                                   (9, 640, 4096), (16, 1, 32), (31, 257, 528), (64, 1024, 2048), (65, 384, 272),
                                   (128, 520, 1040), (200, 777, 1536), (256, 2048, 64), (257, 256, 128),
                                   (1000, 1032, 784), (2049, 2000, 512)])
def test_gemm_i8(cuda, M, N, K, dtype):
    import torch
    import kebab_b200 as kb
    dt = dtype_of(dtype)
    q, s, wq, ws = codes((M, K), M), scales((M,), 1), codes((N, K), N), scales((N,), 2)
    for bias in (None, randn((N,), dt, 3)):
        Y = torch.full((M, N), float("nan"), dtype=dt, device="cuda")
        kb.gemm_i8(q, s, wq, ws, bias=bias, dtype=dt, Y=Y)
        want, size = i8_plain(q, s, wq, ws, bias)
        assert_within(Y, want, i8_bound(want, size, dt), "Y")
    rc, code = kb.device_status()
    assert rc == kb.OK, hex(code)


@pytest.mark.parametrize("M,N,K", [(1, 3, 1), (3, 65, 17), (70, 33, 129), (300, 40, 4100)])
def test_gemm_i8_odd_sizes(cuda, M, N, K):
    import torch
    import kebab_b200 as kb
    q, s, wq, ws = codes((M, K), M), scales((M,), 1), codes((N, K), N), scales((N,), 2)
    y = kb.gemm_i8(q, s, wq, ws, dtype=torch.float16)
    want, size = i8_plain(q, s, wq, ws)
    assert_within(y, want, i8_bound(want, size, torch.float16), "Y")


@pytest.mark.parametrize("M", [1, 5, 40, 300])
def test_gemm_i8_pitched_and_unaligned(cuda, M):
    import torch
    import kebab_b200 as kb
    N, K = 264, 272
    q, s, wq, ws = codes((M, K), M), scales((M,), 1), codes((N, K), N), scales((N,), 2)
    bias = randn((N,), torch.float16, 4)
    want = kb.gemm_i8(q, s, wq, ws, bias=bias, dtype=torch.float16)
    for extra, shift in ((16, 16), (1, 0), (0, 5), (32, 0)):
        got = kb.gemm_i8(pitched(q, extra, shift), s, pitched(wq, extra, shift), ws, bias=bias, dtype=torch.float16)
        assert torch.equal(got, want)
        out = pitched(torch.zeros_like(want), extra, shift)
        assert torch.equal(kb.gemm_i8(q, s, wq, ws, bias=bias, dtype=torch.float16, Y=out), want)


@pytest.mark.parametrize("M", [1, 64, 300])
def test_gemm_i8_largest_sums(cuda, M):
    """Codes of -127 and 127 throughout: the largest sums the codes can make."""
    import torch
    import kebab_b200 as kb
    K = 16384
    q = torch.full((M, K), -127, dtype=torch.int8, device="cuda")
    wq = torch.full((300, K), 127, dtype=torch.int8, device="cuda")
    s, ws = torch.full((M,), 2.0 ** -20, device="cuda"), torch.full((300,), 2.0 ** -6, device="cuda")
    y = kb.gemm_i8(q, s, wq, ws, dtype=torch.bfloat16)
    want, size = i8_plain(q, s, wq, ws)
    assert_within(y, want, i8_bound(want, size, torch.bfloat16), "Y")


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("M,N,K", [(1, 512, 8192), (3, 260, 1040), (8, 1024, 4096), (33, 512, 2048), (300, 264, 336), (2, 64, 37)])
def test_linear_i8(cuda, M, N, K, dtype):
    import torch
    import kebab_b200 as kb
    dt = dtype_of(dtype)
    x, bias = randn((M, K), dt, M), randn((N,), dt, 2)
    wq, ws = kb.quantize_i8(randn((N, K), torch.float32, 1))
    q, s = quantize_plain(x.float().cpu().numpy())
    y = kb.linear_i8(x, wq, ws, bias=bias)
    assert y.dtype == dt
    want, size = i8_plain(torch.from_numpy(q).cuda(), torch.from_numpy(s).cuda(), wq, ws, bias)
    assert_within(y, want, i8_bound(want, size, dt), "Y")
    assert torch.equal(kb.linear_i8(pitched(x, 24, 8), wq, ws, bias=bias), y)


@pytest.mark.parametrize("R,E,N,K,kind", [(1, 1, 256, 256, "even"), (2, 8, 512, 1024, "ragged"), (8, 64, 256, 512, "ragged"),
                                          (50, 3, 264, 528, "ends"), (700, 5, 1000, 272, "ragged"), (600, 2, 512, 1024, "one"),
                                          (1021, 40, 384, 128, "ragged"), (90, 3, 65, 50, "ragged")])
def test_grouped_i8(cuda, R, E, N, K, kind):
    import torch
    import kebab_b200 as kb
    counts = counts_of(kind, R, E, R)
    offsets = offsets_of(counts)
    x = randn((R, K), torch.bfloat16, 1)
    wq, ws = kb.quantize_i8(randn((E, N, K), torch.float32, 2))
    q, s = (torch.from_numpy(t).cuda() for t in quantize_plain(x.float().cpu().numpy()))
    want, size, at = torch.zeros((R, N), dtype=torch.float64, device="cuda"), torch.zeros((R, N), dtype=torch.float64, device="cuda"), 0
    for e, c in enumerate(counts):
        want[at:at + c], size[at:at + c] = i8_plain(q[at:at + c], s[at:at + c], wq[e], ws[e])
        at += c
    bound = i8_bound(want, size, torch.bfloat16)
    Y = torch.full((R, N), float("nan"), dtype=torch.bfloat16, device="cuda")
    kb.gemm_grouped_i8(q, s, wq, ws, offsets, Y=Y)
    assert_within(Y, want, bound, "Y")
    assert_within(kb.linear_grouped_i8(x, wq, ws, offsets), want, bound, "linear")


def test_no_rows(cuda):
    import torch
    import kebab_b200 as kb
    wq, ws = codes((64, 32), 1), scales((64,), 2)
    x = torch.zeros((0, 32), dtype=torch.float16, device="cuda")
    assert kb.linear_i8(x, wq, ws).shape == (0, 64)
    assert kb.linear_grouped_i8(x, wq[None], ws[None], offsets_of([0])).shape == (0, 64)


@pytest.mark.parametrize("M", [1, 8, 64, 500])
def test_streams_and_repeats(cuda, M):
    """Bit for bit the same on repeats, on other streams and in a CUDA graph."""
    import torch
    import kebab_b200 as kb
    x, (wq, ws) = randn((M, 2048), torch.bfloat16, 1), kb.quantize_i8(randn((1024, 2048), torch.float32, 2))
    want = kb.linear_i8(x, wq, ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = [kb.linear_i8(x, wq, ws, stream=side if i % 2 else None) for i in range(6)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = kb.linear_i8(x, wq, ws)
    for _ in range(2):
        captured.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        outs.append(captured.clone())
    for o in outs:
        assert torch.equal(o, want)
