"""Microscaled 4-bit floating point: codes and scales bit by bit, products
against 64 bits."""
import pytest

from operator_util import assert_within, counts_of, dtype_of, offsets_of, pitched, product_bound, randn

pytestmark = pytest.mark.gpu


def grid(device="cuda"):
    import torch
    g = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=device)
    return torch.cat([g, -g])


def reference(x):
    """(codes [.., B * 32], scale bytes [.., B]) of rows in 64 bits, by the distances to the grid."""
    import torch
    x = torch.nn.functional.pad(x.double(), (0, -x.shape[-1] % 32))
    b = x.reshape(*x.shape[:-1], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    ok = torch.isfinite(top)
    b = torch.where(ok, b, 0.0)
    top = torch.where(ok, top, 0.0)
    e = torch.where(top > 0, torch.round(torch.log2(torch.where(top > 0, top, 1.0) / 6)), -127.0)
    e = (e + (top > 6 * torch.exp2(e)).double()).clamp(min=-127)  # the logarithm itself may be off by a little
    v = b / torch.exp2(e)
    far = (v.abs()[..., None] - grid(x.device)[:8]).abs()
    near = far.amin(-1, keepdim=True)
    tied = far == near
    even = torch.arange(8, device=x.device) % 2 == 0
    # Of two equally near ones the even code: argmax of a score that prefers it.
    code = (tied.int() * 2 + (tied & even).int()).argmax(-1)
    code = code + 8 * torch.signbit(b).long()
    code = torch.where(ok, code, 0)
    return code.flatten(-2), torch.where(ok, e + 127, 255.0)[..., 0].long()


def unpacked(codes):
    import torch
    return torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()


def weight_scales(q):
    """Scale bytes [N, B] in plain order."""
    import torch
    N, B = q.codes.shape[-2], q.codes.shape[-1] // 16
    n, b = torch.arange(N, device="cuda")[:, None], torch.arange(B, device="cuda")[None, :]
    return q.scales[..., n // 128, b // 4, n % 32 * 16 + n % 128 // 32 * 4 + b % 4].long()


def token_scales(q):
    import torch
    M, B = q.codes.shape[0], q.codes.shape[1] // 16
    r, b = torch.arange(M, device="cuda")[:, None], torch.arange(B, device="cuda")[None, :]
    first = q.scales[b // 4, r, b % 4].long()
    for part in (1, 2, 3):  # the other places of the same scale
        at = (r - 32 * part).clamp(min=0)
        other = q.scales[b // 4, at, 4 * part + b % 4].long()
        assert torch.equal(torch.where(r >= 32 * part, other, first), first)
    return first


def values(codes, scales):
    import torch
    v = grid()[codes].reshape(*scales.shape, 32) * torch.exp2(scales.double() - 127)[..., None]
    return torch.where(scales[..., None] == 255, float("nan"), v).flatten(-2)


def specials(dtype):
    """Rows at the edges: every tie of the grid, amax on and next to 6 and its half, the smallest and largest numbers, zeros, infinities, NaN."""
    import torch
    f = torch.finfo(dtype)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, -0.0], dtype=torch.float64)
    rows = []
    for scale in (1.0, 2.0 ** -9, 2.0 ** 9):
        rows += [ties.repeat(2) * scale, torch.cat([ties, torch.zeros(16, dtype=torch.float64)]) * scale]
    one = torch.zeros(32, dtype=torch.float64)
    for top in (6.0, 6.0 * (1 + f.eps), 6.0 * (1 - f.eps), 3.0, 3.0 * (1 + f.eps), 4.0, f.tiny, f.smallest_normal / 4 if dtype != torch.float32 else 2.0 ** -149,
                f.max, f.max / 2, 0.0, float("inf"), float("nan"), -float("inf")):
        row = one.clone()
        row[5], row[17], row[31] = top, -top / 3 if top == top and abs(top) != float("inf") else 1.0, 0.5
        rows.append(row)
        rows.append(torch.full((32,), top, dtype=torch.float64))
    return torch.stack(rows).to(dtype).cuda()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
def test_special_blocks(cuda, dtype):
    import torch
    import kebab_b200 as kb
    x = specials(dtype_of(dtype))
    codes, scales = reference(x)
    q, t = kb.quantize_f4(x), kb.quantize_f4_tokens(x)
    for got, s in ((q.codes, weight_scales(q)), (t.codes, token_scales(t))):
        assert torch.equal(s, scales)
        assert torch.equal(unpacked(got), codes)
    assert_within(kb.dequantize_f4(q, 32), values(codes, scales).float(), 0.0)


@pytest.mark.parametrize("N,K", [(1, 1), (1, 32), (3, 31), (128, 128), (130, 129), (257, 1000), (64, 4096), (1000, 264), (7, 8200)])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("extra,shift", [(0, 0), (8, 0), (3, 1)])
def test_quantize(cuda, N, K, dtype, extra, shift):
    import torch
    import kebab_b200 as kb
    x = randn((N, K), dtype_of(dtype), N + K) * torch.exp2(torch.randint(-20, 10, (N, 1), device="cuda").float()).to(dtype_of(dtype))
    codes, scales = reference(x)
    view = pitched(x, extra, shift)
    q, t = kb.quantize_f4(view), kb.quantize_f4_tokens(view)
    B = (K + 31) // 32
    assert q.codes.shape == t.codes.shape == (N, B * 16) and q.scales.shape == ((N + 127) // 128, (K + 127) // 128, 512)
    for got, s in ((q.codes, weight_scales(q)), (t.codes, token_scales(t))):
        assert torch.equal(s, scales) and torch.equal(unpacked(got), codes)
    # Places of no row or block hold 0.
    assert int(q.scales.long().sum()) == int(scales.sum())
    for out in (torch.float32, torch.bfloat16, torch.float16):
        assert_within(kb.dequantize_f4(q, K, out), values(codes, scales)[:, :K].to(out), 0.0)
    stack = kb.quantize_f4(torch.stack([x, -x, x]).contiguous())
    assert torch.equal(stack.codes[0], q.codes) and torch.equal(stack.scales[1], q.scales)
    assert torch.equal(kb.dequantize_f4(stack, K)[1], -kb.dequantize_f4(q, K))


def operands(M, N, K, seed=1, dtype="bfloat16", E=0):
    X, W = randn((M, K), dtype_of(dtype), seed), randn((E, N, K) if E else (N, K), dtype_of(dtype), seed + 1)
    return X, W


def exact_values(X):
    codes, scales = reference(X)
    return values(codes, scales)[..., : X.shape[-1]]


def check(Y, X, W, bias=None):
    """Y of the quantised X and W, both given unquantised."""
    x, w = exact_values(X), exact_values(W)
    want, size = x @ w.T, x.abs() @ w.abs().T
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    assert_within(Y, want, product_bound(want, size, X.shape[1] + 1, Y.dtype))


SHAPES = [(1, 128, 128), (1, 1, 1), (1, 8192, 8192), (7, 129, 100), (16, 256, 512), (33, 1000, 1024), (64, 520, 4096), (65, 384, 300), (128, 257, 640),
          (129, 1024, 256), (200, 4096, 2048), (500, 2056, 1000), (1021, 1024, 1152), (241, 512, 64), (2050, 776, 520), (3000, 2304, 264)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_linear(cuda, M, N, K, dtype):
    import torch
    import kebab_b200 as kb
    X, W = operands(M, N, K, M + N, dtype)
    q = kb.quantize_f4(W)
    Y = kb.linear_f4(X, q)
    check(Y, X, W)
    bias = randn((N,), dtype_of(dtype), 9)
    out = torch.full((M, N), float("nan"), dtype=X.dtype, device="cuda")
    assert kb.linear_f4(X, q, bias=bias, Y=out) is out
    check(out, X, W, bias)
    assert torch.equal(kb.gemm_f4(kb.quantize_f4_tokens(X), q, dtype=X.dtype), Y)


@pytest.mark.parametrize("M,N,K", [(1, 300, 512), (16, 128, 256), (100, 300, 384), (300, 520, 512), (1000, 1536, 256), (2000, 3000, 128)])
def test_exact_sums(cuda, M, N, K):
    """Small multiples of the scales, whose sums FP32 holds exactly: every place has to be right, not only near."""
    import torch
    import kebab_b200 as kb
    g = torch.Generator(device="cuda")
    g.manual_seed(M)

    def make(rows):
        v = grid()[torch.randint(0, 16, (rows, K), generator=g, device="cuda")].reshape(rows, -1, 32)
        v[..., 0] = 6.0  # so that the scale is the one that is meant
        return (v * torch.exp2(torch.randint(-1, 3, (rows, K // 32, 1), generator=g, device="cuda").double())).flatten(1)

    x, w = make(M), make(N)
    # |sum| <= 512 * 36 * 16 in quarters of 1/4: below 2^24 of them.
    Y = kb.linear_f4(x.bfloat16(), kb.quantize_f4(w.bfloat16()))
    assert torch.equal(Y, (x @ w.T).float().bfloat16())


@pytest.mark.parametrize("kind", ["even", "one", "ragged", "ends"])
@pytest.mark.parametrize("R,E,N,K", [(1, 4, 128, 128), (8, 64, 256, 512), (100, 3, 300, 1000), (600, 7, 1032, 520), (1500, 5, 512, 256),
                                     (3000, 9, 2056, 264), (700, 200, 264, 96)])
def test_grouped(cuda, kind, R, E, N, K):
    import torch
    import kebab_b200 as kb
    X, W = operands(R, N, K, R + E, "float16", E)
    counts = counts_of(kind, R, E, R)
    q, offsets = kb.quantize_f4(W), offsets_of(counts)
    Y = kb.linear_grouped_f4(X, q, offsets)
    at = 0
    for e, c in enumerate(counts):
        if c:
            check(Y[at: at + c], X[at: at + c], W[e])
        at += c
    assert torch.equal(kb.gemm_grouped_f4(kb.quantize_f4_tokens(X), q, offsets, dtype=torch.float16), Y)


def test_rows_of_no_expert_are_left(cuda):
    import torch
    import kebab_b200 as kb
    for R, first, counts in ((300, 7, [100, 0, 150]), (20, 3, [5, 4, 0])):
        X, W = operands(R, 256, 256, 1, "bfloat16", 3)
        q = kb.quantize_f4(W)
        Y = torch.full((R, 256), 7.0, dtype=torch.bfloat16, device="cuda")
        kb.linear_grouped_f4(X, q, offsets_of(counts, first=first), Y=Y)
        assert (Y[:first] == 7).all() and (Y[first + sum(counts):] == 7).all()
        at = first
        for e, c in enumerate(counts):
            if c:
                check(Y[at: at + c], X[at: at + c], W[e])
            at += c


def test_output_at_a_pitch(cuda):
    import torch
    import kebab_b200 as kb
    for M, N, K in ((5, 300, 256), (300, 520, 512), (900, 1001, 96)):
        X, W = operands(M, N, K)
        q = kb.quantize_f4(W)
        want = kb.linear_f4(X, q)
        for extra, shift in ((8, 0), (3, 1)):
            Y = pitched(torch.zeros((M, N), dtype=X.dtype, device="cuda"), extra, shift)
            around = Y.as_strided((M - 1, extra), Y.stride(), Y.storage_offset() + N)
            kb.linear_f4(pitched(X, extra, shift), q, Y=Y)
            assert torch.equal(Y, want) and torch.isnan(around).all()


@pytest.mark.parametrize("M", [3, 70, 300, 1500])
def test_non_finite_rows_stay_to_themselves(cuda, M):
    import torch
    import kebab_b200 as kb
    X, W = operands(M, 520, 512, M)
    q, clean = kb.quantize_f4(W), None
    clean = kb.linear_f4(X, q)
    X[1, 40] = float("inf")
    X[M - 1, 511] = float("nan")
    Y = kb.linear_f4(X, q)
    bad = torch.zeros(M, dtype=torch.bool, device="cuda")
    bad[[1, M - 1]] = True
    assert torch.isnan(Y[bad]).all() and torch.equal(Y[~bad], clean[~bad])
    W[7, 100] = float("inf")
    Y = kb.linear_f4(X, kb.quantize_f4(W))
    assert torch.isnan(Y[:, 7]).all() and torch.equal(Y[~bad][:, 8:], clean[~bad][:, 8:])


def test_zero_blocks_and_small_scales(cuda):
    import torch
    import kebab_b200 as kb
    X, W = operands(40, 256, 512)
    X[:, 64:256] = 0
    W[:, 300:] = 0
    X[3] = 0
    check(kb.linear_f4(X, kb.quantize_f4(W)), X, W)
    X, W = operands(40, 256, 512)
    check(kb.linear_f4(X * 2.0 ** -60, kb.quantize_f4(W * 2.0 ** -50)), X * 2.0 ** -60, W * 2.0 ** -50)
    check(kb.linear_f4(X * 2.0 ** 60, kb.quantize_f4(W * 2.0 ** 50)), X * 2.0 ** 60, W * 2.0 ** 50)


def test_empty(cuda):
    import torch
    import kebab_b200 as kb
    X, W = operands(4, 64, 96, E=2)
    q = kb.quantize_f4(W)
    assert kb.linear_f4(X[:0], kb.quantize_f4(W[0])).shape == (0, 64)
    assert kb.linear_grouped_f4(X[:0], q, offsets_of([0, 0])).shape == (0, 64)
    assert kb.quantize_f4_tokens(X[:0]).codes.shape == (0, 48)
    Y = torch.full((4, 64), 7.0, dtype=X.dtype, device="cuda")
    kb.linear_grouped_f4(X, q, offsets_of([0, 0]), Y=Y)
    assert (Y == 7).all()


def test_captured(cuda):
    import torch
    import kebab_b200 as kb
    W = randn((5, 512, 1024), torch.bfloat16, 2)
    q, one = kb.quantize_f4(W), kb.quantize_f4(W[0])
    offsets = offsets_of([3, 0, 200, 90, 7])
    for M in (300,):
        X = randn((M, 1024), torch.bfloat16, 1)
        step = lambda: (kb.linear_f4(X, one), kb.linear_f4(X[:5], one), kb.linear_grouped_f4(X, q, offsets))  # noqa: E731
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for seed in (5, 6):
            X.copy_(randn((M, 1024), torch.bfloat16, seed))
            graph.replay()
            for a, b in zip(out, step()):
                assert torch.equal(a, b)


def test_other_stream(cuda):
    import torch
    import kebab_b200 as kb
    X, W = operands(300, 512, 1024)
    want = kb.linear_f4(X, kb.quantize_f4(W))
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    got = kb.linear_f4(X, kb.quantize_f4(W, stream=stream), stream=stream)
    stream.synchronize()
    assert torch.equal(got, want)


def test_refusals(cuda):
    import torch
    import kebab_b200 as kb
    X, W = operands(4, 64, 96)
    q, t, off = kb.quantize_f4(W), kb.quantize_f4_tokens(X), offsets_of([2, 2])
    stack = kb.quantize_f4(torch.stack([W, W]))
    for call in (lambda: kb.linear_f4(X, W), lambda: kb.linear_f4(X, t), lambda: kb.linear_f4(X[:, :64], q), lambda: kb.linear_f4(X, stack),
                 lambda: kb.linear_grouped_f4(X, q, off), lambda: kb.linear_grouped_f4(X, stack, off[:2]), lambda: kb.linear_grouped_f4(X, stack, None),
                 lambda: kb.linear_f4(X.float(), q), lambda: kb.linear_f4(X, q, bias=X[0, :64].float()), lambda: kb.linear_f4(X, q, Y=X),
                 lambda: kb.gemm_f4(q, q), lambda: kb.gemm_f4(t, q, dtype=torch.float32), lambda: kb.gemm_f4(kb.F4Tokens(t.codes[:3], t.scales), q),
                 lambda: kb.gemm_f4(t, kb.F4(q.codes, q.scales[:, :0])), lambda: kb.quantize_f4(X[0]), lambda: kb.quantize_f4(W[:0]),
                 lambda: kb.quantize_f4(W.T), lambda: kb.quantize_f4_tokens(X[:, :0]), lambda: kb.dequantize_f4(q, 200), lambda: kb.dequantize_f4(q, 96, torch.int8),
                 lambda: kb.dequantize_f4(t, 96), lambda: kb.linear_f4(X, kb.F4(q.codes[::2], q.scales))):
        with pytest.raises(kb.KebabError):
            call()
