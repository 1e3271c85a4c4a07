"""4-bit linear layers of so few rows that the product quantises them itself:
the same bits as the quantisation and the product one after the other."""
import pytest

from operator_util import dtype_of, offsets_of, pitched, randn
from test_grouped_aborts_gpu import check_aborts

pytestmark = pytest.mark.gpu


def same(a, b):
    """The same bits, or NaN in both."""
    import torch
    return torch.equal(torch.nan_to_num(a, nan=7.0), torch.nan_to_num(b, nan=7.0)) and torch.equal(a.isnan(), b.isnan())


@pytest.mark.parametrize("N,K", [(1, 1), (130, 31), (64, 129), (257, 1000), (1024, 2048), (300, 8200), (8192, 776), (96, 20008)])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_linear(cuda, N, K, dtype):
    import torch
    import kebab_b200 as kb
    W, bias = kb.quantize_f4(randn((N, K), dtype_of(dtype), 1)), randn((N,), dtype_of(dtype), 2)
    for M in range(1, 9):
        X = randn((M, K), dtype_of(dtype), M) * torch.logspace(-3, 3, M, device="cuda").to(dtype_of(dtype))[:, None]
        want = kb.gemm_f4(kb.quantize_f4_tokens(X), W, bias=bias, dtype=X.dtype)
        for extra, shift in ((0, 0), (8, 0), (3, 1)):
            assert torch.equal(kb.linear_f4(pitched(X, extra, shift), W, bias=bias), want), (M, extra, shift)


@pytest.mark.parametrize("K", [96, 1000, 4096])
def test_blocks_without_values(cuda, K):
    """Zeros, subnormal blocks, infinities and NaN, each in a block of its own row."""
    import torch
    import kebab_b200 as kb
    W = kb.quantize_f4(randn((200, K), torch.bfloat16, 1))
    X = randn((6, K), torch.bfloat16, 2)
    X[0] = 0
    X[1, 32:64] = 1e-39
    X[2, K - 1] = float("inf")
    X[3, 5] = float("nan")
    X[4, :32] = 0
    Y = kb.linear_f4(X, W)
    assert same(Y, kb.gemm_f4(kb.quantize_f4_tokens(X), W))
    assert not Y[0].any() and Y[2:4].isnan().all() and Y[4:].isfinite().all()


@pytest.mark.parametrize("counts", [[0, 1, 0, 5], [6, 0, 0, 0], [1, 1, 1, 1], [0, 0, 0, 2], [0, 0, 0, 0]])
def test_grouped(cuda, counts):
    import torch
    import kebab_b200 as kb
    N, K = 264, 1032
    W = kb.quantize_f4(randn((4, N, K), torch.float16, 1))
    X, rows = randn((6, K), torch.float16, 2), sum(counts)
    Y = torch.full((6, N), 3.0, dtype=X.dtype, device="cuda")
    kb.linear_grouped_f4(X, W, offsets_of(counts), Y=Y)
    want = kb.gemm_grouped_f4(kb.quantize_f4_tokens(X), W, offsets_of(counts), dtype=X.dtype)
    assert torch.equal(Y[:rows], want[:rows]) and (Y[rows:] == 3).all()


@pytest.mark.parametrize("M", [1, 4, 6, 7, 40])
def test_output_on_the_input(cuda, M):
    """Y in X's place, and beside X in the rows of one buffer."""
    import torch
    import kebab_b200 as kb
    H = 1024
    W = kb.quantize_f4(randn((H, H), torch.bfloat16, 1))
    X = randn((M, H), torch.bfloat16, 2)
    want = kb.linear_f4(X, W)
    for _ in range(20):
        Y = X.clone()
        assert torch.equal(kb.linear_f4(Y, W, Y=Y), want)
    both = torch.cat([X, X], 1)
    kb.linear_f4(both[:, :H], W, Y=both[:, H:])
    assert torch.equal(both[:, H:], want) and torch.equal(both[:, :H], X)


def test_a_chain_of_layers(cuda):
    """Each call reads what the one before wrote, captured too: nothing starts on old rows."""
    import torch
    import kebab_b200 as kb
    H = 2048
    W = [kb.quantize_f4(randn((H, H), torch.bfloat16, i) * H ** -0.5) for i in range(4)]
    x = randn((3, H), torch.bfloat16, 9)

    def chain(step, x):
        for i in range(40):
            x = step(x, W[i % 4])
        return x

    want = chain(lambda x, w: kb.gemm_f4(kb.quantize_f4_tokens(x), w), x)
    assert torch.equal(chain(kb.linear_f4, x), want)
    graph, held = torch.cuda.CUDAGraph(), x.clone()
    with torch.cuda.graph(graph):
        out = chain(kb.linear_f4, held)
    for seed in (10, 11):
        held.copy_(randn((3, H), torch.bfloat16, seed))
        graph.replay()
        assert torch.equal(out, chain(lambda x, w: kb.gemm_f4(kb.quantize_f4_tokens(x), w), held))


@pytest.mark.parametrize("M,N,K", [(1, 1024, 8192), (6, 128, 20000), (5, 40000, 1024)])
def test_waits_that_run_out(cuda, M, N, K):
    import torch
    import kebab_b200 as kb
    X, W = randn((M, K), torch.bfloat16, 1), kb.quantize_f4(randn((N, K), torch.bfloat16, 2))
    check_aborts(lambda: kb.linear_f4(X, W))
    check_aborts(lambda: kb.linear_grouped_f4(X, kb.F4(W.codes[None], W.scales[None]), offsets_of([M])))


def test_several_streams(cuda):
    """Few rows on four streams at once, between layers and norms: the same bits as alone."""
    import torch
    import kebab_b200 as kb
    H, D, E = 1024, 512, 8
    W = kb.quantize_f4(randn((H, H), torch.bfloat16, 1) * H ** -0.5)
    stack = kb.quantize_f4(randn((3, H, H), torch.bfloat16, 2) * H ** -0.5)
    router, w_in, w_out = randn((E, H), torch.float32, 3), randn((E, 2 * D, H), torch.bfloat16, 4) * 0.03, randn((E, H, D), torch.bfloat16, 5) * 0.04
    w = torch.ones(H, device="cuda")
    offsets = [offsets_of([0, M - M // 2, M // 2]) for M in range(7)]

    def steps(x):
        for _ in range(6):
            x = kb.linear_f4(x, W)
            x = kb.linear_grouped_f4(x, stack, offsets[len(x)])
            x = kb.expert_layer(x, router, w_in, w_out, 2)
            x = kb.rms_norm(x, w)[0]
        return x

    xs = [randn((M, H), torch.bfloat16, M) for M in (1, 2, 5, 6)]
    want = [steps(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(5):
        got = []
        for x, s in zip(xs, streams):
            with torch.cuda.stream(s):
                got.append(steps(x))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
