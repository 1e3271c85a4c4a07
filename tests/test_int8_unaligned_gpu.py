"""8-bit products of operands on any boundary: the same bits as of aligned copies
(sums are exact, so that the order of their terms does not count)."""
import pytest

from operator_util import counts_of, offsets_of, pitched, randn
from test_grouped_aborts_gpu import check_aborts

pytestmark = pytest.mark.gpu


def codes(shape, seed):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-128, 128, shape, generator=g, device="cuda", dtype=torch.int8)


def scales(shape, seed):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.rand(shape, generator=g, device="cuda") + 0.5


def aligned(t):
    """`t` with rows padded to 16 bytes."""
    import torch
    wide = torch.zeros((*t.shape[:-1], -(-t.shape[-1] // 16) * 16), dtype=t.dtype, device=t.device)
    wide[..., : t.shape[-1]] = t
    return wide[..., : t.shape[-1]]


@pytest.mark.parametrize("M,N", [(1, 1), (3, 130), (40, 264), (130, 127), (300, 520)])
@pytest.mark.parametrize("K", [1, 15, 16, 17, 31, 33, 63, 127, 128, 129, 160, 255, 272, 1385])
def test_dense(cuda, M, N, K):
    import torch
    import kebab_b200 as kb
    q, s, wq, ws = codes((M, K), M), scales((M,), 1), codes((N, K), N), scales((N,), 2)
    bias = randn((N,), torch.bfloat16, 3)
    want = kb.gemm_i8(aligned(q), s, aligned(wq), ws, bias=bias)
    for extra, shift in ((0, 0), (1, 0), (0, 5), (3, 15), (16, 1), (5, 8)):
        assert torch.equal(kb.gemm_i8(pitched(q, extra, shift), s, pitched(wq, extra, shift), ws, bias=bias), want), (extra, shift)
    assert torch.equal(kb.gemm_i8(aligned(q), s, pitched(wq, 1, 3), ws, bias=bias), want)
    assert torch.equal(kb.gemm_i8(pitched(q, 1, 3), s, aligned(wq), ws, bias=bias), want)


@pytest.mark.parametrize("kind", ["even", "one", "ragged", "ends"])
@pytest.mark.parametrize("R,E,N,K", [(1, 4, 128, 129), (100, 3, 300, 1000), (600, 7, 200, 333), (1500, 5, 130, 72)])
def test_grouped(cuda, kind, R, E, N, K):
    import torch
    import kebab_b200 as kb
    counts = counts_of(kind, R, E)
    q, s, wq, ws, offsets = codes((R, K), 1), scales((R,), 2), codes((E, N, K), 3), scales((E, N), 4), offsets_of(counts)
    want = kb.gemm_grouped_i8(aligned(q), s, aligned(wq), ws, offsets)
    got = kb.gemm_grouped_i8(q, s, wq, ws, offsets)
    rows = sum(counts)
    assert torch.equal(got[:rows], want[:rows])


@pytest.mark.parametrize("H", [100, 1385, 4100])
def test_normed_single_token(cuda, H):
    """A token's codes have a pitch of whole 16 bytes, which one row does not show."""
    import torch
    import kebab_b200 as kb
    x, w = randn((1, H), torch.bfloat16, 1), torch.ones(H, device="cuda")
    wq, ws = codes((200, H), 2), scales((200,), 3)
    n = kb.rms_norm_i8(x, w)
    want = kb.gemm_i8(aligned(n.codes), n.scale, aligned(wq), ws)
    assert torch.equal(kb.gemm_i8(n.codes, n.scale, wq, ws), want)
    assert torch.equal(kb.gemm_i8(n.codes, n.scale, aligned(wq), ws), want)


@pytest.mark.parametrize("M,N,K", [(5, 300, 20001), (700, 2000, 1001)])
def test_waits_that_run_out(cuda, M, N, K):
    import kebab_b200 as kb
    q, s, wq, ws = codes((M, K), 1), scales((M,), 2), codes((N, K), 3), scales((N,), 4)
    check_aborts(lambda: kb.gemm_i8(q, s, wq, ws))


def test_captured_and_on_several_streams(cuda):
    import torch
    import kebab_b200 as kb
    cases = [(codes((M, K), M), scales((M,), 1), codes((300, K), K), scales((300,), 2)) for M, K in ((1, 1001), (70, 333), (400, 2047), (9, 4100))]
    want = [kb.gemm_i8(*c) for c in cases]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [kb.gemm_i8(*c) for c in cases]
    for _ in range(3):
        for t in out:
            t.zero_()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(10):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append([kb.gemm_i8(*c) for _ in range(3)])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, b in zip(got, want) for a in g)
