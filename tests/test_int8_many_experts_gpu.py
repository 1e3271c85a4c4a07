"""Grouped 8-bit products of unaligned rows over many experts, and of short rows: the same bits as of aligned copies."""
import pytest

from operator_util import counts_of, offsets_of, pitched, randn
from test_int8_unaligned_gpu import aligned, codes, scales

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["even", "one", "ragged", "ends"])
@pytest.mark.parametrize("R,E,N,K", [(1021, 1024, 130, 101), (1021, 256, 72, 333), (5, 1000, 64, 17), (3000, 257, 8, 65), (700, 1024, 200, 9)])
def test_many_experts(cuda, kind, R, E, N, K):
    import torch
    import kebab_b200 as kb
    q, s, wq, ws, offsets = codes((R, K), 1), scales((R,), 2), codes((E, N, K), 3), scales((E, N), 4), offsets_of(counts_of(kind, R, E))
    want = kb.gemm_grouped_i8(aligned(q), s, aligned(wq), ws, offsets)
    assert torch.equal(kb.gemm_grouped_i8(q, s, wq, ws, offsets), want)


def test_rows_of_no_expert_are_left(cuda):
    """Rows before the first and behind the last group keep what was there."""
    import torch
    import kebab_b200 as kb
    for K in (9, 333):
        q, s, wq, ws = codes((300, K), 1), scales((300,), 2), codes((300, 40, K), 3), scales((300, 40), 4)
        offsets = offsets_of([0] * 100 + [150] + [0] * 198 + [70], first=40)
        Y = torch.full((300, 40), 7.0, dtype=torch.bfloat16, device="cuda")
        kb.gemm_grouped_i8(q, s, wq, ws, offsets, Y=Y)
        want = kb.gemm_grouped_i8(aligned(q), s, aligned(wq), ws, offsets)
        assert torch.equal(Y[40:260], want[40:260]) and (Y[:40] == 7).all() and (Y[260:] == 7).all()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("M,N", [(1, 1), (70, 64), (130, 300), (5000, 64), (20000, 8)])
@pytest.mark.parametrize("K", [1, 9, 31, 33, 50, 63])
def test_short_rows(cuda, M, N, K, dtype):
    """On both sides of the choice of kernel, with a bias."""
    import torch
    import kebab_b200 as kb
    dt = getattr(torch, dtype)
    q, s, wq, ws, bias = codes((M, K), M), scales((M,), 1), codes((N, K), N), scales((N,), 2), randn((N,), dt, 3)
    want = kb.gemm_i8(aligned(q), s, aligned(wq), ws, bias=bias, dtype=dt)
    assert torch.equal(kb.gemm_i8(q, s, wq, ws, bias=bias, dtype=dt), want)
    assert torch.equal(kb.gemm_i8(pitched(q, 1, 3), s, pitched(wq, 2, 5), ws, bias=bias, dtype=dt), want)
