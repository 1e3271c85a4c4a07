"""Products whose waits run out: the call ends, the status says so, and the
next call is right."""
import pytest

from operator_util import counts_of, offsets_of, randn

pytestmark = pytest.mark.gpu


def check_aborts(call, expires=False):
    """Repeats with a budget of 1 us a wait. Whether a short wait reaches it is
    chance (it is looked at every 64 polls); an epilogue's wait for a main loop
    of a millisecond does."""
    import torch
    import kebab_b200 as kb
    want = call()
    assert kb.device_status()[0] == kb.OK
    kb.set_wait_timeout_us(1)
    try:
        for _ in range(4 if expires else 20):
            got = call()
            rc, code = kb.device_status()
            assert rc == kb.ETIMEOUT or (rc == kb.OK and not expires and torch.equal(got, want)), hex(code)
    finally:
        kb.set_wait_timeout_us(2000000)
    for _ in range(3):
        assert torch.equal(call(), want)
    assert kb.device_status()[0] == kb.OK


@pytest.mark.parametrize("R,E,N,K", [(8, 1, 1024, 8192), (100, 3, 520, 4096), (60, 40, 1024, 512)])
def test_few_rows(cuda, R, E, N, K):
    """Split over k by clusters (the first two) and by single CTAs."""
    import torch
    import kebab_b200 as kb
    X, W, offsets = randn((R, K), torch.bfloat16, 1), randn((E, N, K), torch.bfloat16, 2), offsets_of(counts_of("even", R, E))
    check_aborts(lambda: kb.gemm_grouped(X, W, offsets))
    wq, ws = kb.quantize_i8(W[0])
    check_aborts(lambda: kb.linear_i8(X, wq, ws))


@pytest.mark.parametrize("N", [2056, 8200])
def test_persistent(cuda, N):
    """Panels of 256 and of 512 rows, groups with odd ends and without rows."""
    import torch
    import kebab_b200 as kb
    counts, K = [900, 0, 257, 1, 1500, 255, 1024, 33, 512, 130], 520
    R, E, offsets = sum(counts), len(counts), offsets_of(counts)
    X, W, dY = randn((R, K), torch.float16, 1), randn((E, N, K), torch.float16, 2), randn((R, N), torch.float16, 3)
    check_aborts(lambda: kb.gemm_grouped(X, W, offsets))
    check_aborts(lambda: kb.gemm_grouped(dY, W, offsets, opmode="RR"))
    check_aborts(lambda: kb.gemm_grouped_dw(X, dY, offsets))
    wq, ws = kb.quantize_i8(W)
    check_aborts(lambda: kb.linear_grouped_i8(X, wq, ws, offsets))


def ramp(*shape):
    """Small whole numbers, their sums exact."""
    import torch
    return (torch.arange(shape[-1], device="cuda") % 7).to(torch.bfloat16).expand(*shape).contiguous()


@pytest.mark.parametrize("R,N,K", [(8, 128, 1 << 22), (8, 20480, 1 << 18), (512, 5120, 1 << 19)])
def test_epilogue_gives_up(cuda, R, N, K):
    """Clusters that split k, single CTAs, and pairs with several tiles each."""
    import kebab_b200 as kb
    X, W, offsets = ramp(R, K), ramp(1, N, K), offsets_of([R])
    check_aborts(lambda: kb.gemm_grouped(X, W, offsets), expires=True)


def test_epilogue_gives_up_in_dw(cuda):
    import kebab_b200 as kb
    R = (1 << 20) + 5
    X, dY, offsets = ramp(R, 2560), ramp(R, 2560), offsets_of([R, 0])
    check_aborts(lambda: kb.gemm_grouped_dw(X, dY, offsets), expires=True)


def test_epilogue_gives_up_in_split_gemm(cuda):
    """The dense swap-AB rung, which splits k over a cluster in the same way."""
    import kebab_b200 as kb
    A, B = ramp(8, 1 << 22), ramp(128, 1 << 22)
    check_aborts(lambda: kb.gemm(A, B, version=106), expires=True)
