"""Waits that certainly run out in the few-token layers and the 4-bit products: a budget of a microsecond for waits that
last hundreds (blocks without hidden values wait for those that have them, epilogues for a whole main loop)."""
import pytest

from operator_util import offsets_of
from test_grouped_aborts_gpu import check_aborts, ramp
from test_int8_unaligned_gpu import codes, scales

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_layer_gives_up_at_the_grid_barrier(cuda, dtype):
    """64 of the blocks have one hidden value each, of 2^20 terms; the others wait for it."""
    import torch
    import kebab_b200 as kb
    dt, H, D = getattr(torch, dtype), 1 << 20, 64
    x, w_in, w_out = ramp(8, H).to(dt) * 2.0 ** -10, ramp(1, 2 * D, H).to(dt), ramp(1, H, D).to(dt) * 2.0 ** -20
    check_aborts(lambda: kb.expert_layer(x, torch.zeros((1, H), device="cuda"), w_in, w_out, 1), expires=True)


def test_8_bit_layer_gives_up_at_the_grid_barrier(cuda):
    """The same with rows that are copied value by value."""
    import torch
    import kebab_b200 as kb
    H, D = 131071, 64
    x, qi, qo, si, so = ramp(8, H), codes((1, 2 * D, H), 1), codes((1, H, D), 2), scales((1, 2 * D), 3) * 2.0 ** -20, scales((1, H), 4)
    check_aborts(lambda: kb.expert_layer_i8(x, torch.zeros((1, H), device="cuda"), qi, si, qo, so, 1), expires=True)


@pytest.mark.parametrize("R,N,K", [(8, 128, 1 << 22), (8, 20480, 1 << 18), (512, 5120, 1 << 19)])
def test_f4_epilogue_gives_up(cuda, R, N, K):
    """Clusters that split k, single CTAs, and pairs with several tiles each."""
    import kebab_b200 as kb
    q, X, offsets = kb.quantize_f4(ramp(1, N, K)), kb.quantize_f4_tokens(ramp(R, K)), offsets_of([R])
    check_aborts(lambda: kb.gemm_grouped_f4(X, q, offsets), expires=True)
