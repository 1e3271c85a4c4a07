"""Refusals of the expert operators that take CUDA tensors to reach."""
import pytest

from operator_util import randn

pytestmark = pytest.mark.gpu


def test_sizes_that_would_be_negative(cuda):
    import torch
    import kebab_b200 as kb
    x = randn((4, 8), torch.float16, 1)
    slots = torch.zeros((4, 1), dtype=torch.int32, device="cuda")
    for call in (lambda: kb.gemm_grouped_dw(x, x, torch.zeros(0, dtype=torch.int32, device="cuda")),
                 lambda: kb.gemm_grouped_dw(x, x, torch.zeros(1, dtype=torch.int32, device="cuda")),
                 lambda: kb.dispatch(x, slots, rows=-1)):
        with pytest.raises(kb.KebabError) as e:
            call()
        assert e.value.code == kb.EINVAL
