"""Which operators a served layer takes for a few tokens: those that the few-token layer refuses, or is slow for, go
through the separate ones, to the same bits."""
import pytest

from operator_util import randn

pytestmark = pytest.mark.gpu


def layer(width, hidden, experts, k):
    import torch
    from kebab_b200.moe import MoE
    torch.manual_seed(1)
    return MoE(width, hidden, experts, k)


def test_weights_that_are_not_contiguous(cuda):
    import torch
    m = layer(64, 32, 8, 2)
    x = randn((3, 64), torch.bfloat16, 1)
    with torch.no_grad():
        want = m(x)[0]
        m.w_in.data = torch.empty((8, 64, 128), dtype=torch.bfloat16, device="cuda")[:, :, :64].copy_(m.w_in.data)
        assert torch.equal(m.serve(16)(x), want)


@pytest.mark.parametrize("width,hidden,bits", [(2048, 1000, 8), (2047, 1001, 16), (2047, 1001, 8)])
def test_large_unaligned_weights(cuda, width, hidden, bits):
    import torch
    m = layer(width, hidden, 8, 4)
    x = randn((5, width), torch.bfloat16, 1)
    with torch.no_grad():
        assert torch.equal(m.serve(bits)(x), m(x)[0] if bits == 16 else m.quantize()(x))


@pytest.mark.parametrize("width,hidden,bits", [(65, 33, 8), (65, 33, 16), (512, 128, 8), (512, 128, 16), (2048, 1000, 16)])
def test_the_others_take_the_layer(cuda, width, hidden, bits):
    import torch
    import kebab_b200 as kb
    m = layer(width, hidden, 8, 4)
    x = randn((5, width), torch.bfloat16, 1)
    with torch.no_grad():
        if bits == 16:
            want = kb.expert_layer(x, m.router, m.w_in, m.w_out, 4)
        else:
            want = kb.expert_layer_i8(x, m.router, *kb.quantize_i8(m.w_in), *kb.quantize_i8(m.w_out), 4)
        assert torch.equal(m.serve(bits)(x), want)
