"""How much of a hidden value few-token layers keep, on whole numbers whose sums are exact."""
import pytest

from operator_util import UNIT, assert_within, dtype_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("T", [1, 5, 16])
def test_hidden_values_keep_their_bits(cuda, T, dtype):
    """Hidden values of 21 bits, pairs of which differ in the last seven: their differences are the outputs. Every
    product, sum and difference is a whole number of 2^-14 below 2^21 of them, exact in FP32 and (seven bits) in the
    output's type; silu(32) is 32 in FP32."""
    import torch
    import kebab_b200 as kb
    H, D, dt = 64, 96, dtype_of(dtype)
    g = torch.Generator(device="cuda")
    g.manual_seed(T)
    digits = torch.randint(64, 128, (D, 3), generator=g, device="cuda").double()
    digits[1::2, :2] = digits[::2, :2]  # a pair differs in the last digit
    x = torch.zeros((T, H), device="cuda")
    x[:, 0], x[:, 1], x[:, 2] = 1, 2.0 ** -7, 2.0 ** -14
    w_in = torch.zeros((1, 2 * D, H), device="cuda")
    w_in[0, :D, 0] = 32
    w_in[0, D:, :3] = digits.float()
    w_out = torch.zeros((1, H, D), device="cuda")
    n = torch.arange(H, device="cuda") % (D // 2)
    w_out[0, torch.arange(H), 2 * n], w_out[0, torch.arange(H), 2 * n + 1] = 1, -1
    y = kb.expert_layer(x.to(dt), torch.zeros((1, H), device="cuda"), w_in.to(dt), w_out.to(dt), 1)
    want = 32 * 2.0 ** -14 * (digits[::2, 2] - digits[1::2, 2])[n].expand(T, H)
    assert torch.equal(y.double(), want)


def test_hidden_values_up_to_the_largest(cuda):
    """A hidden value between the largest of BF16 and that of FP32, brought back by a small weight: 2^128 (1 - 2^-11)
    times 2^-120, rounded once."""
    import torch
    import kebab_b200 as kb
    x = torch.zeros((2, 64), device="cuda")
    x[:, :2] = 2.0 ** 32
    w_in = torch.zeros((1, 16, 64), device="cuda")
    w_in[0, 0, 0] = 2.0 ** 32
    w_in[0, 8, 0], w_in[0, 8, 1] = 2.0 ** 32, -2.0 ** 21
    w_out = torch.zeros((1, 64, 8), device="cuda")
    w_out[0, :, 0] = 2.0 ** -120
    y = kb.expert_layer(x.bfloat16(), torch.zeros((1, 64), device="cuda"), w_in.bfloat16(), w_out.bfloat16(), 1)
    assert torch.equal(y, torch.full_like(y, 256.0))


# What a sum of N positive numbers loses where the matrix unit adds 512 of them, 16 a step, and the rest is added in
# FP32: a step cuts off at most 2^-22 of what has been summed, so 32 steps 2^-17 of a run's sum; up to 64 additions of
# runs, to nearest, lose half of 2^-18 of the whole. In one run, N / 16 steps would lose about as many times 2^-25.
LONG, LOST = 32768, 2.0 ** -16


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("T", [1, 11])
def test_long_sums_of_the_first_product(cuda, T, dtype):
    """Up values that are long sums of positive numbers, less the same sum rounded to BF16: what is left shows the sum's
    low bits in the output."""
    import torch
    import kebab_b200 as kb
    H, D, dt = LONG, 32, dtype_of(dtype)
    g = torch.Generator(device="cuda")
    g.manual_seed(T)
    up = (0.5 + 0.5 * torch.rand((D, H), generator=g, device="cuda")).bfloat16().to(dt).double()
    x = (0.5 + 0.5 * torch.rand((H,), generator=g, device="cuda")).bfloat16().to(dt)
    x[0] = 1
    S = up[::2] @ x.double()
    up[1::2] = 0
    up[1::2, 0] = S.bfloat16().double()
    w_in = torch.zeros((1, 2 * D, H), dtype=dt, device="cuda")
    w_in[0, :D, 0] = 32
    w_in[0, D:] = up.to(dt)
    assert torch.equal(w_in[0, D:].double(), up)
    w_out = torch.zeros((1, H, D), dtype=dt, device="cuda")
    n = torch.arange(H, device="cuda") % (D // 2)
    w_out[0, torch.arange(H), 2 * n], w_out[0, torch.arange(H), 2 * n + 1] = 2.0 ** -10, -2.0 ** -10
    y = kb.expert_layer(x.repeat(T, 1), torch.zeros((1, H), device="cuda"), w_in, w_out, 1)
    want = (2.0 ** -5 * (S - up[1::2, 0]))[n].expand(T, H)
    # F16 keeps 22 bits of the two hidden values.
    assert_within(y, want, 2.0 ** -5 * S[n] * (LOST + 2.0 ** -21) + UNIT[dtype] * (want.abs() + S[n] * 2.0 ** -20))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("T", [1, 11])
def test_long_sums_of_the_second_product(cuda, T, dtype):
    """Outputs that are long sums of positive numbers, less the same sum rounded to BF16, which comes first."""
    import torch
    import kebab_b200 as kb
    H, D, dt = 64, LONG, dtype_of(dtype)
    g = torch.Generator(device="cuda")
    g.manual_seed(T)
    x = torch.zeros((T, H), dtype=dt, device="cuda")
    x[:, 0] = 1
    w_in = torch.zeros((1, 2 * D, H), dtype=dt, device="cuda")
    w_in[0, :D, 0] = 32
    h = (0.5 + 0.5 * torch.rand((D,), generator=g, device="cuda")).bfloat16().to(dt)
    h[0] = 1
    w_in[0, D:, 0] = h / 32  # the hidden values are h
    out = (0.5 + 0.5 * torch.rand((H, D), generator=g, device="cuda")).bfloat16().to(dt).double()
    S = out[:, 1:] @ h[1:].double()
    out[:, 0] = -S.bfloat16().double()
    w_out = out.to(dt)[None].contiguous()
    assert torch.equal(w_out[0].double(), out)
    y = kb.expert_layer(x, torch.zeros((1, H), device="cuda"), w_in, w_out, 1)
    want = (S + out[:, 0]).expand(T, H)
    # The run with the first number loses of S, the others of their own sums.
    assert_within(y, want, 2 * LOST * S + UNIT[dtype] * (want.abs() + 2 * LOST * S))


def test_codes_of_the_largest_tokens(cuda):
    """Rows of x whose largest value times 127 is beyond FP32, against 64 bits; the weights' scales bring the hidden
    values back to ordinary ones."""
    import torch
    import kebab_b200 as kb
    from test_layer_gpu import make, reference
    x, router, w_in, w_out = make(6, 1, 256, 64, "bfloat16", 9)
    top = torch.tensor([torch.finfo(torch.bfloat16).max, 2.0 ** 127, 2.8e36, 2.6e36, 2.0 ** 100, 2.0 ** 121], device="cuda")
    x = (x.float() / x.float().abs().amax(1, keepdim=True) * top[:, None]).clamp(-top[0], top[0]).bfloat16()
    assert torch.isfinite(x).all()
    (qi, si), (qo, so) = kb.quantize_i8(w_in), kb.quantize_i8(w_out)
    si = si * 2.0 ** -120
    y = kb.expert_layer_i8(x, router * 0, qi, si, qo, so, 1)
    want, bound = reference(x, router * 0, qi, qo, 1, True, (si, so))
    assert (want.abs().amax(1)[:4] > 2.0 ** -12).all()
    assert_within(y, want, bound)
