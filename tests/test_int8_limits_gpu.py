"""8-bit integer operators: the stream that a copy inside a call runs on, the
longest sums, and weights that are written right before they are read."""
import pytest

from operator_util import assert_within, randn
from test_int8_gpu import i8_bound

pytestmark = pytest.mark.gpu


def test_quantize_strided_stack_on_a_stream(cuda):
    """A stack that cannot be viewed as rows is copied in the call: on the
    stream of the call, not on the current one (which is held back here)."""
    import torch
    import kebab_b200 as kb
    X = randn((3, 512, 1024), torch.bfloat16, 1).transpose(1, 2)
    want = kb.quantize_i8(X.contiguous())
    side = torch.cuda.Stream()
    junk = torch.full((3, 1024, 512), 77.0, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    del junk  # the memory that a copy on the current stream would take
    torch.cuda._sleep(200_000_000)
    q, scale = kb.quantize_i8(X, stream=side)
    side.synchronize()
    with torch.cuda.stream(side):
        same = torch.equal(q, want[0]) and torch.equal(scale, want[1])
    torch.cuda.synchronize()
    assert q.shape == X.shape and scale.shape == X.shape[:-1] and same


def test_quantize_refuses_empty_rows(cuda):
    import torch
    import kebab_b200 as kb
    for shape in ((0,), (2, 0), (2, 3, 0), (0, 4, 0)):
        with pytest.raises(kb.KebabError) as e:
            kb.quantize_i8(torch.zeros(shape, device="cuda"))
        assert e.value.code == kb.EINVAL, shape
    q, scale = kb.quantize_i8(torch.zeros((0, 3, 8), device="cuda"))
    assert q.shape == (0, 3, 8) and scale.shape == (0, 3)


@pytest.mark.parametrize("M,N", [(3, 300), (200, 300), (1000, 2561)])
def test_longest_sums(cuda, M, N):
    """Codes of -128 on both sides over the longest K that is admitted: sums
    just below 2^31, in each kernel."""
    import torch
    import kebab_b200 as kb
    K = 131071
    q = torch.full((M, K + 1), -128, dtype=torch.int8, device="cuda")
    wq = torch.full((N, K + 1), -128, dtype=torch.int8, device="cuda")
    s, ws = torch.full((M,), 2.0 ** -20, device="cuda"), torch.full((N,), 2.0 ** -6, device="cuda")
    want = torch.full((M, N), float(K << 14) * 2.0 ** -26, dtype=torch.float64, device="cuda")
    bound = i8_bound(want, want.abs(), torch.bfloat16)
    assert_within(kb.gemm_i8(q[:, :K], s, wq[:, :K], ws), want, bound, "Y")
    offsets = torch.tensor([0, M], dtype=torch.int32, device="cuda")
    assert_within(kb.gemm_grouped_i8(q[:, :K], s, wq[None, :, :K], ws[None], offsets), want, bound, "grouped")
    if M == 3:  # rows that TMA cannot address
        a, b = q.view(-1)[:M * K].view(M, K), wq.view(-1)[:N * K].view(N, K)
        assert_within(kb.gemm_i8(a, s, b, ws), want, bound, "Y")


def test_longest_sums_refused(cuda):
    import torch
    import kebab_b200 as kb
    K = 131072
    q = torch.full((8, K), -128, dtype=torch.int8, device="cuda")
    s = torch.ones(8, device="cuda")
    for call in (lambda: kb.gemm_i8(q, s, q, s),
                 lambda: kb.gemm_grouped_i8(q, s, q[None], s[None], torch.tensor([0, 8], dtype=torch.int32, device="cuda"))):
        with pytest.raises(kb.KebabError) as e:
            call()
        assert e.value.code == kb.EINVAL and "overflow" in str(e.value)
    # Codes of linear_i8's activations end at -127: K = 131072 stays below 2^31.
    x = torch.ones((8, K), dtype=torch.bfloat16, device="cuda")
    y = kb.linear_i8(x, q, s * 2.0 ** -20)
    want = torch.full((8, 8), -127.0 * 128 * K * 2.0 ** -20 / 127, dtype=torch.float64, device="cuda")
    assert_within(y, want, i8_bound(want, want.abs(), torch.bfloat16) + want.abs() * 2.0 ** -23, "Y")


@pytest.mark.parametrize("M", [1, 64, 300])
def test_weights_written_right_before(cuda, M):
    """linear_i8 fetches weights while it still quantises; what the stream
    wrote into them just before has to be there."""
    import torch
    import kebab_b200 as kb
    N, K = 2048, 4096
    x = randn((M, K), torch.bfloat16, 1)
    stacks = [randn((N, K), torch.bfloat16, 2 + i) for i in range(3)]
    want = []
    for w in stacks:
        q = kb.quantize_i8(w)
        torch.cuda.synchronize()
        want.append(kb.linear_i8(x, *q))
        torch.cuda.synchronize()
    wq, ws = torch.zeros((N, K), dtype=torch.int8, device="cuda"), torch.zeros(N, device="cuda")
    got = []
    for i in range(30):
        q, s = kb.quantize_i8(stacks[i % 3])
        if i % 2:  # written by a plain copy, or by the framework's own kernel
            wq.copy_(q), ws.copy_(s)
            q, s = wq, ws
        got.append(kb.linear_i8(x, q, s))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % 3]), i
