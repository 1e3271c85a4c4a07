"""8-bit integer operators: the stream that a copy inside a call runs on."""
import pytest

from operator_util import randn

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
