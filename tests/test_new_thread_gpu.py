"""Calls that are the first of a host thread: it has no CUDA context yet, which
the tensor maps of the products need."""
import threading

import pytest

from operator_util import offsets_of, randn

pytestmark = pytest.mark.gpu


def test_first_call_of_a_thread(cuda):
    import torch
    import kebab_b200 as kb
    X, W = randn((300, 512), torch.bfloat16, 1), randn((2, 1024, 512), torch.bfloat16, 2)
    offsets, (wq, ws), q = offsets_of([100, 200]), kb.quantize_i8(W[0]), kb.quantize_f4(W)
    xq, xs = kb.quantize_i8(X)
    t = kb.quantize_f4_tokens(X)
    few, router, w_out = X[:3].contiguous(), randn((2, 512), torch.float32, 3), randn((2, 512, 512), torch.bfloat16, 4)
    calls = [lambda: kb.gemm_grouped(X, W, offsets), lambda: kb.gemm_i8(xq, xs, wq, ws), lambda: kb.gemm_grouped_f4(t, q, offsets),
             lambda: kb.gemm_f4(t, kb.F4(q.codes[0], q.scales[0])), lambda: kb.expert_layer(few, router, W, w_out, 1),
             lambda: kb.gemm(X[:296], W[0], version=104), lambda: kb.rms_norm(X, ws[:512].contiguous())[0]]
    for call in calls:
        want, got = call(), []  # the first call leaves the allocator's cache full
        torch.cuda.synchronize()

        def run():
            try:
                got.append(call())
            except Exception as e:  # noqa: BLE001
                got.append(e)

        thread = threading.Thread(target=run)
        thread.start()
        thread.join()
        torch.cuda.synchronize()
        assert isinstance(got[0], torch.Tensor), got[0]
        assert torch.equal(got[0], want)
