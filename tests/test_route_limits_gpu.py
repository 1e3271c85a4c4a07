"""Routing from several host threads, at the sizes where a block passes 48 KB of
shared memory, and its gradient where a choice names no expert."""
import threading

import numpy as np
import pytest

from operator_util import UNIT, assert_within, dtype_of, randn
from test_experts_gpu import check_route

pytestmark = pytest.mark.gpu


def test_route_from_two_threads(cuda):
    """Threads that need different amounts of shared memory of one kernel (the
    C function by itself, so that they meet in it and not in the interpreter)."""
    import torch
    import kebab_b200 as kb
    from kebab_b200._call import function
    T, E = 300, 1024
    x = randn((T, E), torch.bfloat16, 1)
    want = {k: kb.route(x, k) for k in (9, 32)}
    f, size = function("kebab_route"), 148 * E * 4
    codes, differ = [], []

    def work(k):
        stream = torch.cuda.Stream()
        r = kb.Routing(*(torch.empty_like(t) for t in want[k]))
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        args = (kb.BF16, x.data_ptr(), E, T, E, k, 1, *(t.data_ptr() for t in r), ws.data_ptr(), size, stream.cuda_stream)
        torch.cuda.synchronize()
        codes.append({f(*args) for _ in range(20000)})
        stream.synchronize()
        differ.append([i for i, (a, b) in enumerate(zip(r, want[k])) if not torch.equal(a, b)])

    threads = [threading.Thread(target=work, args=(k,)) for k in (9, 32, 9, 32)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert codes == [{kb.OK}] * 4, kb.last_error()
    assert differ == [[]] * 4


@pytest.mark.parametrize("T,E,k", [(414, 831, 12), (414, 810, 12), (200, 840, 12), (100, 831, 10), (128, 1001, 5), (129, 1024, 8),
                                   (300, 512, 19), (300, 512, 20), (77, 600, 16), (300, 520, 20)])
def test_route_around_48_kb(cuda, T, E, k):
    check_route(randn((T, E), dtype_of("float32"), T), k, True)


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("T,E,k,dtype", [(5, 8, 3, "float32"), (77, 64, 6, "bfloat16"), (50, 130, 7, "float16"), (33, 1024, 32, "float32")])
def test_route_backward_dropped_choices(cuda, T, E, k, dtype, renormalize):
    """A choice whose expert is outside [0, E) contributes nothing: not to its
    own logit and not, through <w, dw>, to the others of its token."""
    import torch
    import kebab_b200 as kb
    logits, dw = randn((T, E), dtype_of(dtype), T), randn((T, k), torch.float32, 2)
    r = kb.route(logits, k, renormalize=renormalize)
    gone = torch.rand((T, k), generator=torch.Generator().manual_seed(3)) < 0.4
    gone[0], gone[1] = True, False
    far = torch.where(torch.arange(k) % 2 == 0, -1, E).expand(T, k)
    experts = torch.where(gone, far, r.experts.cpu()).int().cuda()
    got = kb.route_backward(logits, r._replace(experts=experts), dw, renormalize=renormalize)
    x, w, d = logits.double().cpu().numpy(), r.weights.double().cpu().numpy(), dw.double().cpu().numpy()
    live = ~gone.numpy()
    chosen = r.experts.cpu().numpy().astype(np.int64)
    g, p = np.zeros_like(x), np.zeros_like(x)
    np.put_along_axis(g, chosen, np.where(live, d, 0.0), 1)
    if renormalize:
        np.put_along_axis(p, chosen, np.where(live, w, 0.0), 1)
    else:
        p = np.exp(x - x.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
    dot = (w * d * live).sum(1, keepdims=True)
    want = p * (g - dot)
    size = p * (np.abs(g) + (w * np.abs(d) * live).sum(1, keepdims=True))
    # As for the gradient of whole rows: the exponent's rounding, sums over E and k terms.
    spread = (x.max(1) - x.min(1))[:, None]
    bound = 2.0 ** -22 * (2 * spread + E + 40) * size + UNIT[dtype] * np.abs(want) + 2.0 ** -25
    assert_within(got.cpu(), torch.from_numpy(want), torch.from_numpy(bound), "dlogits")
