"""Routing from several host threads."""
import threading

import pytest

from operator_util import randn

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
