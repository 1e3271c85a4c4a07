"""Operators of several host threads and streams at once: their kernels share
the SMs in every mix, and each result is the one that it is alone."""
import random
import threading
import time

import pytest

from operator_util import counts_of, offsets_of, randn

pytestmark = pytest.mark.gpu


def operators():
    import torch
    import kebab_b200 as kb
    dt, ops = torch.bfloat16, []
    for i, (R, E, N, K) in enumerate([(8, 64, 512, 1024), (100, 3, 1024, 4096), (600, 7, 1032, 520), (3000, 9, 2056, 512),
                                      (20, 1, 4096, 2048)]):
        X, W, dY = randn((R, K), dt, i + 1), randn((E, N, K), dt, i + 2), randn((R, N), dt, i + 3)
        offsets, (wq, ws) = offsets_of(counts_of("ragged", R, E, i + 1)), kb.quantize_i8(W)
        ops += [lambda X=X, W=W, o=offsets: kb.gemm_grouped(X, W, o), lambda X=X, dY=dY, o=offsets: kb.gemm_grouped_dw(X, dY, o),
                lambda X=X, q=wq, s=ws, o=offsets: kb.linear_grouped_i8(X, q, s, o),
                lambda X=X, q=wq[0], s=ws[0]: kb.linear_i8(X, q, s)]
    for T, E, k in ((1, 128, 8), (500, 64, 6), (3000, 1000, 12)):
        logits, x = randn((T, E), dt, T), randn((T, 512), dt, T)
        r = kb.route(logits, k)
        ops += [lambda x=logits, k=k: kb.route(x, k), lambda x=x, r=r: kb.combine(kb.dispatch(x, r.slots), r.slots, r.weights)]
    for M, N, K in ((64, 1024, 1024), (512, 512, 512), (2048, 2048, 1024)):
        A, B = randn((M, K), dt, 1), randn((N, K), dt, 2)
        ops.append(lambda A=A, B=B: kb.gemm(A, B))
    return ops


def run_together(ops, threads, seconds):
    import torch
    flat = lambda r: [r] if isinstance(r, torch.Tensor) else list(r)  # noqa: E731
    want = [[t.clone() for t in flat(f())] for f in ops]
    torch.cuda.synchronize()
    errors = []

    def work(seed):
        try:
            rng, stream, t0 = random.Random(seed), torch.cuda.Stream(), time.time()
            with torch.cuda.stream(stream):
                while time.time() - t0 < seconds and not errors:
                    batch = [rng.randrange(len(ops)) for _ in range(20)]
                    outs = [flat(ops[i]()) for i in batch]
                    errors.extend(i for i, o in zip(batch, outs) for a, b in zip(o, want[i]) if not torch.equal(a, b))
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    all_of_them = [threading.Thread(target=work, args=(s,)) for s in range(threads)]
    for t in all_of_them:
        t.start()
    for t in all_of_them:
        t.join()
    assert not errors, errors[:3]


def test_several_streams(cuda):
    import kebab_b200 as kb
    run_together(operators(), 4, 3.0)
    rc, code = kb.device_status()
    assert rc == kb.OK, hex(code)


def test_pair_kernels_on_several_streams(cuda):
    """The GEMM rungs of CTA pairs and the 2:4 product beside the grouped ones
    (not stream-K, whose CTAs wait for one another)."""
    import torch
    import kebab_b200 as kb
    ops = []
    for version, (M, N, K) in ((105, (512, 1024, 512)), (105, (2048, 2048, 256)), (107, (512, 1024, 512)), (107, (2048, 4096, 512)),
                               (112, (512, 768, 512)), (112, (2048, 1536, 512)), (104, (1024, 1024, 512))):
        A, B = randn((M, K), torch.bfloat16, 1), randn((N, K), torch.bfloat16, 2)
        ops.append(lambda A=A, B=B, v=version: kb.gemm(A, B, version=v))
    A, B = randn((512, 1024), torch.float16, 3), randn((512, 1024), torch.float16, 4)
    packed, E = kb.sparse24_compress(kb.sparse24_prune(A))
    ops.append(lambda: kb.gemm_sparse24(packed, E, B))
    run_together(ops + operators(), 4, 3.0)
    rc, code = kb.device_status()
    assert rc == kb.OK, hex(code)
