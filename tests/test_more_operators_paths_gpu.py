"""Norms, 4-bit products and few-token layers where calls meet: several streams,
back to back on one, waits that run out, launches without overlap, and tensors
beyond 2^31 values."""
import hashlib
import os
import subprocess
import sys

import pytest

from operator_util import assert_within, counts_of, offsets_of, randn
from test_grouped_aborts_gpu import check_aborts
from test_operators_concurrent_gpu import operators, run_together

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def layer_of(T, E, H, D, dtype, seed=1):
    import torch
    return (randn((T, H), dtype, seed), randn((E, H), torch.float32, seed + 1) * H ** -0.5, randn((E, 2 * D, H), dtype, seed + 2) * H ** -0.5,
            randn((E, H, D), dtype, seed + 3) * D ** -0.5)


def more_operators():
    import torch
    import kebab_b200 as kb
    ops = []
    for T, H in ((1, 8192), (300, 4096), (5000, 100), (64, 1001)):
        x, dy, w = randn((T, H), torch.bfloat16, T), randn((T, H), torch.bfloat16, T + 1), randn((H,), torch.float32, 3)
        ops += [lambda x=x, w=w: kb.rms_norm(x, w, residual=x), lambda x=x, w=w: kb.rms_norm_i8(x, w)[:2],
                lambda x=x, dy=dy, w=w: kb.rms_norm_backward(dy, x, w, dresidual=x)]
    for R, E, N, K in ((1, 1, 1024, 4096), (61, 3, 520, 1000), (600, 7, 1032, 520), (3000, 9, 2056, 512)):
        X, W = randn((R, K), torch.float16, R), randn((E, N, K), torch.float16, R + 1)
        offsets, q, one = offsets_of(counts_of("ragged", R, E, R)), kb.quantize_f4(W), kb.quantize_f4(W[0])
        ops += [lambda X=X, q=q, o=offsets: kb.linear_grouped_f4(X, q, o), lambda X=X, q=one: kb.linear_f4(X, q), lambda W=W: kb.quantize_f4(W)]
    for T, E, H, D, k in ((1, 64, 1024, 512, 8), (13, 16, 512, 1024, 2)):
        a = layer_of(T, E, H, D, torch.float16 if T > 8 else torch.bfloat16)
        (qi, si), (qo, so) = kb.quantize_i8(a[2]), kb.quantize_i8(a[3])
        ops += [lambda a=a, k=k: kb.expert_layer(*a, k), lambda a=a, q=(qi, si, qo, so), k=k: kb.expert_layer_i8(a[0], a[1], *q, k)]
    return ops


def test_several_streams(cuda):
    import kebab_b200 as kb
    run_together(more_operators() + operators()[::3], 4, 4.0)
    rc, code = kb.device_status()
    assert rc == kb.OK, hex(code)


def test_back_to_back(cuda):
    """A chain in which every call reads what the one before wrote, against the same with the GPU waited for in between."""
    import torch
    import kebab_b200 as kb
    H = 1024
    q = kb.quantize_f4(randn((H, H), torch.bfloat16, 1) * H ** -0.5)
    stack = kb.quantize_f4(randn((4, H, H), torch.bfloat16, 2) * H ** -0.5)
    w, args = randn((H,), torch.float32, 3), layer_of(1, 8, H, 512, torch.bfloat16)[1:]
    wq, ws = kb.quantize_i8(randn((H, H), torch.bfloat16, 4))

    def chain(T, wait):
        at, out = randn((T, H), torch.bfloat16, T), []
        steps = [lambda x: kb.rms_norm(x, w)[0], lambda x: kb.linear_f4(x, q), lambda x: kb.rms_norm(x, w, residual=x)[1],
                 lambda x: kb.linear_grouped_f4(x, stack, offsets_of(counts_of("even", T, 4))), lambda x: kb.rms_norm_backward(x, x, w)[0],
                 lambda x: kb.dequantize_f4(kb.quantize_f4(x), H, torch.bfloat16)]
        steps += [lambda x: kb.expert_layer(x, *args, 3)] if T <= 16 else []
        steps += [lambda x: (lambda n: kb.gemm_i8(n.codes, n.scale, wq, ws))(kb.rms_norm_i8(x, w))]
        for _ in range(3):
            for f in steps:
                at = f(at)
                if wait:
                    torch.cuda.synchronize()
                out.append(at)
        torch.cuda.synchronize()
        return out

    for T in (1, 13, 300, 2000):
        for a, b in zip(chain(T, False), chain(T, True)):
            assert torch.isfinite(a.float()).all() and torch.equal(a, b)


def digest():
    import torch
    h = hashlib.sha256()
    for f in more_operators():
        r = f()
        for t in [r] if isinstance(r, torch.Tensor) else r:
            h.update(t.contiguous().view(torch.uint8).cpu().numpy().tobytes())
    return h.hexdigest()


def test_without_overlapping_launches(cuda):
    env = dict(os.environ, KEBAB_PDL="0", PYTHONPATH=os.pathsep.join([ROOT, os.path.join(ROOT, "tests")]))
    r = subprocess.run([sys.executable, "-c", "import test_more_operators_paths_gpu as t; print(t.digest())"], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    assert r.stdout.split()[-1] == digest()


@pytest.mark.parametrize("R,E,N,K", [(8, 1, 1024, 8192), (100, 3, 520, 4096), (1500, 7, 2056, 520), (4000, 3, 8200, 1024)])
def test_f4_waits_that_run_out(cuda, R, E, N, K):
    import torch
    import kebab_b200 as kb
    X, W, offsets = randn((R, K), torch.bfloat16, 1), randn((E, N, K), torch.bfloat16, 2), offsets_of(counts_of("even", R, E))
    q = kb.quantize_f4(W)
    check_aborts(lambda: kb.linear_grouped_f4(X, q, offsets))


@pytest.mark.parametrize("T,dtype", [(1, "bfloat16"), (13, "float16")])
def test_layer_waits_that_run_out(cuda, T, dtype):
    import torch
    import kebab_b200 as kb
    a = layer_of(T, 16, 2048, 1024, getattr(torch, dtype))
    check_aborts(lambda: kb.expert_layer(*a, 4))
    (qi, si), (qo, so) = kb.quantize_i8(a[2]), kb.quantize_i8(a[3])
    check_aborts(lambda: kb.expert_layer_i8(a[0], a[1], qi, si, qo, so, 4))


def test_norm_beyond_31_bits(cuda):
    import torch
    import kebab_b200 as kb
    T, H = (1 << 31) // 8192 + 3, 8192
    x = torch.zeros((T, H), dtype=torch.bfloat16, device="cuda")
    w, ends = randn((H,), torch.float32, 1), [0, T // 2, T - 2, T - 1]
    x[ends] = randn((4, H), torch.bfloat16, 2)
    small = x[ends].clone()
    y, s = kb.rms_norm(x, w, residual=x)
    a, b = kb.rms_norm(small, w, residual=small)
    assert torch.equal(y[ends], a) and torch.equal(s[ends], b) and not y[1].any() and not y[T - 3].any()
    del s
    n = kb.rms_norm_i8(x, w)
    m = kb.rms_norm_i8(small, w)
    assert torch.equal(n.codes[ends], m.codes) and torch.equal(n.scale[ends], m.scale)
    del n
    dx, dw = kb.rms_norm_backward(y, x, w)
    da, _ = kb.rms_norm_backward(y[ends], small, w)
    assert torch.equal(dx[ends], da)
    d = small.double()
    want = (y[ends].double() * d * (d.square().mean(1, keepdim=True) + 1e-6).rsqrt()).sum(0)
    assert_within(dw, want, (H / 32 + 64) * 2.0 ** -22 * (y[ends].double().abs() * d.abs()).sum(0) * 4 + 1e-6)


def test_f4_beyond_31_bits(cuda):
    import torch
    import kebab_b200 as kb
    # Tokens of more than 2^31 values, and outputs of as many.
    M, K, N = (1 << 31) // 4096 + 5, 4096, 4104
    x = torch.zeros((M, K), dtype=torch.bfloat16, device="cuda")
    ends = [0, 1, M // 2, M - 2, M - 1]
    x[ends] = randn((5, K), torch.bfloat16, 1)
    q = kb.quantize_f4(randn((N, K), torch.bfloat16, 2))
    Y = kb.linear_f4(x, q)
    want = kb.linear_f4(x[ends].repeat(100, 1), q)[:5]  # by the same kernel
    assert torch.equal(Y[ends], want) and not Y[2].any() and not Y[M - 3].any()
    del x, Y
    # Weights of more than 2^32 values: 2^31 bytes of codes.
    E, N, K = 9, 32768, 16384
    one, x = randn((N, K), torch.bfloat16, 3), randn((40, K), torch.bfloat16, 4)
    part = kb.quantize_f4(one)
    codes = torch.zeros((E, *part.codes.shape), dtype=torch.uint8, device="cuda")
    scales = torch.zeros((E, *part.scales.shape), dtype=torch.uint8, device="cuda")
    codes[E - 1], scales[E - 1] = part.codes, part.scales
    for rows in (40, 400):
        X = x.repeat(rows // 40, 1)
        Y = kb.linear_grouped_f4(X, kb.F4(codes, scales), offsets_of([rows // 2] + [0] * (E - 2) + [rows - rows // 2]))
        assert not Y[: rows // 2].any() and torch.equal(Y[rows // 2:], kb.linear_f4(X, part)[rows // 2:])


def test_layer_beyond_31_bits(cuda):
    """The last of experts whose first matrices hold more than 2^31 values."""
    import torch
    import kebab_b200 as kb
    E, H, D = 36, 4096, 8192
    x, router, w_in, w_out = layer_of(2, 1, H, D, torch.bfloat16)
    many = torch.zeros((E, H), device="cuda")
    many[E - 1] = x.float().sum(0)  # both tokens choose it
    big_in = torch.zeros((E, 2 * D, H), dtype=torch.bfloat16, device="cuda")
    big_out = torch.zeros((E, H, D), dtype=torch.bfloat16, device="cuda")
    big_in[E - 1], big_out[E - 1] = w_in[0], w_out[0]
    got = kb.expert_layer(x, many, big_in, big_out, 1)
    assert torch.equal(got, kb.expert_layer(x, router, w_in, w_out, 1))
