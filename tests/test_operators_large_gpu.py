"""The expert and 8-bit integer operators on tensors of more than 2^31 elements:
what lies beyond the first 2^31 is read and written in the right place."""
import pytest

from operator_util import assert_within, offsets_of, product_bound, randn

pytestmark = pytest.mark.gpu
H = 8192


def test_exchange(cuda):
    import torch
    import kebab_b200 as kb
    T, k = 36000, 8
    slots = torch.randperm(T * k, device="cuda", dtype=torch.int32).view(T, k)
    x, w = randn((T, H), torch.float16, 1), torch.rand((T, k), device="cuda")
    xs = kb.dispatch(x, slots)
    assert xs.numel() > 2 ** 31
    some = torch.arange(0, T, 997, device="cuda")
    assert torch.equal(xs[slots[some].long()], x[some][:, None].expand(-1, k, -1))
    y = kb.combine(xs, slots, w)
    want = x[some].double() * w[some].double().sum(1, keepdim=True)
    assert_within(y[some], want, product_bound(want, want.abs(), k + 1, torch.float16), "combine")
    dys, dw = kb.combine_backward(y, xs, slots, w)
    got, want = dys[slots[some].long()], y[some].double()[:, None] * w[some].double()[:, :, None]
    assert_within(got, want, want.abs() * 2.0 ** -10 + 2.0 ** -24, "dys")
    want = (y[some].double() * x[some].double()).sum(1, keepdim=True).expand(-1, k)
    assert_within(dw[some], want, H * 2.0 ** -23 * want.abs(), "dweights")


@pytest.mark.parametrize("opmode", ["RC", "RR"])
def test_grouped_weights(cuda, opmode):
    import torch
    import kebab_b200 as kb
    E, dt = 34, torch.bfloat16
    W = torch.zeros((E, H, H), dtype=dt, device="cuda")
    assert W.numel() > 2 ** 31
    W[E - 1] = randn((H, H), dt, 1) * H ** -0.5
    other = "RR" if opmode == "RC" else "RC"
    for R in (5, 300):  # split over k; persistent
        X = randn((R, H), dt, R)
        offsets = offsets_of([0] * (E - 1) + [R])
        for mode in (opmode, other):
            w = W[E - 1].double().T if mode == "RC" else W[E - 1].double()
            want, size = X.double() @ w, X.double().abs() @ w.abs()
            assert_within(kb.gemm_grouped(X, W, offsets, opmode=mode), want, product_bound(want, size, H, dt), mode)
        dW = kb.gemm_grouped_dw(X, X, offsets, opmode=opmode, dW=W.clone())
        want, size = X.double().T @ X.double(), X.double().abs().T @ X.double().abs()
        assert_within(dW[E - 1], want, product_bound(want, size, R, dt), "dW")
        assert (dW[:E - 1].view(torch.int16).amax() == 0) and (dW[:E - 1].view(torch.int16).amin() == 0)
        del dW


def test_grouped_rows(cuda):
    import torch
    import kebab_b200 as kb
    R, N, dt = 270000, 256, torch.float16
    X = torch.zeros((R, H), dtype=dt, device="cuda")
    assert X.numel() > 2 ** 31
    tail = R - 1000
    X[tail:] = randn((1000, H), dt, 1)
    W = randn((2, N, H), dt, 2) * H ** -0.5
    offsets = offsets_of([tail, 1000])
    Y = kb.gemm_grouped(X, W, offsets)
    want, size = X[tail:].double() @ W[1].double().T, X[tail:].double().abs() @ W[1].double().abs().T
    assert (Y[:tail] == 0).all()
    assert_within(Y[tail:], want, product_bound(want, size, H, dt), "Y")
    dW = kb.gemm_grouped_dw(X, Y, offsets)
    want, size = Y[tail:].double().T @ X[tail:].double(), Y[tail:].double().abs().T @ X[tail:].double().abs()
    assert (dW[0] == 0).all()
    assert_within(dW[1], want, product_bound(want, size, 1000, dt), "dW")


def test_i8(cuda):
    import torch
    import kebab_b200 as kb
    N = 270000
    wq = torch.randint(-127, 128, (N, H), dtype=torch.int8, device="cuda")
    assert wq.numel() > 2 ** 31
    ws = torch.rand((N,), device="cuda") * 0.01 + 1e-3
    for M in (3, 200):
        x = randn((M, H), torch.bfloat16, M)
        y = kb.linear_i8(x, wq, ws)
        q, s = kb.quantize_i8(x)
        for part in (slice(0, 100), slice(N - 500, N)):
            want = (q.double() @ wq[part].double().T) * s.double()[:, None] * ws[part].double()
            assert_within(y[:, part], want, want.abs() * (2.0 ** -8 + 2.0 ** -20) + 2.0 ** -120, "Y")


def test_quantize_and_route(cuda):
    import torch
    import kebab_b200 as kb
    M = 270000
    x = torch.zeros((M, H), dtype=torch.float16, device="cuda")
    x[-7:] = randn((7, H), torch.float16, 1)
    q, s = kb.quantize_i8(x)
    want = kb.quantize_i8(x[-7:].clone())
    assert torch.equal(q[-7:], want[0]) and torch.equal(s[-7:], want[1]) and (s[:-7] == 0).all()
    del x, q
    T, E, k = 4200000, 512, 2
    logits = torch.zeros((T, E), dtype=torch.bfloat16, device="cuda")
    assert logits.numel() > 2 ** 31
    logits[-5:, 500:] = 1.0
    r = kb.route(logits, k)
    assert (r.experts[:-5] == torch.tensor([0, 1], device="cuda")).all()
    assert (r.experts[-5:] == torch.tensor([500, 501], device="cuda")).all()
    assert r.offsets[1] == T - 5 and r.offsets[2] == 2 * (T - 5) and r.offsets[500] == 2 * (T - 5) and r.offsets[E] == 2 * T
    assert torch.equal(r.slots[:-5, 0], torch.arange(T - 5, dtype=torch.int32, device="cuda"))
    assert r.slots[-5:, 1].tolist() == [2 * (T - 5) + 5 + i for i in range(5)]
    d = kb.route_backward(logits, r, torch.ones((T, k), device="cuda"), renormalize=False)
    p = torch.softmax(logits[-5:].double(), 1)
    g = torch.zeros_like(p)
    g[:, 500:502] = 1
    w = r.weights[-5:].double()
    assert_within(r.weights[-5:], torch.full_like(w, 0.5), torch.full_like(w, 2.0 ** -20), "weights")
    want = torch.where(g > 0, w.mean() * (1 - w.sum(1, keepdim=True)), -p * w.sum(1, keepdim=True))
    assert_within(d[-5:], want, want.abs() * 2.0 ** -7 + 2.0 ** -18, "dlogits")
