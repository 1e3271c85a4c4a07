"""Routing, dispatch, combine and the grouped products against plain 64-bit
implementations, at the sizes and inputs where they can go wrong."""
import numpy as np
import pytest

from operator_util import (UNIT, assert_within, counts_of, dtype_of, offsets_of, pitched, product_bound, randn)

pytestmark = pytest.mark.gpu


# ----------------------------------------------------------------------------- routing
def route_plain(logits, k, renormalize):
    """Float64 routing of a float64 array: weights, experts, offsets, slots."""
    T, E = logits.shape
    # NaN above +inf, equal logits by expert.
    order = np.lexsort((np.broadcast_to(np.arange(E), logits.shape), -np.nan_to_num(logits, nan=np.inf),
                        ~np.isnan(logits)), axis=1)[:, :k]
    with np.errstate(invalid="ignore"):
        top = np.take_along_axis(logits, order, 1)
        p = np.exp(top - top[:, :1])
        total = p.sum(1) if renormalize else np.exp(logits - top[:, :1]).sum(1)
        w = p / total[:, None]
    w[top[:, 0] == -np.inf] = 0
    flat = order.reshape(-1)
    place = np.empty(T * k, np.int64)
    place[np.argsort(flat, kind="stable")] = np.arange(T * k)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat, minlength=E))]) if T else np.zeros(E + 1, np.int64)
    return w, order, offsets, place.reshape(T, k)


def weights_bound(logits, w, E):
    # The exponent's rounding (2^-24 of its size), expf (2 ulp), the sum of at
    # most E terms and the quotient.
    spread = np.nanmax(np.where(np.isfinite(logits), logits, np.nan), axis=1) - np.nanmin(
        np.where(np.isfinite(logits), logits, np.nan), axis=1) if logits.size else np.zeros(len(logits))
    spread = np.nan_to_num(spread, nan=0.0)[:, None]
    return np.abs(np.nan_to_num(w)) * 2.0 ** -23 * (2 * spread + E + 8) + 2.0 ** -126


def check_route(logits, k, renormalize):
    import torch
    import kebab_b200 as kb
    T, E = logits.shape
    r = kb.route(logits, k, renormalize=renormalize)
    x = logits.double().cpu().numpy()
    w, experts, offsets, slots = route_plain(x, k, renormalize)
    np.testing.assert_array_equal(r.experts.cpu().numpy(), experts)
    np.testing.assert_array_equal(r.offsets.cpu().numpy(), offsets)
    np.testing.assert_array_equal(r.slots.cpu().numpy(), slots)
    assert_within(r.weights.cpu(), torch.from_numpy(w), torch.from_numpy(weights_bound(x, w, E)), "weights")
    return r


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("T,E,k,dtype", [
    (0, 8, 2, "float32"), (1, 1, 1, "float32"), (1, 128, 8, "float32"), (5, 3, 3, "float16"), (127, 32, 32, "bfloat16"),
    (128, 33, 2, "float32"), (129, 64, 6, "bfloat16"), (130, 257, 5, "float16"), (1000, 96, 1, "float32"),
    (4097, 1024, 10, "bfloat16"), (20011, 60, 4, "bfloat16"), (45000, 16, 8, "float32")])
def test_route(cuda, T, E, k, dtype, renormalize):
    check_route(randn((T, E), dtype_of(dtype), T + E), k, renormalize)


@pytest.mark.parametrize("T", [9, 300])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_ties_and_masks(cuda, T, renormalize):
    import torch
    inf = float("inf")
    x = torch.zeros((T, 40), device="cuda")  # all equal: experts 0..k-1
    x[1] = -inf                              # nothing to route to
    x[2, :38] = -inf                         # fewer finite logits than choices
    x[3, 7] = inf
    x[4, 5] = float("nan")
    x[5] = torch.finfo(torch.float32).min    # the type's lowest value as a mask
    x[5, 11] = 3.0
    x[6, ::2] = -0.0                         # equal to +0
    x[7] = torch.linspace(-3e38, 3e38, 40, device="cuda")
    r = check_route(x, 4, renormalize)
    assert (r.weights[1] == 0).all() and r.experts[1].tolist() == [0, 1, 2, 3]
    assert r.experts[2].tolist() == [38, 39, 0, 1] and (r.weights[2, 2:] == 0).all()
    assert torch.isnan(r.weights[3]).all() and torch.isnan(r.weights[4]).all()
    check_route(torch.zeros((T, 40), device="cuda", dtype=torch.float16), 3, renormalize)


def test_route_pitched_rows_and_stream(cuda):
    import torch
    import kebab_b200 as kb
    x = randn((333, 48), torch.bfloat16, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    a = kb.route(pitched(x, 13, 3), 6)
    b = kb.route(x, 6, stream=side)
    side.synchronize()
    for u, v in zip(a, b):
        assert torch.equal(u, v)


def route_grad_plain(x, experts, dw, renormalize):
    """Float64: the gradient of sum(weights * dw) by the logits."""
    T, E = x.shape
    d, m = np.zeros_like(x), np.zeros_like(x)
    np.put_along_axis(d, experts, dw, 1)
    np.put_along_axis(m, experts, 1.0, 1)
    e = np.exp(x - x.max(1, keepdims=True)) * (m if renormalize else 1.0)
    p = e / e.sum(1, keepdims=True)
    return p * (d - (p * d).sum(1, keepdims=True)), p, d


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("T,E,k,dtype", [(1, 1, 1, "float32"), (3, 8, 8, "float32"), (77, 64, 6, "bfloat16"),
                                         (501, 130, 7, "float16"), (65, 1024, 32, "float32")])
def test_route_backward(cuda, T, E, k, dtype, renormalize):
    import torch
    import kebab_b200 as kb
    logits = randn((T, E), dtype_of(dtype), 3 * T + E)
    dw = randn((T, k), torch.float32, 7)
    r = kb.route(logits, k, renormalize=renormalize)
    got = kb.route_backward(logits, r, dw, renormalize=renormalize)
    assert got.dtype == logits.dtype
    x = logits.double().cpu().numpy()
    want, p, d = route_grad_plain(x, r.experts.cpu().numpy().astype(np.int64), dw.double().cpu().numpy(), renormalize)
    spread = (x.max(1) - x.min(1))[:, None]
    size = p * (np.abs(d) + (p * np.abs(d)).sum(1, keepdims=True))
    bound = 2.0 ** -22 * (2 * spread + E + 40) * size + UNIT[dtype] * np.abs(want) + 2.0 ** -25
    assert_within(got.cpu(), torch.from_numpy(want), torch.from_numpy(bound), "dlogits")


@pytest.mark.parametrize("renormalize", [True, False])
def test_route_backward_against_differences(cuda, renormalize):
    """<dlogits, D> against the central difference of sum(weights * dw) along D:
    h^2 / 6 times the third derivative (under 6 sum |dw| max |D|^3 for a
    softmax) plus the forward's rounding over h."""
    import torch
    import kebab_b200 as kb
    T, E, k, h = 19, 24, 5, 2.0 ** -7
    x, D = 3 * randn((T, E), torch.float32, 1), randn((T, E), torch.float32, 2)
    dw = randn((T, k), torch.float32, 3)
    r = kb.route(x, k, renormalize=renormalize)
    # Along D the choice has to stay the same: raise the chosen well above the rest.
    x = x + 8 * torch.zeros_like(x).scatter_(1, r.experts.long(), 1.0)
    r = kb.route(x, k, renormalize=renormalize)
    f = []
    for sign in (1, -1):
        s = kb.route(x + sign * h * D, k, renormalize=renormalize)
        w = torch.zeros_like(x).scatter_(1, s.experts.long(), s.weights)  # by expert: the order within a row may change
        assert torch.equal(s.experts.sort(1).values, r.experts.sort(1).values)
        f.append((w.gather(1, r.experts.long()) * dw).double().sum(1))
    slope = (f[0] - f[1]) / (2 * h)
    got = (kb.route_backward(x, r, dw, renormalize=renormalize).double() * D.double()).sum(1)
    size = dw.abs().double().sum(1)
    bound = size * (h * h * D.abs().amax(1).double() ** 3 + 2.0 ** -24 * 80 / h)
    assert_within(got, slope, bound, "slope")


def test_route_backward_masked_rows(cuda):
    import torch
    import kebab_b200 as kb
    x = torch.zeros((3, 10), device="cuda")
    x[0] = -float("inf")
    x[1, 2:] = -float("inf")
    dw = torch.ones((3, 4), device="cuda")
    for renormalize in (True, False):
        r = kb.route(x, 4, renormalize=renormalize)
        d = kb.route_backward(x, r, dw, renormalize=renormalize)
        assert torch.isfinite(d).all()
        assert (d[0] == 0).all() and (d[1, 2:] == 0).all()


# ----------------------------------------------------------------------------- dispatch and combine
def slots_of(T, k, seed, drop=0.0):
    """A permutation of T * k places; some choices dropped (-1 or far out)."""
    import torch
    rng = np.random.default_rng(seed)
    s = rng.permutation(T * k).astype(np.int32)
    gone = rng.random(T * k) < drop
    s[gone] = np.where(rng.random(gone.sum()) < 0.5, -1, T * k + 5)
    return torch.from_numpy(s.reshape(T, k)).cuda()


@pytest.mark.parametrize("drop", [0.0, 0.3])
@pytest.mark.parametrize("T,k,H,dtype", [(0, 2, 64, "float16"), (1, 1, 8, "bfloat16"), (1, 8, 4096, "float16"),
                                         (33, 3, 7, "bfloat16"), (130, 5, 2056, "bfloat16"), (257, 9, 520, "float16"),
                                         (64, 32, 96, "float16")])
def test_exchange(cuda, T, k, H, dtype, drop):
    import torch
    import kebab_b200 as kb
    dt = dtype_of(dtype)
    R = T * k
    slots = slots_of(T, k, T + k, drop)
    live = (slots >= 0) & (slots < R)
    at = slots.long().clamp(0, max(R - 1, 0))
    x, ys, dy = randn((T, H), dt, 1), randn((R, H), dt, 2), randn((T, H), dt, 3)
    w = torch.rand((T, k), device="cuda")
    xs = kb.dispatch(x, slots)
    assert xs.shape == (R, H)
    if T == 0:
        assert kb.combine(ys, slots, w).shape == (0, H)
        dys, dw = kb.combine_backward(dy, ys, slots, w)
        assert dys.shape == (0, H) and dw.shape == (0, k)
        return
    assert torch.equal(xs[slots[live].long()], x[:, None].expand(T, k, H)[live])
    rows = ys.double()[at] * live[:, :, None]
    for weights in (w, None):
        v = w.double() if weights is not None else torch.ones_like(w).double()
        y = kb.combine(ys, slots, weights)
        want, size = (rows * v[:, :, None]).sum(1), (rows.abs() * v[:, :, None]).sum(1)
        assert_within(y, want, product_bound(want, size, k + 1, dt), "combine")
    dys, dw = kb.combine_backward(dy, ys, slots, w)
    want = (dy.double()[:, None] * w.double()[:, :, None])[live]
    assert_within(dys[slots[live].long()], want, UNIT[dtype] * want.abs() * (1 + 2.0 ** -20) + 2.0 ** -25, "dys")
    want, size = (dy.double()[:, None] * rows).sum(2), (dy.double()[:, None] * rows).abs().sum(2)
    assert_within(dw, want, H * 2.0 ** -23 * size, "dweights")


def test_exchange_pitched_and_unaligned(cuda):
    import torch
    import kebab_b200 as kb
    T, k, H = 41, 3, 128
    slots = slots_of(T, k, 1)
    x, ys, dy = (randn((n, H), torch.float16, i) for i, n in enumerate((T, T * k, T)))
    w = torch.rand((T, k), device="cuda")
    for extra, shift in ((8, 8), (3, 1)):
        p = lambda t: pitched(t, extra, shift)  # noqa: E731
        assert torch.equal(kb.dispatch(p(x), slots), kb.dispatch(x, slots))
        assert torch.equal(kb.combine(p(ys), slots, w), kb.combine(ys, slots, w))
        a, b = kb.combine_backward(p(dy), p(ys), slots, w), kb.combine_backward(dy, ys, slots, w)
        assert torch.equal(a[0], b[0])
        size = (dy.double()[:, None] * ys.double()[slots.long()]).abs().sum(2)
        assert_within(a[1], b[1], 2 * H * 2.0 ** -23 * size, "dweights")  # another order of the same sum


# ----------------------------------------------------------------------------- grouped products
def grouped_plain(X, W, counts, opmode):
    """Float64 product and the sum of its terms' magnitudes."""
    import torch
    N = W.shape[1] if opmode == "RC" else W.shape[2]
    y = torch.zeros((X.shape[0], N), dtype=torch.float64, device=X.device)
    size, at = torch.zeros_like(y), 0
    for e, c in enumerate(counts):
        x, w = X[at:at + c].double(), W[e].double()
        w = w.T if opmode == "RC" else w
        y[at:at + c], size[at:at + c] = x @ w, x.abs() @ w.abs()
        at += c
    return y, size


def dw_plain(X, dY, counts, opmode):
    import torch
    out, size, at = [], [], 0
    for c in counts:
        x, d = X[at:at + c].double(), dY[at:at + c].double()
        a, b = (d, x) if opmode == "RC" else (x, d)
        out.append(a.T @ b)
        size.append(a.abs().T @ b.abs())
        at += c
    return torch.stack(out), torch.stack(size)


def weights_of(E, N, K, dt, opmode, seed):
    return randn((E, N, K) if opmode == "RC" else (E, K, N), dt, seed) * K ** -0.5


def check_grouped(R, E, N, K, dtype, opmode, kind, seed=0, change=lambda t: t):
    import torch
    import kebab_b200 as kb
    dt = dtype_of(dtype)
    counts = counts_of(kind, R, E, seed)
    offsets = offsets_of(counts)
    X, W = randn((R, K), dt, seed + 1), weights_of(E, N, K, dt, opmode, seed + 2)
    dY = randn((R, N), dt, seed + 3)
    Y = torch.full((R, N), float("nan"), dtype=dt, device="cuda")
    assert kb.gemm_grouped(change(X), change(W), offsets, Y=Y, opmode=opmode) is Y
    want, size = grouped_plain(X, W, counts, opmode)
    assert_within(Y, want, product_bound(want, size, K, dt), "Y")
    other = "RR" if opmode == "RC" else "RC"
    dX = kb.gemm_grouped(change(dY), change(W), offsets, opmode=other)
    want, size = grouped_plain(dY, W, counts, other)
    assert_within(dX, want, product_bound(want, size, N, dt), "dX")
    dW = torch.full(W.shape, float("nan"), dtype=dt, device="cuda")
    kb.gemm_grouped_dw(change(X), change(dY), offsets, dW=dW, opmode=opmode)
    want, size = dw_plain(X, dY, counts, opmode)
    assert_within(dW, want, product_bound(want, size, max(counts), dt), "dW")
    rc, code = kb.device_status()
    assert rc == kb.OK, hex(code)


@pytest.mark.parametrize("opmode", ["RC", "RR"])
@pytest.mark.parametrize("R,E,N,K,dtype,kind", [
    (1, 1, 8, 8, "float16", "even"), (8, 64, 256, 512, "bfloat16", "ragged"), (3, 4, 264, 520, "float16", "ragged"),
    (37, 3, 136, 72, "bfloat16", "ends"), (64, 1, 512, 128, "float16", "even"), (255, 2, 512, 1024, "bfloat16", "one"),
    (257, 2, 520, 264, "float16", "one"), (600, 7, 1032, 200, "bfloat16", "ragged"),
    (1500, 5, 640, 640, "float16", "ragged"), (2049, 33, 264, 392, "bfloat16", "ragged"),
    (4096, 4, 1024, 512, "float16", "even"), (3001, 200, 128, 64, "bfloat16", "ragged")])
def test_grouped(cuda, R, E, N, K, dtype, kind, opmode):
    check_grouped(R, E, N, K, dtype, opmode, kind, seed=R)


@pytest.mark.parametrize("opmode", ["RC", "RR"])
@pytest.mark.parametrize("R,E,N,K", [(1, 2, 1, 1), (5, 2, 33, 17), (100, 3, 65, 129), (70, 4, 7, 300)])
def test_grouped_odd_sizes(cuda, R, E, N, K, opmode):
    check_grouped(R, E, N, K, "float16", opmode, "ragged", seed=N)


@pytest.mark.parametrize("extra,shift", [(8, 8), (16, 0), (5, 0), (0, 1), (3, 7)])
def test_grouped_pitched_and_unaligned(cuda, extra, shift):
    check_grouped(150, 3, 264, 136, "bfloat16", "RC", "ragged", change=lambda t: pitched(t, extra, shift))
    check_grouped(150, 3, 264, 136, "float16", "RR", "ragged", change=lambda t: pitched(t, extra, shift))


def test_grouped_pitched_output(cuda):
    import torch
    import kebab_b200 as kb
    counts = [100, 0, 61]
    X, W = randn((161, 128), torch.float16, 1), weights_of(3, 264, 128, torch.float16, "RC", 2)
    want = kb.gemm_grouped(X, W, offsets_of(counts))
    for extra, shift in ((8, 8), (1, 0), (0, 3)):
        buf = pitched(torch.zeros((161, 264), dtype=torch.float16, device="cuda"), extra, shift)
        assert torch.equal(kb.gemm_grouped(X, W, offsets_of(counts), Y=buf), want)


@pytest.mark.parametrize("rows", [3, 400])
def test_grouped_rows_of_no_group(cuda, rows):
    """Rows before the first and after the last offset are neither read nor written."""
    import torch
    import kebab_b200 as kb
    counts, first = [rows, 0, rows + 5], 11
    R = sum(counts) + first + 20
    X, W = randn((R, 256), torch.bfloat16, 1), weights_of(3, 512, 256, torch.bfloat16, "RC", 2)
    dY = randn((R, 512), torch.bfloat16, 3)
    inner = slice(first, first + sum(counts))
    for t in (X, dY):
        t[:first] = float("nan")
        t[first + sum(counts):] = float("inf")
    offsets = offsets_of(counts, first=first)
    Y = torch.full((R, 512), 7.0, dtype=torch.bfloat16, device="cuda")
    kb.gemm_grouped(X, W, offsets, Y=Y)
    want, size = grouped_plain(X[inner], W, counts, "RC")
    assert_within(Y[inner], want, product_bound(want, size, 256, torch.bfloat16), "Y")
    assert (Y[:first] == 7).all() and (Y[first + sum(counts):] == 7).all()
    dW = kb.gemm_grouped_dw(X, dY, offsets)
    want, size = dw_plain(X[inner], dY[inner], counts, "RC")
    assert_within(dW, want, product_bound(want, size, max(counts), torch.bfloat16), "dW")
    assert (dW[1] == 0).all()


@pytest.mark.parametrize("opmode", ["RC", "RR"])
@pytest.mark.parametrize("N,K,extra", [(1032, 1048, 0), (1031, 1047, 9)])
@pytest.mark.parametrize("counts", [
    [0, 1, 15, 16, 17, 63, 0, 64, 65, 79, 127, 128, 129, 130, 0, 0, 200, 255, 320, 3],
    [0] * 9 + [1000, 1023, 1, 0, 2] + [0] * 3])
def test_grouped_gradient_ends(cuda, counts, N, K, extra, opmode):
    """dW of groups that end anywhere in a 64-row block and of groups without
    rows, enough tiles for the widest panels, outputs on even and odd pitches,
    and neighbours whose rows are not finite."""
    import torch
    import kebab_b200 as kb
    dt = torch.bfloat16
    R = sum(counts)
    X, dY = randn((R, K), dt, 1), randn((R, N), dt, 2)
    shape = (len(counts), N, K) if opmode == "RC" else (len(counts), K, N)

    def run(x, dy):
        dW = torch.full(shape, float("nan"), dtype=dt, device="cuda")
        return kb.gemm_grouped_dw(pitched(x, extra, 0), pitched(dy, extra, 0), offsets_of(counts), dW=dW, opmode=opmode)
    got = run(X, dY)
    want, size = dw_plain(X, dY, counts, opmode)
    assert_within(got, want, product_bound(want, size, max(counts), dt), "dW")
    odd = [e for e in range(len(counts)) if counts[e] and e % 2]
    at = 0
    for e, c in enumerate(counts):
        if e in odd:
            X[at:at + c], dY[at:at + c] = float("inf"), float("nan")
        at += c
    again = run(X, dY)
    for e in range(len(counts)):
        assert torch.isnan(again[e]).all() if e in odd else torch.equal(again[e], got[e])
    rc, code = kb.device_status()
    assert rc == kb.OK, hex(code)


def test_grouped_infinities_stay_in_their_group(cuda):
    """A group's NaN and infinite rows do not reach its neighbours, in the
    products or in dW, although tiles read past a group's end."""
    import torch
    import kebab_b200 as kb
    counts = [37, 83, 5, 130]
    R = sum(counts)
    X, W = randn((R, 136), torch.float16, 1), weights_of(4, 264, 136, torch.float16, "RC", 2)
    dY = randn((R, 264), torch.float16, 3)
    clean = kb.gemm_grouped(X, W, offsets_of(counts)), kb.gemm_grouped_dw(X, dY, offsets_of(counts))
    X[37:120], dY[37:120] = float("nan"), float("inf")
    W[1] = float("inf")
    Y, dW = kb.gemm_grouped(X, W, offsets_of(counts)), kb.gemm_grouped_dw(X, dY, offsets_of(counts))
    for e, (a, b) in enumerate(((0, 37), (37, 120), (120, 125), (125, R))):
        if e != 1:
            assert torch.equal(Y[a:b], clean[0][a:b]) and torch.equal(dW[e], clean[1][e])
        else:
            assert torch.isnan(Y[a:b]).all() and torch.isnan(dW[e]).all()


def test_grouped_wild_offsets(cuda):
    """Offsets out of range or falling are clamped: nothing outside the tensors
    is touched and every group that is in order is right."""
    import torch
    import kebab_b200 as kb
    X, W = randn((50, 64), torch.float16, 1), weights_of(4, 64, 64, torch.float16, "RC", 2)
    offsets = torch.tensor([-9, 20, 20, 50, 90], dtype=torch.int32, device="cuda")
    Y = kb.gemm_grouped(X, W, offsets)
    want, size = grouped_plain(X, W, [20, 0, 30, 0], "RC")
    assert_within(Y, want, product_bound(want, size, 64, torch.float16), "Y")
    assert (kb.gemm_grouped_dw(X, Y, torch.tensor([30, 10, 60, 5, 2], dtype=torch.int32, device="cuda"))[0] == 0).all()


def test_grouped_no_rows(cuda):
    import torch
    import kebab_b200 as kb
    X, W = randn((0, 64), torch.float16, 1), weights_of(3, 128, 64, torch.float16, "RC", 2)
    offsets = offsets_of([0, 0, 0])
    assert kb.gemm_grouped(X, W, offsets).shape == (0, 128)
    dW = torch.full((3, 128, 64), float("nan"), dtype=torch.float16, device="cuda")
    kb.gemm_grouped_dw(X, randn((0, 128), torch.float16, 2), offsets, dW=dW)
    assert (dW == 0).all()


@pytest.mark.parametrize("R", [6, 700])
def test_grouped_gradients_against_differences(cuda, R):
    """The products are linear in X and in W, so differences are exact up to
    rounding: <dY, Y(X + D) - Y(X)> = <dX, D>, and the same for W."""
    import torch
    import kebab_b200 as kb
    E, N, K, dt = 3, 136, 264, torch.float16
    counts = counts_of("ragged", R, E, 4)
    offsets = offsets_of(counts)
    # Multiples of 1/4 and small: every sum below is exact in FP32, and the
    # rounding to FP16 is the only error.
    q = lambda shape, seed: (randn(shape, torch.float32, seed) * 2).round().clamp(-4, 4).to(dt) / 4  # noqa: E731
    X, DX, W, DW, dY = q((R, K), 1), q((R, K), 2), q((E, N, K), 3), q((E, N, K), 4), q((R, N), 5)
    f = lambda a, b: kb.gemm_grouped(a, b, offsets).double()  # noqa: E731
    y, u = f(X, W), UNIT["float16"]
    d = dY.double()
    for moved, grad, D in ((f(X + DX, W), kb.gemm_grouped(dY, W, offsets, opmode="RR"), DX),
                           (f(X, W + DW), kb.gemm_grouped_dw(X, dY, offsets), DW)):
        slope = (d * (moved - y)).sum()
        bound = u * ((d * moved).abs().sum() + (d * y).abs().sum() + (grad.double() * D.double()).abs().sum()) * 1.01
        assert abs(float((grad.double() * D.double()).sum() - slope)) <= float(bound)


@pytest.mark.parametrize("R", [8, 500])
def test_grouped_streams_and_repeats(cuda, R):
    """Bit for bit the same on repeats, on other streams and in a CUDA graph."""
    import torch
    import kebab_b200 as kb
    counts = counts_of("ragged", R, 6, 2)
    offsets = offsets_of(counts)
    X, W = randn((R, 512), torch.bfloat16, 1), weights_of(6, 512, 512, torch.bfloat16, "RC", 2)
    dY = randn((R, 512), torch.bfloat16, 3)
    want = kb.gemm_grouped(X, W, offsets), kb.gemm_grouped_dw(X, dY, offsets)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for i in range(4):
        s = side if i % 2 else None
        outs.append((kb.gemm_grouped(X, W, offsets, stream=s), kb.gemm_grouped_dw(X, dY, offsets, stream=s)))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = kb.gemm_grouped(X, W, offsets), kb.gemm_grouped_dw(X, dY, offsets)
    for _ in range(2):
        for t in captured:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        outs.append(tuple(t.clone() for t in captured))
    for o in outs:
        assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])
