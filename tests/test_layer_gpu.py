"""A whole mixture-of-experts layer for a few tokens against 64 bits."""
import pytest

from operator_util import TINY, UNIT, assert_within, dtype_of, pitched, randn

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def make(T, E, H, D, dtype, seed=1):
    import torch
    dt = dtype_of(dtype)
    x, router = randn((T, H), dt, seed), randn((E, H), torch.float32, seed + 1) * H ** -0.5
    return x, router, randn((E, 2 * D, H), dt, seed + 2) * H ** -0.5, randn((E, H, D), dt, seed + 3) * D ** -0.5


def codes_of(v):
    """8-bit codes in 64 bits, and the scale."""
    top = v.abs().amax()
    return (v * 127 / top).round() if top >= 1e-30 else v * 0, top / 127 if top >= 1e-30 else top * 0


def reference(x, router, w_in, w_out, k, renorm, scales=None):
    """(y, bound) in 64 bits; the bound adds up what FP32 sums, products and roundings may lose on the way."""
    import torch
    T, H = x.shape
    D = w_out.shape[2]
    xd = x.double()
    logits = xd @ router.double().T
    near = H * 2 * U * (xd.abs() @ router.double().abs().T).amax(1)  # a logit's error
    order = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
    p = torch.exp(logits - logits.amax(1, keepdim=True))
    top = torch.gather(p, 1, order)
    weights = top / (top if renorm else p).sum(1, keepdim=True)
    y, bound = torch.zeros_like(xd), torch.zeros_like(xd)
    for t in range(T):
        w_rel = 4 * near[t] + 16 * U
        for j in range(k):
            e, w = int(order[t, j]), weights[t, j]
            win, wout = w_in[e].double(), w_out[e].double()
            if scales is None:
                h = win @ xd[t]
                dh = 2 * U * H * (win.abs() @ xd[t].abs())
            else:
                q, s = codes_of(xd[t])
                h = (win @ q) * s * scales[0][e].double()
                dh = 8 * U * h.abs()
            g, u, dg, du = h[:D], h[D:], dh[:D], dh[D:]
            sg = torch.sigmoid(g)
            a = g * sg * u
            da = 1.1 * dg * (u.abs() + du) + (g * sg).abs() * du + 16 * U * a.abs()  # |silu'| <= 1.1
            if scales is None:
                o, size = wout @ a, wout.abs() @ a.abs()
                do = wout.abs() @ da + size * (2 * U * D + 2.0 ** -16)  # a in at least 16 bits
            else:
                q, s = codes_of(a)
                o = (wout @ q) * s * scales[1][e].double()
                # A code may be the neighbour where a / s is as near to a tie as its error.
                frac = a / s if s > 0 else a * 0
                slack = (da / s if s > 0 else da * 0) + (da.amax() / (127 * s) + 8 * U if s > 0 else 0) * frac.abs()
                flip = ((frac - frac.floor() - 0.5).abs() <= slack).double()
                do = (wout.abs() @ flip) * s * scales[1][e].double() + o.abs() * (8 * U + (da.amax() / (127 * s) if s > 0 else 0))
            y[t] += w * o
            bound[t] += w * (do + (o.abs() + do) * w_rel)
    name = str(x.dtype).replace("torch.", "")
    bound = bound + 64 * U * y.abs()
    return y, bound + UNIT[name] * (y.abs() + bound) + TINY[name]


SHAPES = [(1, 8, 64, 64, 2), (1, 128, 2048, 256, 8), (1, 1, 8, 8, 1), (16, 16, 256, 128, 4), (13, 64, 1024, 200, 6), (5, 8, 512, 1024, 2), (3, 300, 136, 72, 32),
          (7, 4, 2056, 1000, 4), (9, 5, 4104, 40, 3), (2, 1024, 64, 16, 1), (16, 7, 88, 2504, 1)]


@pytest.mark.parametrize("T,E,H,D,k", SHAPES)
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("renorm", [True, False])
def test_layer(cuda, T, E, H, D, k, dtype, renorm):
    import torch
    import kebab_b200 as kb
    x, router, w_in, w_out = make(T, E, H, D, dtype, T + E)
    y = kb.expert_layer(x, router, w_in, w_out, k, renorm)
    want, bound = reference(x, router, w_in, w_out, k, renorm)
    assert_within(y, want, bound)
    assert torch.equal(kb.expert_layer(x, router, w_in, w_out, k, renorm), y)


@pytest.mark.parametrize("T,E,H,D,k", SHAPES)
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_layer_i8(cuda, T, E, H, D, k, dtype):
    import torch
    import kebab_b200 as kb
    x, router, w_in, w_out = make(T, E, H, D, dtype, T + E)
    (qi, si), (qo, so) = kb.quantize_i8(w_in), kb.quantize_i8(w_out)
    y = kb.expert_layer_i8(x, router, qi, si, qo, so, k)
    want, bound = reference(x, router, qi, qo, k, True, (si, so))
    assert_within(y, want, bound)
    assert torch.equal(kb.expert_layer_i8(x, router, qi, si, qo, so, k), y)


@pytest.mark.parametrize("H,D", [(1, 1), (7, 5), (65, 33), (130, 1000), (1001, 77), (260, 132)])
def test_odd_sizes(cuda, H, D):
    import kebab_b200 as kb
    x, router, w_in, w_out = make(3, 6, H, D, "bfloat16", H)
    want, bound = reference(x, router, w_in, w_out, 2, True)
    assert_within(kb.expert_layer(x, router, w_in, w_out, 2), want, bound)
    (qi, si), (qo, so) = kb.quantize_i8(w_in), kb.quantize_i8(w_out)
    want, bound = reference(x, router, qi, qo, 2, True, (si, so))
    assert_within(kb.expert_layer_i8(x, router, qi, si, qo, so, 2), want, bound)


@pytest.mark.parametrize("extra,shift", [(8, 0), (3, 1)])
def test_tokens_at_a_pitch(cuda, extra, shift):
    import torch
    import kebab_b200 as kb
    x, router, w_in, w_out = make(5, 8, 256, 128, "float16")
    want = kb.expert_layer(x, router, w_in, w_out, 3)
    assert torch.equal(kb.expert_layer(pitched(x, extra, shift), router, w_in, w_out, 3), want)


def test_weights_on_odd_addresses(cuda):
    import torch
    import kebab_b200 as kb
    x, router, w_in, w_out = make(5, 8, 256, 128, "float16")
    want = kb.expert_layer(x, router, w_in, w_out, 3)

    def moved(t):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:]
        return buf.view(t.shape).copy_(t)

    assert torch.equal(kb.expert_layer(x, moved(router), moved(w_in), moved(w_out), 3), want)


def test_what_an_expert_holds_reaches_its_tokens_only(cuda):
    """Infinities and NaN in experts, in tokens and in experts that nobody chose."""
    import torch
    import kebab_b200 as kb
    x, router, w_in, w_out = make(6, 16, 256, 128, "bfloat16", 3)
    r = kb.route(x.float() @ router.T, 2)
    clean = kb.expert_layer(x, router, w_in, w_out, 2)
    bad = int(r.experts[0, 0])
    hit = (r.experts == bad).any(1)
    assert hit.any() and not hit.all()
    unused = [e for e in range(16) if not (r.experts == e).any()]
    w2, o2 = w_in.clone(), w_out.clone()
    w2[bad, 3, 5], o2[bad, 7, 9] = float("inf"), float("nan")
    for e in unused:
        w2[e], o2[e] = float("nan"), float("inf")
    y = kb.expert_layer(x, router, w2, o2, 2)
    assert torch.equal(y[~hit], clean[~hit])
    assert torch.isnan(y[hit][:, 7]).all()
    x2 = x.clone()
    x2[1, 4] = float("nan")
    y = kb.expert_layer(x2, router, w_in, w_out, 2)
    keep = [0, 2, 3, 4, 5]
    assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[1]).all()
    (qi, si), (qo, so) = kb.quantize_i8(w_in), kb.quantize_i8(w_out)
    clean = kb.expert_layer_i8(x, router, qi, si, qo, so, 2)
    y = kb.expert_layer_i8(x2, router, qi, si, qo, so, 2)
    assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[1]).all()
    si2 = si.clone()
    si2[bad, 3] = float("nan")
    y = kb.expert_layer_i8(x, router, qi, si2, qo, so, 2)
    assert torch.equal(y[~hit], clean[~hit]) and torch.isnan(y[hit]).all()


def test_large_hidden_values(cuda):
    """Hidden values beyond FP16's largest number, summed back into range by small weights."""
    import kebab_b200 as kb
    x, router, w_in, w_out = make(4, 4, 256, 128, "float16", 5)
    x, w_in, w_out = x * 16, w_in * 64, w_out * 2.0 ** -10
    want, bound = reference(x, router, w_in, w_out, 2, True)
    assert_within(kb.expert_layer(x, router, w_in, w_out, 2), want, bound)


def test_equal_logits_take_the_lower_expert(cuda):
    import torch
    import kebab_b200 as kb
    x, router, w_in, w_out = make(3, 8, 128, 64, "bfloat16", 5)
    router[1:] = router[0].clone()
    y = kb.expert_layer(x, router, w_in, w_out, 3)
    want, bound = reference(x, router, w_in, w_out, 3, True)
    assert_within(y, want, bound)
    router[:] = 0
    w_in[3:], w_out[3:] = float("nan"), float("nan")
    assert torch.isfinite(kb.expert_layer(x, router, w_in, w_out, 3)).all()


def test_matches_the_separate_operators(cuda):
    """The layer beside route, dispatch, grouped products and combine, whose hidden values are rounded to 16 bits: the
    gate and up values (each by u = 2^-8), the activation's two roundings, the rows before the sum: about six of u, over
    terms whose magnitudes sum to `size`."""
    import torch
    import kebab_b200 as kb
    from kebab_b200.moe import MoE
    torch.manual_seed(0)
    layer = MoE(512, 256, 16, 4)
    x = randn((11, 512), torch.bfloat16, 3)
    with torch.no_grad():
        separate, r = layer(x)
        y = kb.expert_layer(x, layer.router, layer.w_in, layer.w_out, 4)
        h = torch.stack([layer.w_in.float()[r.experts[:, j].long()] @ x.float()[:, :, None] for j in range(4)])[..., 0]
        a = torch.nn.functional.silu(h[..., :256]) * h[..., 256:]
        size = sum(r.weights[:, j, None] * (layer.w_out.float().abs()[r.experts[:, j].long()] @ a[j].abs()[:, :, None])[..., 0] for j in range(4))
    assert_within(y, separate, 2.0 ** -8 * 8 * size.double() + 2.0 ** -7 * y.double().abs())


def test_empty(cuda):
    import torch
    import kebab_b200 as kb
    x, router, w_in, w_out = make(3, 8, 64, 64, "bfloat16")
    assert kb.expert_layer(x[:0], router, w_in, w_out, 2).shape == (0, 64)
    assert torch.equal(kb.expert_layer(x[:1], router, w_in, w_out, 2), kb.expert_layer(x, router, w_in, w_out, 2)[:1])


def test_captured(cuda):
    """Two graphs with calls of their own, replayed in turn and after one another."""
    import torch
    import kebab_b200 as kb
    x, router, w_in, w_out = make(7, 16, 512, 256, "bfloat16")
    (qi, si), (qo, so) = kb.quantize_i8(w_in), kb.quantize_i8(w_out)
    step = lambda: (kb.expert_layer(x, router, w_in, w_out, 4), kb.expert_layer_i8(x, router, qi, si, qo, so, 4),  # noqa: E731
                    kb.expert_layer(x[:1], router, w_in, w_out, 2))
    step()
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(step())
    for seed in (5, 6):
        x.copy_(randn((7, 512), torch.bfloat16, seed))
        want = step()
        for g, out in zip(graphs, outs):
            g.replay()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_many_calls_on_several_streams(cuda):
    """Layers of several streams beside one another and beside products: each result is the one that it is alone."""
    from test_operators_concurrent_gpu import operators, run_together
    import kebab_b200 as kb
    ops = []
    for T, E, H, D, k in ((1, 64, 1024, 512, 8), (13, 16, 512, 1024, 2), (4, 8, 2048, 256, 2)):
        a = make(T, E, H, D, "bfloat16", T)
        ops.append(lambda a=a, k=k: kb.expert_layer(*a, k))
    run_together(ops + operators()[:8], 4, 3.0)
    rc, code = kb.device_status()
    assert rc == kb.OK, hex(code)


def test_refusals(cuda):
    import torch
    import kebab_b200 as kb
    x, router, w_in, w_out = make(3, 8, 64, 32, "bfloat16")
    (qi, si), (qo, so) = kb.quantize_i8(w_in), kb.quantize_i8(w_out)
    many = randn((kb.FEW_TOKENS + 1, 64), torch.bfloat16, 1)
    for call in (lambda: kb.expert_layer(many, router, w_in, w_out, 2), lambda: kb.expert_layer(x, router.half(), w_in, w_out, 2),
                 lambda: kb.expert_layer(x, router[:, :63], w_in, w_out, 2), lambda: kb.expert_layer(x, router, w_in[:, :63], w_out, 2),
                 lambda: kb.expert_layer(x, router, w_in, w_out[:7], 2), lambda: kb.expert_layer(x, router, w_in.half(), w_out, 2),
                 lambda: kb.expert_layer(x, router, w_in, w_out, 0), lambda: kb.expert_layer(x, router, w_in, w_out, 9),
                 lambda: kb.expert_layer(x.float(), router, w_in, w_out, 2), lambda: kb.expert_layer(x, router, w_in.transpose(1, 2), w_out, 2),
                 lambda: kb.expert_layer_i8(x, router, qi, si[:, :63], qo, so, 2), lambda: kb.expert_layer_i8(x, router, qi, None, qo, so, 2),
                 lambda: kb.expert_layer_i8(x, router, w_in, si, w_out, so, 2), lambda: kb.expert_layer(x, router, w_in, None, 2)):
        with pytest.raises(kb.KebabError):
            call()
