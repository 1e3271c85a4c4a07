"""Cases of the normalisation, 4-bit product and few-token expert-layer operators: their inputs, their plain forms and
their 64-bit values.

Three families of operators, told apart by a case's "op":

  norm    the root-mean-square norm of tokens with the residual's addition before it (with "train": all gradients too;
          "out" i8: the normed tokens in 8-bit integers with a scale each, which an 8-bit projection reads)
  f4      microscaled 4-bit floating point, 32 values to a power-of-two scale: products of tokens that are quantised in
          the call with weights that were quantised beforehand ("experts" 0 is one weight matrix, otherwise one an
          expert), or ("weights") the quantisation of weights and the values that the codes stand for
  layer   a whole mixture-of-experts layer for a few tokens, from the router to the sum over the experts, with experts
          in 16 bits or in 8-bit integers

With `own` false, run() is elementary torch in 32 bits; with `own` true it calls kebab_b200.
"""
import numpy as np
import torch

own = False

F = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # One token's residual stream before a projection: what counts is the latency of the call.
        {"name": "norm token", "op": "norm", "rows": 1, "width": 8192, "dtype": "bf16", "weight": "bf16", "residual": True, "train": False, "out": "same", "n": 0},
        # A prompt of odd length, normed into 8-bit codes for a projection to a few heads.
        {"name": "norm prompt i8", "op": "norm", "rows": 4093, "width": 8192, "dtype": "f16", "weight": "f32", "residual": True, "train": False, "out": "i8", "n": 1024},
        # A training step's norm with every gradient: bound by memory.
        {"name": "norm train", "op": "norm", "rows": 16381, "width": 4096, "dtype": "bf16", "weight": "f32", "residual": True, "train": True, "out": "same", "n": 0},
        # Weights as they are quantised when a model is loaded, and read back.
        {"name": "f4 weights", "op": "weights", "rows": 8192, "k": 8192, "dtype": "bf16"},
        # One token through a quantised projection: the weights are read once.
        {"name": "f4 token", "op": "f4", "rows": 1, "experts": 0, "idle": 0, "n": 8192, "k": 8192, "dtype": "bf16", "skew": 0.0, "bias": False},
        # A serving batch of 61 sequences through the same projection, with a bias.
        {"name": "f4 batch", "op": "f4", "rows": 61, "experts": 0, "idle": 0, "n": 8192, "k": 8192, "dtype": "f16", "skew": 0.0, "bias": True},
        # A prompt of odd length through the up-projection of a large model's feed-forward layer: bound by the matrix units.
        {"name": "f4 prompt", "op": "f4", "rows": 4093, "experts": 0, "idle": 0, "n": 28672, "k": 8192, "dtype": "bf16", "skew": 0.0, "bias": False},
        # A serving batch through quantised experts, two of them idle.
        {"name": "f4 experts", "op": "f4", "rows": 1021, "experts": 32, "idle": 2, "n": 4096, "k": 4096, "dtype": "f16", "skew": 0.6, "bias": False},
        # One sequence that produces one token, many small experts.
        {"name": "layer token", "op": "layer", "tokens": 1, "experts": 128, "k": 8, "width": 2048, "hidden": 1024, "dtype": "bf16", "bits": 16, "renorm": True},
        # A small serving batch: most experts are read for a token or two.
        {"name": "layer batch", "op": "layer", "tokens": 13, "experts": 64, "k": 6, "width": 2048, "hidden": 1272, "dtype": "f16", "bits": 16, "renorm": False},
        # One token through experts in 8-bit integers.
        {"name": "layer token i8", "op": "layer", "tokens": 1, "experts": 64, "k": 8, "width": 4096, "hidden": 2048, "dtype": "bf16", "bits": 8, "renorm": True},
        # Five drafted tokens to be verified, few and large experts.
        {"name": "layer drafted", "op": "layer", "tokens": 5, "experts": 8, "k": 2, "width": 4096, "hidden": 8192, "dtype": "bf16", "bits": 16, "renorm": True},
    ]


def _spread(rng, low, high, step=1):
    """A multiple of `step` between the two, spread evenly over the logarithm."""
    v = int(round(low * (high / low) ** rng.random()))
    return max(low, min(high, v // step * step))


def draw(rng):
    op = rng.choice(("norm", "norm", "f4", "f4", "weights", "layer", "layer"))
    dtype = rng.choice(("f16", "bf16"))
    if op == "norm":
        width = _spread(rng, 64, 16384, rng.choice((1, 8, 8)))
        out = rng.choice(("same", "same", "i8"))
        rows = _spread(rng, 1, max(1, min(65536, 16381 * 4096 // width)))
        train = out == "same" and rng.random() < 0.5
        dtype = rng.choice((dtype, dtype, "f32")) if out == "same" else dtype
        n = 0 if out == "same" else _spread(rng, 128, 1024, 8)
        if out == "i8":
            rows = min(rows, 4093)
        return {"op": op, "rows": rows, "width": width, "dtype": dtype, "weight": rng.choice((dtype, "f32")), "residual": rng.random() < 0.7, "train": train, "out": out, "n": n}
    if op == "weights":
        k = _spread(rng, 64, 16384, rng.choice((1, 32, 32)))
        return {"op": op, "rows": _spread(rng, 16, 8192 * 8192 // k), "k": k, "dtype": rng.choice((dtype, "f32"))}
    if op == "f4":
        n, k = _spread(rng, 512, 8192, 8), _spread(rng, 512, 8192, 8)
        experts = rng.choice((0, 0, _spread(rng, 2, max(2, min(128, (1 << 30) // (n * k))))))
        rows = _spread(rng, 1, max(1, min(16384, 4093 * 28672 * 8192 // (n * k))))
        return {"op": op, "rows": rows, "experts": experts, "idle": rng.randint(0, experts // 2), "n": n + rng.choice((0, 0, 1, 3)), "k": k + rng.choice((0, 0, 5)), "dtype": dtype,
                "skew": round(rng.random(), 2), "bias": not experts and rng.random() < 0.5}
    bits = rng.choice((16, 16, 8))
    tokens, experts = rng.randint(1, 16), _spread(rng, 8, 256)
    k = rng.randint(1, 8)
    # What the experts hold, and what the tokens' choices read of it.
    most = min((1 << 30) // (3 * experts), 360000000 // (tokens * k))
    step = rng.choice((16, 8)) if bits == 16 else 16
    width = _spread(rng, 256, max(256, min(8192, most // 256)), step)
    return {"op": op, "tokens": tokens, "experts": experts, "k": k, "width": width, "hidden": _spread(rng, 128, max(128, min(8192, most // width)), step), "dtype": dtype,
            "bits": bits, "renorm": rng.random() < 0.5}


def _counts(case):
    """Rows of each expert, most popular first: popularity falls as rank to the power -skew, and `idle` experts have none."""
    busy = max(1, case["experts"] - case["idle"])
    p = np.arange(1, busy + 1, dtype=np.float64) ** -case["skew"]
    at = np.floor(np.cumsum(p) / p.sum() * case["rows"] + 1e-9).astype(np.int64)
    at[-1] = case["rows"]
    return np.diff(at, prepend=0).tolist() + [0] * (case["experts"] - busy)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _tokens(g, rows, width, dtype):
    """Activations with a few channels much larger than the others, as models meet them."""
    return (_randn(g, rows, width) * (1 + 9 * (torch.rand(width, generator=g, device="cuda") < 0.01))).to(dtype)


def _int8(w):
    scale = w.abs().amax(-1) / 127
    return torch.round(w / scale[..., None]).to(torch.int8), scale


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    op, dt = case["op"], F[case["dtype"]]
    if op == "norm":
        T, H = case["rows"], case["width"]
        s["x"] = _tokens(g, T, H, dt)
        s["w"] = (1 + 0.1 * _randn(g, H)).to(F[case["weight"]])
        if case["residual"]:
            s["r"] = (4 * _randn(g, T, H)).to(dt)
        if case["train"]:
            s["dy"] = _randn(g, T, H).to(dt)
            if case["residual"]:
                s["ds"] = _randn(g, T, H).to(dt)
        if case["out"] == "i8":
            s["wq"], s["ws"] = _int8(_randn(g, case["n"], H) * H ** -0.5)
        return s
    if op == "weights":
        s["w"] = (_randn(g, case["rows"], case["k"]) * case["k"] ** -0.5).to(dt)
        return s
    if op == "f4":
        R, N, K, E = case["rows"], case["n"], case["k"], case["experts"]
        if E:
            # Which experts are the popular ones is the seed's.
            counts = [_counts(case)[i] for i in torch.randperm(E, generator=torch.Generator().manual_seed(seed)).tolist()]
            s["counts"] = counts
            s["offsets"] = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")
        s["x"] = _tokens(g, R, K, dt)
        W = torch.empty((max(E, 1), N, K), dtype=dt, device="cuda")
        for e in range(max(E, 1)):
            W[e] = _randn(g, N, K) * K ** -0.5
        # Quantised when the model was loaded: two codes a byte, lower channel first, and the scales' exponents.
        packed = [_packed(w) for w in W]
        s["codes"], s["exponents"] = (torch.stack(t) for t in zip(*packed))
        if own:
            import kebab_b200 as kb

            s["q"] = kb.quantize_f4(W if E else W[0])
        if case["bias"]:
            s["b"] = _randn(g, N).to(dt)
        return s
    T, E, H, D = case["tokens"], case["experts"], case["width"], case["hidden"]
    s["x"] = _tokens(g, T, H, dt)
    s["router"] = _randn(g, E, H) * H ** -0.5
    # Gate rows, then up rows, of every expert.
    w_in, w_out = torch.empty((E, 2 * D, H), dtype=dt, device="cuda"), torch.empty((E, H, D), dtype=dt, device="cuda")
    for e in range(E):
        w_in[e], w_out[e] = _randn(g, 2 * D, H) * H ** -0.5, _randn(g, H, D) * D ** -0.5
    if case["bits"] == 8:
        ins, outs = zip(*(_int8(w.float()) for w in w_in)), zip(*(_int8(w.float()) for w in w_out))
        (s["w_in"], s["in_scale"]), (s["w_out"], s["out_scale"]) = (torch.stack(t) for t in ins), (torch.stack(t) for t in outs)
    else:
        s["w_in"], s["w_out"] = w_in, w_out
    return s


def _ours(s):
    import kebab_b200 as kb

    op = s["op"]
    if op == "norm":
        if s["out"] == "i8":
            n = kb.rms_norm_i8(s["x"], s["w"], EPS, residual=s.get("r"))
            out = {"y": kb.gemm_i8(n.codes, n.scale, s["wq"], s["ws"], dtype=s["x"].dtype)}
            if "r" in s:
                out["s"] = n.residual
            return out
        y, res = kb.rms_norm(s["x"], s["w"], EPS, residual=s.get("r"))
        out = {"y": y}
        if "r" in s:
            out["s"] = res
        if s["train"]:
            out["dx"], out["dw"] = kb.rms_norm_backward(s["dy"], res, s["w"], EPS, dresidual=s.get("ds"))
        return out
    if op == "weights":
        return kb.dequantize_f4(kb.quantize_f4(s["w"]), s["k"], s["w"].dtype)
    if op == "f4":
        if s["experts"]:
            return kb.linear_grouped_f4(s["x"], s["q"], s["offsets"])
        return kb.linear_f4(s["x"], s["q"], bias=s.get("b"))
    if s["bits"] == 8:
        return kb.expert_layer_i8(s["x"], s["router"], s["w_in"], s["in_scale"], s["w_out"], s["out_scale"], s["k"], renormalize=s["renorm"])
    return kb.expert_layer(s["x"], s["router"], s["w_in"], s["w_out"], s["k"], renormalize=s["renorm"])


def _int8_tokens(x):
    """The values that 8-bit codes of the rows stand for, without the scale, and the scale."""
    top = x.abs().amax(-1, keepdim=True)
    return torch.where(top > 0, torch.round(x * 127 / top), 0.0), top / 127


def _norm(s):
    x, w, dt = s["x"].float(), s["w"].float(), s["x"].dtype
    if "r" in s:
        stored = (x + s["r"].float()).to(dt)  # the norm is of the sum as it is kept
        x = stored.float()
    rstd = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
    y = x * rstd * w
    if s["out"] == "i8":
        q, scale = _int8_tokens(y)
        y = q @ s["wq"].float().T * s["ws"] * scale
    out = {"y": y.to(dt)}
    if "r" in s:
        out["s"] = stored
    if s["train"]:
        dy = s["dy"].float()
        g = dy * w
        dx = rstd * (g - x * rstd * rstd * (g * x).mean(1, keepdim=True))
        out["dx"] = (dx + s["ds"].float() if "ds" in s else dx).to(dt)
        out["dw"] = (dy * x * rstd).sum(0).to(s["w"].dtype)
    return out


def _blocks(x):
    """Rows in blocks of 32, the last one filled up with zeros."""
    x = torch.nn.functional.pad(x, (0, -x.shape[-1] % 32))
    return x.reshape(*x.shape[:-1], -1, 32)


def _f4_parts(x):
    """Blocks as multiples of their scale on the grid 0, 1/2, 1, 3/2, 2, 3, 4, 6 (nearest, ties to the even code), and the
    scales' exponents: the least that keep every magnitude within 6, from -127."""
    x = _blocks(x)
    m, e = torch.frexp(x.abs().amax(-1, keepdim=True))  # amax = m 2^e, 1/2 <= m < 1
    e = torch.where(m == 0, -127, torch.where(m <= 0.75, e - 3, e - 2)).clamp(min=-127)
    v = torch.ldexp(x, -e)
    a = v.abs()
    a = torch.where(a < 2, torch.round(2 * a) / 2, torch.where(a < 4, torch.round(a), 2 * torch.round(a / 2)))
    return torch.copysign(a, v), e


def _f4_values(x):
    v, e = _f4_parts(x)
    return torch.ldexp(v, e).flatten(-2)[..., : x.shape[-1]]


def _packed(w):
    v, e = _f4_parts(w.float())
    a = v.abs()
    code = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8) + 8 * torch.signbit(v).to(torch.uint8)
    code = code.flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, e[..., 0].to(torch.int8)


def _grid(device, dtype):
    g = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=dtype, device=device)
    return torch.cat([g, -g])


def _unpacked(codes, exponents, k):
    grid = _grid(codes.device, torch.float32)
    v = torch.stack([grid[(codes & 15).int()], grid[(codes >> 4).int()]], -1).flatten(-2)
    v = torch.ldexp(v.reshape(*exponents.shape, 32), exponents[..., None].int())
    return v.flatten(-2)[..., :k]


def _weights(s):
    return _f4_values(s["w"].float()).to(s["w"].dtype)


def _f4(s):
    dt, k = s["x"].dtype, s["k"]
    x = _f4_values(s["x"].float())
    if s["experts"]:
        parts = zip(torch.split(x, s["counts"]), s["codes"], s["exponents"])
        y = torch.cat([a @ _unpacked(c, e, k).T for a, c, e in parts if len(a)])
    else:
        y = x @ _unpacked(s["codes"][0], s["exponents"][0], k).T
    if "b" in s:
        y = y + s["b"].float()
    return y.to(dt)


def _layer(s):
    x, k = s["x"].float(), s["k"]
    logits = x @ s["router"].T
    order = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
    p = torch.exp(logits - logits.amax(1, keepdim=True))
    top = torch.gather(p, 1, order)
    weights = top / (top if s["renorm"] else p).sum(1, keepdim=True)
    e = order.reshape(-1)
    rows = x.repeat_interleave(k, 0)[:, :, None]  # a token once a choice
    if s["bits"] == 8:
        q, scale = _int8_tokens(rows[:, :, 0])
        h = torch.bmm(s["w_in"].index_select(0, e).float(), q[:, :, None])[:, :, 0] * s["in_scale"].index_select(0, e) * scale
    else:
        h = torch.bmm(s["w_in"].index_select(0, e).float(), rows)[:, :, 0]
    gate, up = h.chunk(2, dim=1)
    h = gate / (1 + torch.exp(-gate)) * up
    if s["bits"] == 8:
        q, scale = _int8_tokens(h)
        y = torch.bmm(s["w_out"].index_select(0, e).float(), q[:, :, None])[:, :, 0] * s["out_scale"].index_select(0, e) * scale
    else:
        y = torch.bmm(s["w_out"].index_select(0, e).float(), h[:, :, None])[:, :, 0]
    return (y.view(-1, k, y.shape[1]) * weights[:, :, None]).sum(1).to(s["x"].dtype)


def run(state):
    if own:
        return _ours(state)
    return {"norm": _norm, "weights": _weights, "f4": _f4, "layer": _layer}[state["op"]](state)


def work(case):
    """What a pass cannot do without: each input read once, each output written once, two operations a product term. 4-bit
    weights are half a byte and a 32nd of a byte for the scale; of the experts of a layer, those that count are as many as
    independent choices name on average."""
    op, b = case["op"], F[case["dtype"]].itemsize
    if op == "norm":
        T, H, res = case["rows"], case["width"], case["residual"]
        w = H * F[case["weight"]].itemsize
        row = T * H * b
        size, flops = row * (1 + 2 * res) + w, 5 * T * H
        if case["out"] == "i8":
            return {"bytes": size + case["n"] * (H + 4) + T * case["n"] * b, "flops": flops + 2 * T * case["n"] * H}
        size += row
        if case["train"]:  # dy, the gradient of the sum, and the sum once more
            size += row * (3 + res) + 2 * w
            flops += 10 * T * H
        return {"bytes": size, "flops": flops}
    if op == "weights":
        return {"bytes": case["rows"] * case["k"] * (2 * b + 2 * 17 / 32), "flops": 4 * case["rows"] * case["k"]}
    if op == "f4":
        R, N, K, E = case["rows"], case["n"], case["k"], case["experts"]
        busy = sum(c > 0 for c in _counts(case)) if E else 1
        return {"bytes": b * (R * K + R * N + N * case["bias"]) + busy * N * K * 17 / 32 + 4 * (E + 1), "flops": 2 * R * N * K}
    T, E, H, D, k = case["tokens"], case["experts"], case["width"], case["hidden"], case["k"]
    busy = E * (1 - (1 - k / E) ** T)
    one = 3 * D * H * 2 if case["bits"] == 16 else 3 * D * H + 4 * (2 * D + H)
    return {"bytes": busy * one + 4 * E * H + 2 * b * T * H, "flops": 2 * T * E * H + 6 * T * k * D * H}


def _exact_norm(s):
    x, w = s["x"].double(), s["w"].double()
    if "r" in s:
        x = (x + s["r"].double()).to(s["x"].dtype).double()
    inv = 1 / torch.sqrt(torch.linalg.vecdot(x, x)[:, None] / x.shape[1] + EPS)
    hat = x * inv
    y = hat * w
    if s["out"] == "i8":
        top = y.abs().amax(1)
        q = torch.where(top[:, None] > 0, torch.round(127 * y / top[:, None]), 0.0)
        y = torch.einsum("rk,nk->rn", q, s["wq"].double()) * torch.outer(top / 127, s["ws"].double())
    out = {"y": y}
    if "r" in s:
        out["s"] = x
    if s["train"]:
        dy = s["dy"].double()
        out["dw"] = torch.einsum("tk,tk->k", dy, hat)
        d = dy * w
        out["dx"] = inv * (d - hat * (torch.linalg.vecdot(d, hat) / x.shape[1])[:, None])
        if "ds" in s:
            out["dx"] = out["dx"] + s["ds"].double()
    return out


def _exact_f4(x):
    """The values of the 4-bit codes, by the distances to the grid."""
    x = x.double()
    b = _blocks(x)
    top = b.abs().amax(-1, keepdim=True)
    e = torch.where(top > 0, torch.round(torch.log2(torch.where(top > 0, top, 1.0) / 6)), -127.0)
    e = (e + (top > 6 * torch.exp2(e)).double()).clamp(min=-127)  # the logarithm itself may be off by a little
    v = b.abs() / torch.exp2(e)
    middle = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 1e300], dtype=torch.float64, device=x.device)
    code = torch.bucketize(v, middle)  # how many of them are below v; on one: the lower code, unless that is odd
    code = code + ((v == middle[code]) & (code % 2 == 1))
    return (_grid(x.device, torch.float64)[code] * torch.exp2(e) * torch.sign(b)).flatten(-2)[:, : x.shape[1]]


def _exact_products(s):
    E, at = max(s["experts"], 1), 0
    counts = s.get("counts", [s["rows"]])
    x = _exact_f4(s["x"])
    y = torch.zeros(s["rows"], s["n"], dtype=torch.float64, device="cuda")
    grid = _grid("cuda", torch.float64)
    for e in range(E):
        c, r = s["codes"][e], slice(at, at + counts[e])
        w = torch.empty(s["n"], 2 * c.shape[1], dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = grid[(c % 16).long()], grid[(c // 16).long()]
        w *= torch.exp2(s["exponents"][e].double()).repeat_interleave(32, 1)
        y[r] = torch.einsum("rk,nk->rn", x[r], w[:, : s["k"]])
        at += counts[e]
    return y + s["b"].double() if "b" in s else y


def _exact_layer(s):
    x, k, D = s["x"].double(), s["k"], s["hidden"]
    logits = (x @ s["router"].double().T).cpu().numpy()
    y = torch.zeros_like(x)
    for t in range(s["tokens"]):
        chosen = np.lexsort((np.arange(s["experts"]), -logits[t]))[:k]
        e = np.exp(logits[t] - logits[t].max())
        p = e[chosen] / (e[chosen] if s["renorm"] else e).sum()
        for e, w in zip(chosen.tolist(), p.tolist()):
            a, step = x[t], 1.0
            if s["bits"] == 8:
                step = a.abs().amax() / 127
                a = torch.round(127 * a / a.abs().amax())
            h = torch.mv(s["w_in"][e].double(), a)
            h = h * step * s["in_scale"][e].double() if s["bits"] == 8 else h
            h = h[:D] * torch.sigmoid(h[:D]) * h[D:]
            if s["bits"] == 8:
                step = h.abs().amax() / 127
                h = torch.round(127 * h / h.abs().amax())
            o = torch.mv(s["w_out"][e].double(), h)
            y[t] += w * (o * step * s["out_scale"][e].double() if s["bits"] == 8 else o)
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "weights":
        return _exact_f4(s["w"])
    return {"norm": _exact_norm, "f4": _exact_products, "layer": _exact_layer}[s["op"]](s)
