"""Cases of the mixture-of-experts and 8-bit integer operators: their inputs, their plain forms and their 64-bit values.

Four families of operators, told apart by a case's "op":

  route     top-k routing of tokens to experts: the weights, the experts, and the plan that sorts the tokens by expert
            (with "train": the gradient of the logits too)
  exchange  rows of tokens laid out by expert, and the experts' rows summed back into tokens with the routing weights
            (with "train": all gradients too)
  grouped   products grouped by expert with ragged sizes, Y[r] = X[r] W_e for the rows r of expert e (with "train": the
            gradients of X and W too)
  i8        products in 8-bit integers with one scale a token and one a channel: the tokens are quantised in the call, the
            weights beforehand; "experts" 0 is one weight matrix, otherwise one an expert

With `own` false, run() is elementary torch in 32 bits; with `own` true it calls kebab_b200.
"""
import numpy as np
import torch

own = False

F = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # One sequence that produces one token: what counts is the latency of the call.
        {"name": "route token", "op": "route", "tokens": 1, "experts": 128, "k": 8, "dtype": "f32", "renorm": True, "train": False},
        # The router of one layer in a training step, 16-bit logits (so ties occur), weights of the softmax over all experts.
        {"name": "route train", "op": "route", "tokens": 32768, "experts": 64, "k": 6, "dtype": "bf16", "renorm": False, "train": True},
        # A serving batch's tokens to their experts' rows and back.
        {"name": "exchange batch", "op": "exchange", "tokens": 33, "experts": 64, "k": 8, "width": 4096, "dtype": "f16", "train": False},
        # The same in a training step, with every gradient: bound by memory.
        {"name": "exchange train", "op": "exchange", "tokens": 16384, "experts": 64, "k": 4, "width": 4096, "dtype": "bf16", "train": True},
        # One token through its 8 experts: 8 weight matrices are read for one row each.
        {"name": "experts token", "op": "grouped", "rows": 8, "experts": 64, "idle": 56, "n": 4096, "k": 2048, "dtype": "bf16", "skew": 0.0, "opmode": "RC", "train": False},
        # A serving batch: every expert's weights are read for a few rows each; weights stored K x N.
        {"name": "experts batch", "op": "grouped", "rows": 509, "experts": 64, "idle": 3, "n": 2048, "k": 4096, "dtype": "f16", "skew": 0.5, "opmode": "RR", "train": False},
        # A long prompt through few, large experts: bound by the matrix units.
        {"name": "experts prompt", "op": "grouped", "rows": 32768, "experts": 8, "idle": 0, "n": 8192, "k": 4096, "dtype": "bf16", "skew": 0.3, "opmode": "RC", "train": False},
        # A training step of one layer's products, unevenly loaded, two experts idle, with both gradients.
        {"name": "experts train", "op": "grouped", "rows": 16381, "experts": 16, "idle": 2, "n": 4096, "k": 2048, "dtype": "bf16", "skew": 0.8, "opmode": "RC", "train": True},
        # One token through a quantised projection: the weights are read once.
        {"name": "i8 token", "op": "i8", "rows": 1, "experts": 0, "idle": 0, "n": 8192, "k": 8192, "dtype": "bf16", "skew": 0.0, "bias": False},
        # A serving batch of 64 sequences through the same projection, with a bias.
        {"name": "i8 batch", "op": "i8", "rows": 64, "experts": 0, "idle": 0, "n": 8192, "k": 8192, "dtype": "f16", "skew": 0.0, "bias": True},
        # A prompt of odd length through the up-projection of a large model's feed-forward layer.
        {"name": "i8 prompt", "op": "i8", "rows": 4093, "experts": 0, "idle": 0, "n": 28672, "k": 8192, "dtype": "bf16", "skew": 0.0, "bias": False},
        # A serving batch through quantised experts.
        {"name": "i8 experts", "op": "i8", "rows": 1021, "experts": 32, "idle": 2, "n": 4096, "k": 4096, "dtype": "f16", "skew": 0.6, "bias": False},
    ]


def _spread(rng, low, high, step=1):
    """A multiple of `step` between the two, spread evenly over the logarithm."""
    v = int(round(low * (high / low) ** rng.random()))
    return max(low, min(high, v // step * step))


def draw(rng):
    op = rng.choice(("route", "exchange", "grouped", "grouped", "i8", "i8"))
    if op == "route":
        experts = _spread(rng, 8, 512)
        tokens = _spread(rng, 1, max(1, min(65536, 32768 * 64 // experts)))
        return {"op": op, "tokens": tokens, "experts": experts, "k": rng.randint(1, min(10, experts)), "dtype": rng.choice(("f16", "bf16", "f32")),
                "renorm": rng.random() < 0.5, "train": rng.random() < 0.5}
    if op == "exchange":
        k, width = rng.randint(1, 8), _spread(rng, 256, 8192, 8)
        return {"op": op, "tokens": _spread(rng, 1, max(1, 16384 * 4096 * 4 // (width * k))), "experts": _spread(rng, max(8, k), 256), "k": k, "width": width,
                "dtype": rng.choice(("f16", "bf16")), "train": rng.random() < 0.5}
    n, k, skew = _spread(rng, 512, 8192, 8), _spread(rng, 512, 8192, 8), round(rng.random(), 2)
    if op == "grouped":
        experts = _spread(rng, 2, max(2, min(128, (1 << 30) // (n * k))))
        train = rng.random() < 0.4
        rows = _spread(rng, 1, max(1, min(32768, 32768 * 8192 * 4096 // (n * k * (3 if train else 1)))))
        return {"op": op, "rows": rows, "experts": experts, "idle": rng.randint(0, experts // 2), "n": n, "k": k, "dtype": rng.choice(("f16", "bf16")), "skew": skew,
                "opmode": rng.choice(("RC", "RR")), "train": train}
    k = k // 16 * 16
    experts = rng.choice((0, 0, _spread(rng, 2, max(2, min(128, (1 << 30) // (n * k))))))
    rows = _spread(rng, 1, max(1, min(16384, 4093 * 28672 * 8192 // (n * k))))
    return {"op": op, "rows": rows, "experts": experts, "idle": rng.randint(0, experts // 2), "n": n + rng.choice((0, 0, 1, 3)), "k": k, "dtype": rng.choice(("f16", "bf16")),
            "skew": skew, "bias": not experts and rng.random() < 0.5}


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


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    op = case["op"]
    if op in ("route", "exchange"):
        T, E, k = case["tokens"], case["experts"], case["k"]
        # A router's logits: a preference that all tokens share, and each token's own.
        logits = 1.5 * _randn(g, T, E) + 0.7 * _randn(g, E)
        if op == "route":
            s["logits"] = logits.to(F[case["dtype"]])
            if case["train"]:
                s["dweights"] = _randn(g, T, k)
            return s
        top = torch.topk(logits, k, dim=1)
        s["weights"] = torch.softmax(top.values, dim=1)
        order = torch.argsort(top.indices.reshape(-1), stable=True)
        slots = torch.empty(T * k, dtype=torch.int32, device="cuda")
        slots[order] = torch.arange(T * k, dtype=torch.int32, device="cuda")
        s["slots"] = slots.view(T, k)
        dt, H = F[case["dtype"]], case["width"]
        s["x"] = _randn(g, T, H).to(dt)
        s["ys"] = _randn(g, T * k, H).to(dt)
        if case["train"]:
            s["dy"] = _randn(g, T, H).to(dt)
            s["dxs"] = _randn(g, T * k, H).to(dt)
        return s
    R, N, K, E, dt = case["rows"], case["n"], case["k"], case["experts"], F[case["dtype"]]
    if E:
        # Which experts are the popular ones is the seed's.
        counts = [_counts(case)[i] for i in torch.randperm(E, generator=torch.Generator().manual_seed(seed)).tolist()]
        s["counts"] = counts
        s["offsets"] = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")
    s["x"] = _randn(g, R, K).to(dt)
    if op == "grouped":
        W = torch.empty((E, N, K) if case["opmode"] == "RC" else (E, K, N), dtype=dt, device="cuda")
        for e in range(E):
            W[e] = _randn(g, *W.shape[1:]) * K ** -0.5
        s["w"] = W
        if case["train"]:
            s["dy"] = _randn(g, R, N).to(dt)
        return s
    # Activations with a few channels much larger than the others, as quantised models meet them.
    s["x"] = s["x"] * (1 + 9 * (torch.rand(K, generator=g, device="cuda") < 0.01)).to(dt)
    s["wq"] = torch.empty((max(E, 1), N, K), dtype=torch.int8, device="cuda")
    s["ws"] = torch.empty((max(E, 1), N), dtype=torch.float32, device="cuda")
    for e in range(max(E, 1)):
        w = _randn(g, N, K) * K ** -0.5
        s["ws"][e] = w.abs().amax(1) / 127
        s["wq"][e] = torch.round(w / s["ws"][e][:, None]).to(torch.int8)
    if not E:
        s["wq"], s["ws"] = s["wq"][0], s["ws"][0]
        if case["bias"]:
            s["b"] = _randn(g, N).to(dt)
    return s


def _ours(s):
    import kebab_b200 as kb

    op = s["op"]
    if op == "route":
        r = kb.route(s["logits"], s["k"], renormalize=s["renorm"])
        out = {"weights": r.weights, "experts": r.experts, "offsets": r.offsets, "slots": r.slots}
        if s["train"]:
            out["dlogits"] = kb.route_backward(s["logits"], r, s["dweights"], renormalize=s["renorm"])
        return out
    if op == "exchange":
        out = {"xs": kb.dispatch(s["x"], s["slots"]), "y": kb.combine(s["ys"], s["slots"], s["weights"])}
        if s["train"]:
            out["dys"], out["dweights"] = kb.combine_backward(s["dy"], s["ys"], s["slots"], s["weights"])
            out["dx"] = kb.combine(s["dxs"], s["slots"])
        return out
    if op == "grouped":
        out = {"y": kb.gemm_grouped(s["x"], s["w"], s["offsets"], opmode=s["opmode"])}
        if s["train"]:
            out["dx"] = kb.gemm_grouped(s["dy"], s["w"], s["offsets"], opmode="RR" if s["opmode"] == "RC" else "RC")
            out["dw"] = kb.gemm_grouped_dw(s["x"], s["dy"], s["offsets"], opmode=s["opmode"])
        return out
    if s["experts"]:
        return kb.linear_grouped_i8(s["x"], s["wq"], s["ws"], s["offsets"])
    return kb.linear_i8(s["x"], s["wq"], s["ws"], bias=s.get("b"))


def _route(s):
    x, k = s["logits"].float(), s["k"]
    T, E = x.shape
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]  # equal logits: the lower expert first
    p = torch.exp(x - x.amax(1, keepdim=True))
    top = torch.gather(p, 1, order)
    weights = top / (top if s["renorm"] else p).sum(1, keepdim=True)
    flat = order.reshape(-1)
    rows = torch.argsort(flat, stable=True)
    slots = torch.empty(T * k, dtype=torch.int32, device=x.device)
    slots[rows] = torch.arange(T * k, dtype=torch.int32, device=x.device)
    offsets = torch.zeros(E + 1, dtype=torch.int32, device=x.device)
    offsets[1:] = torch.cumsum(torch.bincount(flat, minlength=E), 0)
    out = {"weights": weights, "experts": order.to(torch.int32), "offsets": offsets, "slots": slots.view(T, k)}
    if s["train"]:
        g = torch.zeros_like(x)
        if s["renorm"]:
            g.scatter_(1, order, weights * (s["dweights"] - (weights * s["dweights"]).sum(1, keepdim=True)))
        else:
            p = p / p.sum(1, keepdim=True)
            g.scatter_(1, order, s["dweights"])
            g = p * (g - (p * g).sum(1, keepdim=True))
        out["dlogits"] = g.to(s["logits"].dtype)
    return out


def _exchange(s):
    slots, dt = s["slots"].long(), s["x"].dtype
    xs = torch.empty_like(s["ys"])
    xs[slots.reshape(-1)] = s["x"].repeat_interleave(s["k"], 0)
    ys = s["ys"].float()[slots]  # [tokens, k, width]
    out = {"xs": xs, "y": (ys * s["weights"][:, :, None]).sum(1).to(dt)}
    if s["train"]:
        dy = s["dy"].float()[:, None, :]
        out["dys"] = torch.empty_like(s["ys"])
        out["dys"][slots.reshape(-1)] = (dy * s["weights"][:, :, None]).to(dt).reshape(-1, s["width"])
        out["dweights"] = (dy * ys).sum(2)
        out["dx"] = s["dxs"].float()[slots].sum(1).to(dt)
    return out


def _parts(s, *tensors):
    return zip(*(torch.split(t.float(), s["counts"]) for t in tensors))


def _grouped(s):
    dt, W = s["x"].dtype, s["w"]
    W = W if s["opmode"] == "RC" else W.transpose(1, 2)  # [experts, N, K]
    out = {"y": torch.cat([x @ w.float().T for (x,), w in zip(_parts(s, s["x"]), W) if len(x)]).to(dt)}
    if s["train"]:
        out["dx"] = torch.cat([dy @ w.float() for (dy,), w in zip(_parts(s, s["dy"]), W) if len(dy)]).to(dt)
        dw = torch.stack([dy.T @ x for dy, x in _parts(s, s["dy"], s["x"])])
        out["dw"] = (dw if s["opmode"] == "RC" else dw.transpose(1, 2).contiguous()).to(dt)
    return out


def _i8(s):
    dt, x = s["x"].dtype, s["x"].float()
    top = x.abs().amax(1, keepdim=True)
    scale = top / 127
    q = torch.round(x * torch.where(top > 0, 127 / top, 0.0))
    if s["experts"]:
        y = torch.cat([a @ w.float().T * v for a, w, v in zip(torch.split(q, s["counts"]), s["wq"], s["ws"]) if len(a)])
    else:
        y = q @ s["wq"].float().T * s["ws"]
    y = y * scale
    if "b" in s:
        y = y + s["b"].float()
    return y.to(dt)


def run(state):
    if own:
        return _ours(state)
    return {"route": _route, "exchange": _exchange, "grouped": _grouped, "i8": _i8}[state["op"]](state)


def work(case):
    """What a pass cannot do without: each input read once, each output written once, two operations a product term."""
    op = case["op"]
    if op == "route":
        T, E, k, b = case["tokens"], case["experts"], case["k"], F[case["dtype"]].itemsize
        return {"bytes": T * E * b + 12 * T * k + 4 * (E + 1) + case["train"] * (4 * T * k + T * E * b), "flops": 4 * T * E * (1 + case["train"])}
    if op == "exchange":
        T, k, H = case["tokens"], case["k"], case["width"]
        row, plan = 2 * T * H, 8 * T * k
        # x to xs; ys to y; with gradients: dy (and ys once more) to dys and the weights' gradient; dxs to dx.
        b = row * (1 + k) + row * (k + 1) + plan
        f = 2 * T * k * H
        if case["train"]:
            b += row * (1 + 2 * k) + row * (k + 1) + 4 * T * k
            f += 4 * T * k * H
        return {"bytes": b, "flops": f}
    R, N, K, E = case["rows"], case["n"], case["k"], case["experts"]
    busy = sum(c > 0 for c in _counts(case)) if E else 1
    if op == "grouped":
        b, f = 2 * (R * K + R * N + busy * N * K), 2 * R * N * K
        if case["train"]:  # X, dY, W read; Y, dX, dW (of every expert) written
            b, f = b + 2 * (R * N + R * K + E * N * K), 3 * f
        return {"bytes": b + 4 * (E + 1), "flops": f}
    return {"bytes": 2 * R * K + 2 * R * N + busy * N * (K + 4) + 2 * N * case["bias"], "flops": 2 * R * N * K}


def _exact_route(s):
    x = s["logits"].double().cpu().numpy()
    T, E, k = x.shape[0], x.shape[1], s["k"]
    chosen = np.lexsort((np.broadcast_to(np.arange(E), x.shape), -x), axis=1)[:, :k]
    e = np.exp(x - np.max(x, axis=1, keepdims=True))
    mask = np.zeros_like(x)
    np.put_along_axis(mask, chosen, 1.0, axis=1)
    p = e / np.sum(e * (mask if s["renorm"] else 1.0), axis=1, keepdims=True)
    out = {"weights": np.take_along_axis(p, chosen, 1), "experts": None, "offsets": None, "slots": None}
    if s["train"]:
        if s["renorm"]:
            p = p * mask
        d = np.zeros_like(x)
        np.put_along_axis(d, chosen, s["dweights"].double().cpu().numpy(), axis=1)
        out["dlogits"] = p * d - p * np.sum(p * d, axis=1, keepdims=True)
    return out


def _exact_exchange(s):
    T, k, H = s["tokens"], s["k"], s["width"]
    flat = s["slots"].reshape(-1).long()
    token_of = torch.empty_like(flat)
    token_of[flat] = torch.arange(T * k, device=flat.device) // k
    out = {"xs": s["x"].double()[token_of]}
    y = torch.zeros(T, H, dtype=torch.float64, device=flat.device)
    for j in range(k):
        y += s["weights"][:, j : j + 1].double() * s["ys"][s["slots"][:, j].long()].double()
    out["y"] = y
    if s["train"]:
        w_of = torch.empty(T * k, dtype=torch.float64, device=flat.device)
        w_of[flat] = s["weights"].reshape(-1).double()
        out["dys"] = s["dy"].double()[token_of] * w_of[:, None]
        out["dweights"] = torch.stack([(s["dy"].double() * s["ys"][s["slots"][:, j].long()].double()).sum(1) for j in range(k)], 1)
        dx = torch.zeros_like(y)
        for j in range(k):
            dx += s["dxs"][s["slots"][:, j].long()].double()
        out["dx"] = dx
    return out


def _exact_products(s):
    E, at = max(s["experts"], 1), 0
    counts = s.get("counts", [s["rows"]])
    new = lambda *shape: torch.zeros(shape, dtype=torch.float64, device="cuda")  # noqa: E731
    if s["op"] == "i8":
        x = s["x"].double()
        step = x.abs().amax(1) / 127
        q = torch.where(step[:, None] > 0, torch.round(x / step[:, None]), 0.0)
        wq, ws = s["wq"].view(E, s["n"], s["k"]), s["ws"].view(E, s["n"])
        y = new(s["rows"], s["n"])
        for e in range(E):
            r = slice(at, at + counts[e])
            y[r] = torch.einsum("rk,nk->rn", q[r], wq[e].double()) * torch.outer(step[r], ws[e].double())
            at += counts[e]
        return y + s["b"].double() if "b" in s else y
    rc = s["opmode"] == "RC"
    out = {"y": new(s["rows"], s["n"])}
    if s["train"]:
        out["dx"], out["dw"] = new(s["rows"], s["k"]), new(*s["w"].shape)
    for e in range(E):
        r = slice(at, at + counts[e])
        w, x = s["w"][e].double(), s["x"][r].double()
        out["y"][r] = torch.einsum("rk,nk->rn" if rc else "rk,kn->rn", x, w)
        if s["train"]:
            dy = s["dy"][r].double()
            out["dx"][r] = torch.einsum("rn,nk->rk" if rc else "rn,kn->rk", dy, w)
            out["dw"][e] = torch.einsum("rn,rk->nk" if rc else "rn,rk->kn", dy, x)
        at += counts[e]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"route": _exact_route, "exchange": _exact_exchange, "grouped": _exact_products, "i8": _exact_products}[case["op"]](s)
