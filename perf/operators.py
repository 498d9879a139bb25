"""Timed cases of three operators that stand between the package's kernels:

* ``route``   -- the choice of experts that ``device_ops.smoe_experts`` takes: scores from logits, an optional balance
                 bias, groups, top-k, renormalised weights; with the gradient of the logits;
* ``norm``    -- the norm after a block, its gate and residual scale, and the norm before the next block; with gradients;
* ``adapter`` -- low-rank adapters of many requests beside a projection that they share.

``own`` False: plain torch forms in 32 bits (64 for the choice of experts).  ``own`` True: the package's kernels.
"""

import math

import torch

own = False

CHANNEL, ROW, FULL = "channel", "row", "full"


def listed():
    return [
        # one token through the gate of the encoder's SMoE (8 experts, top-2): a request scored by itself
        dict(name="route one token", op="route", tokens=1, experts=8, k=2, score="softmax", bias=False, groups=1,
             topk_groups=1, group_top=1, renorm=False, scale=1.0, dtype="bfloat16", probs=True, train=False),
        # the same gate on a batch of 1024 users, with the probabilities that the balance loss sums
        dict(name="route 103k of 8", op="route", tokens=103725, experts=8, k=2, score="softmax", bias=False, groups=1,
             topk_groups=1, group_top=1, renorm=False, scale=1.0, dtype="bfloat16", probs=True, train=False),
        # many small experts in groups, balanced by a bias instead of a loss
        dict(name="route 16k of 256 grouped", op="route", tokens=16411, experts=256, k=8, score="sigmoid", bias=True,
             groups=8, topk_groups=4, group_top=2, renorm=True, scale=2.5, dtype="float32", probs=False, train=False),
        # a training step's routing: weights and probabilities forward, the logits' gradient backward
        dict(name="route train 24k of 64", op="route", tokens=24490, experts=64, k=6, score="softmax", bias=False,
             groups=1, topk_groups=1, group_top=1, renorm=True, scale=1.0, dtype="bfloat16", probs=True, train=True),
        # one token between two blocks at the encoder's width
        dict(name="norm one row", op="norm", rows=1, width=512, post="layer", pre="layer", gate=CHANNEL, act="none",
             scale=1.0, dtype="bfloat16", wdtype="bfloat16", train=False),
        # a batch of 1024 users between two blocks of the encoder
        dict(name="norm 103k x 512", op="norm", rows=103725, width=512, post="layer", pre="layer", gate=CHANNEL,
             act="none", scale=1.0, dtype="bfloat16", wdtype="bfloat16", train=False),
        # a training step with a gate computed per element
        dict(name="norm train 24k x 512", op="norm", rows=24490, width=512, post="layer", pre="layer", gate=FULL,
             act="sigmoid", scale=0.5, dtype="float16", wdtype="float16", train=True),
        # a wide model's training step: RMS norms with 32-bit weights, one gate a row, a width off the power of two
        dict(name="norm train 4k x 5000 rms", op="norm", rows=4099, width=5000, post="rms", pre="rms", gate=ROW,
             act="none", scale=0.7, dtype="bfloat16", wdtype="float32", train=True),
        # one new token for each of 64 requests, each with an adapter of its own choice, beside a fused q/k/v projection
        dict(name="adapter 64 requests", op="adapter", tokens=64, inputs=512, outputs=1536, rank=16, adapters=32,
             run=1, dtype="bfloat16"),
        # a batch of 1024 users (100 items each on average), an adapter per user, beside a 512 x 512 projection
        dict(name="adapter 103k x 512", op="adapter", tokens=103725, inputs=512, outputs=512, rank=16, adapters=32,
             run=100, dtype="bfloat16"),
        # beside the RepEncoder's Linear(14336 -> 512)
        dict(name="adapter 4k x 14336", op="adapter", tokens=4099, inputs=14336, outputs=512, rank=32, adapters=16,
             run=100, dtype="bfloat16"),
        # short requests in fp16 with sizes off every tile
        dict(name="adapter 9k ragged", op="adapter", tokens=9001, inputs=1000, outputs=1544, rank=8, adapters=24,
             run=7, dtype="float16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("route", "norm", "adapter"))
    dtype = rng.choice(("bfloat16", "bfloat16", "float16", "float32"))
    if op == "route":
        train = rng.random() < 0.4
        if rng.random() < 0.5:
            experts, groups = rng.randint(2, 384), 1
        else:
            groups = rng.choice((2, 4, 8))
            experts = groups * rng.randint(2, 48)
        topk_groups = rng.randint(1, groups)
        k = rng.randint(1, min(10, experts // groups * topk_groups))
        tokens = max(1, min(_log(rng, 1, 200000), 4200000 // experts))
        return dict(op="route", tokens=tokens, experts=experts, k=k, score=rng.choice(("softmax", "sigmoid")),
                    bias=rng.random() < 0.5, groups=groups, topk_groups=topk_groups, group_top=rng.choice((1, 2)),
                    renorm=k > 1 and rng.random() < 0.5, scale=rng.choice((1.0, 2.5)), dtype=dtype, probs=rng.random() < 0.5,
                    train=train)
    if op == "norm":
        width = rng.choice((512, 512, 1024, 2048, 8 * rng.randint(4, 1024), rng.randint(33, 8192)))
        train = rng.random() < 0.5
        most = 20000000 // width if train else 50000000 // width
        return dict(op="norm", rows=max(1, min(_log(rng, 1, 100000), most)), width=width,
                    post=rng.choice(("layer", "rms", "none")), pre=rng.choice(("layer", "rms", "none")),
                    gate=rng.choice(("none", CHANNEL, ROW, FULL)), act=rng.choice(("none", "sigmoid")),
                    scale=rng.choice((1.0, 0.5)), dtype=dtype,
                    wdtype=dtype if rng.random() < 0.5 else "float32", train=train)
    dtype = rng.choice(("bfloat16", "bfloat16", "float16"))
    inputs = 8 * _log(rng, 8, 1792)
    outputs = rng.choice((512, 1536, 8 * _log(rng, 8, 512), rng.randint(65, 2000)))
    rank = rng.choice((8, 16, 16, 32, 64))
    adapters = rng.randint(1, 1024 // rank)
    tokens = max(1, min(_log(rng, 1, 100000), 50000000 // max(inputs, outputs)))
    return dict(op="adapter", tokens=tokens, inputs=inputs, outputs=outputs, rank=rank, adapters=adapters,
                run=_log(rng, 1, 200), dtype=dtype)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case, seed):
    g = _gen(seed)
    dtype = getattr(torch, case["dtype"])

    def normal(*shape, std=1.0, mean=0.0, to=dtype):
        return torch.randn(shape, device="cuda", generator=g).mul_(std).add_(mean).to(to)

    s = dict(case=case)
    if case["op"] == "route":
        T, E, k = case["tokens"], case["experts"], case["k"]
        # some experts are liked more than others, and a few tokens may not use some experts (masked: -inf)
        s["logits"] = normal(T, E, to=torch.float32).add_(normal(E, std=0.5, to=torch.float32)).to(dtype)
        if T > 64 and E > 4 * k and case["groups"] == 1:
            s["logits"][::61, : E // 4] = -math.inf
        s["bias"] = normal(E, std=0.05, to=torch.float32) if case["bias"] else None
        if case["train"]:
            s["grad_score"] = normal(T, k)
            s["grad_probs"] = normal(T, E, std=0.01) if case["probs"] else None
    elif case["op"] == "norm":
        N, D, wt = case["rows"], case["width"], getattr(torch, case["wdtype"])
        s["x"], s["h"] = normal(N, D, std=2.0), normal(N, D, std=0.7, mean=0.1)
        for which in ("post", "pre"):
            kind = case[which]
            s[which + "_weight"] = normal(D, std=0.1, mean=1.0, to=wt) if kind != "none" else None
            s[which + "_bias"] = normal(D, std=0.05, to=wt) if kind == "layer" else None
        shape = {CHANNEL: (D,), ROW: (N, 1), FULL: (N, D)}.get(case["gate"])
        s["gate"] = normal(*shape, std=0.5, mean=0.5) if shape else None
        if case["train"]:
            s["grad_y"] = normal(N, D)
            s["grad_z"] = normal(N, D) if case["pre"] != "none" else None
    else:
        T, K, N, r, R = (case[n] for n in ("tokens", "inputs", "outputs", "rank", "adapters"))
        s["x"], s["y"] = normal(T, K), normal(T, N)
        s["a"], s["b"] = normal(R, r, K, std=K ** -0.5), normal(R, N, r, std=r ** -0.5)
        s["scale"] = torch.rand(R, device="cuda", generator=g).add_(0.5)
        # requests of `run` tokens on average, each with one adapter; one in nine has none
        starts = torch.rand(T, device="cuda", generator=g) < 1.0 / case["run"]
        request = starts.long().cumsum(0)
        chosen = torch.randint(0, R, (T + 1,), device="cuda", generator=g)
        chosen[::9] = -1
        s["adapter"] = chosen[request].to(torch.int32)
    return s


# -------------------------------------------------------------- plain forms
def _masked(logits):
    return logits <= torch.finfo(logits.dtype).min


def _scores(logits, kind, to):
    out = _masked(logits)
    v = logits.to(to)
    if kind == "sigmoid":
        return (1.0 / (1.0 + torch.exp(-v))).masked_fill(out, 0.0)
    top = v.masked_fill(out, -math.inf).amax(-1, keepdim=True)
    e = torch.exp(v - top).masked_fill(out, 0.0)
    total = e.sum(-1, keepdim=True)
    return torch.where(total == 0, torch.zeros_like(e), e / total)


def _choose(case, logits, bias):
    """The chosen experts [T, k], decided in 64 bits, ties to the lowest index."""
    T, E = logits.shape
    G = case["groups"]
    c = _scores(logits, case["score"], torch.float64)
    if bias is not None:
        c = c + bias.double()
    elif case["group_top"] == 1 or G == 1:
        c = logits.double()  # the scores' own order
    c = c.masked_fill(_masked(logits), -math.inf)
    if G > 1:
        each = c.view(T, G, E // G)
        value = torch.sort(each, dim=-1, descending=True).values[..., : case["group_top"]].sum(-1)
        best = torch.sort(value, dim=-1, descending=True, stable=True).indices[:, : case["topk_groups"]]
        keep = torch.zeros(T, G, dtype=torch.bool, device=c.device).scatter_(1, best, True)
        # the experts of other groups come behind every expert of the chosen groups, masked ones included
        rank = torch.sort(c, dim=-1, descending=True, stable=True).indices
        kept = keep.repeat_interleave(E // G, 1).gather(1, rank)
        order = torch.sort((~kept).to(torch.int8), dim=-1, stable=True).indices
        return rank.gather(1, order)[:, : case["k"]]
    return torch.sort(c, dim=-1, descending=True, stable=True).indices[:, : case["k"]]


def _route(s):
    case, logits = s["case"], s["logits"]
    idx = _choose(case, logits, s["bias"])
    p = _scores(logits, case["score"], torch.float32)
    picked = p.gather(1, idx)
    total = picked.sum(-1, keepdim=True)
    w = torch.where(total == 0, torch.zeros_like(picked), picked / total) if case["renorm"] else picked
    out = dict(idx=idx, score=(w * case["scale"]).to(logits.dtype))
    if case["probs"]:
        out["probs"] = p.to(logits.dtype)
    if case["train"]:
        dw = s["grad_score"].float() * case["scale"]
        if case["renorm"]:
            dw = torch.where(total == 0, torch.zeros_like(dw), (dw - (dw * w).sum(-1, keepdim=True)) / total)
        ds = torch.zeros_like(p).scatter_(1, idx, dw)
        if s["grad_probs"] is not None:
            ds = ds + s["grad_probs"].float()
        if case["score"] == "sigmoid":
            dl = ds * p * (1.0 - p)
        else:
            dl = p * (ds - (ds * p).sum(-1, keepdim=True))
        out["grad_logits"] = dl.to(logits.dtype)
    return out


def _norm(v, kind, weight, bias):
    """(normalised and scaled, normalised, 1 / deviation)"""
    if kind == "none":
        return v, None, None
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-5)
    hat = v * r
    out = hat * weight.float()
    return (out if bias is None else out + bias.float()), hat, r


def _norm_backward(d, hat, r, kind, weight):
    if kind == "none":
        return d
    d = d * weight.float()
    back = d - hat * (d * hat).mean(-1, keepdim=True)
    if kind == "layer":
        back = back - d.mean(-1, keepdim=True)
    return back * r


def _sandwich(s):
    case = s["case"]
    x, h = s["x"].float(), s["h"].float()
    n, h_hat, h_r = _norm(h, case["post"], s["post_weight"], s["post_bias"])
    g = s["gate"]
    if g is None:
        a = torch.ones((), device=x.device)
    else:
        a = 1.0 / (1.0 + torch.exp(-g.float())) if case["act"] == "sigmoid" else g.float()
    y = x + case["scale"] * a * n
    z, y_hat, y_r = _norm(y, case["pre"], s["pre_weight"], s["pre_bias"])
    out = dict(y=y.to(s["x"].dtype))
    if case["pre"] != "none":
        out["z"] = z.to(s["x"].dtype)
    if case["train"]:
        t = s["grad_y"].float()
        if s["grad_z"] is not None:
            dz = s["grad_z"].float()
            t = t + _norm_backward(dz, y_hat, y_r, case["pre"], s["pre_weight"])
            out["grad_pre_weight"] = (dz * y_hat).sum(0).to(s["pre_weight"].dtype)
            if s["pre_bias"] is not None:
                out["grad_pre_bias"] = dz.sum(0).to(s["pre_bias"].dtype)
        out["grad_x"] = t.to(s["x"].dtype)
        dn = case["scale"] * a * t
        if g is not None:
            dg = case["scale"] * n * t
            if case["act"] == "sigmoid":
                dg = dg * a * (1.0 - a)
            out["grad_gate"] = dg.sum_to_size(g.shape).to(g.dtype)
        if case["post"] != "none":
            out["grad_post_weight"] = (dn * h_hat).sum(0).to(s["post_weight"].dtype)
            if s["post_bias"] is not None:
                out["grad_post_bias"] = dn.sum(0).to(s["post_bias"].dtype)
        out["grad_h"] = _norm_backward(dn, h_hat, h_r, case["post"], s["post_weight"]).to(s["h"].dtype)
    return out


def _adapter(s):
    x, y, a, b, i = s["x"].float(), s["y"].float(), s["a"].float(), s["b"].float(), s["adapter"].long()
    R, r, K = a.shape
    every = x @ a.view(R * r, K).t()  # every adapter's products, then each token's own
    mine = (i[:, None] == torch.arange(R, device=i.device)).float() * s["scale"]
    every = every.view(-1, R, r) * mine[..., None]
    delta = every.view(-1, R * r) @ b.permute(0, 2, 1).reshape(R * r, -1)
    return dict(out=(y + delta).to(s["y"].dtype))


# ------------------------------------------------------- the package's calls
def _own_route(s):
    from baidu_cti_grab_b200 import device_ops

    case = s["case"]
    how = dict(score=case["score"], renormalize=case["renorm"], scale=case["scale"])
    idx, score, probs, _ = device_ops.route_topk(
        s["logits"], case["k"], bias=s["bias"], groups=case["groups"], topk_groups=case["topk_groups"],
        group_top=case["group_top"], want_probs=case["probs"], **how)
    out = dict(idx=idx, score=score)
    if case["probs"]:
        out["probs"] = probs
    if case["train"]:
        out["grad_logits"] = device_ops.route_topk_backward(s["logits"], idx, s["grad_score"], s["grad_probs"], **how)
    return out


def _own_norm(s):
    from baidu_cti_grab_b200 import device_ops

    case = s["case"]
    kind = {"none": None}
    how = dict(post=kind.get(case["post"], case["post"]), post_weight=s["post_weight"], post_bias=s["post_bias"],
               gate=s["gate"], gate_act=case["act"], scale=case["scale"],
               pre=kind.get(case["pre"], case["pre"]), pre_weight=s["pre_weight"], pre_bias=s["pre_bias"])
    y, z, stats = device_ops.sandwich_norm(s["x"], s["h"], want_stats=case["train"], **how)
    out = dict(y=y)
    if z is not None:
        out["z"] = z
    if case["train"]:
        grads = device_ops.sandwich_norm_backward(s["grad_y"], s["grad_z"], s["x"], s["h"], stats, **how)
        names = ("grad_x", "grad_h", "grad_gate", "grad_post_weight", "grad_post_bias", "grad_pre_weight",
                 "grad_pre_bias")
        out.update((n, v) for n, v in zip(names, grads) if v is not None)
    return out


def _own_adapter(s):
    from baidu_cti_grab_b200 import device_ops

    return dict(out=device_ops.low_rank_add(s["y"], s["x"], s["a"], s["b"], s["adapter"], s["scale"]))


def run(state):
    op = state["case"]["op"]
    if own:
        return {"route": _own_route, "norm": _own_norm, "adapter": _own_adapter}[op](state)
    return {"route": _route, "norm": _sandwich, "adapter": _adapter}[op](state)


# ---------------------------------------------------------------- the work
def _size(name):
    return 4 if name == "float32" else 2


def work(case):
    e = _size(case["dtype"])
    if case["op"] == "route":
        T, E, k = case["tokens"], case["experts"], case["k"]
        n = T * E * e * (1 + case["probs"]) + T * k * (8 + e)
        f = T * E * 4
        if case["train"]:  # the logits and choices are read once for both directions
            n += T * k * e + T * E * e * (1 + case["probs"])
            f += T * E * 4
        return dict(bytes=n, flops=f)
    if case["op"] == "norm":
        N, D, w = case["rows"], case["width"], _size(case["wdtype"])
        gate = {CHANNEL: D, ROW: N, FULL: N * D}.get(case["gate"], 0) * e
        affine = D * w * sum({"layer": 2, "rms": 1, "none": 0}[case[p]] for p in ("post", "pre"))
        second = case["pre"] != "none"
        n, f = N * D * e * (3 + second) + gate + affine, N * D * 14
        if case["train"]:
            n += N * D * e * (3 + second) + gate + affine
            f += N * D * 24
        return dict(bytes=n, flops=f)
    T, K, N, r, R = (case[n] for n in ("tokens", "inputs", "outputs", "rank", "adapters"))
    used = min(R, T)
    return dict(bytes=e * (T * K + 2 * T * N + used * r * (K + N)) + 4 * T + 4 * R, flops=2 * T * r * (K + N))


# ------------------------------------------- the definitions, in 64 bits
def _exact_route(case, s):
    l = s["logits"].double().requires_grad_(case["train"])
    T, E = l.shape
    hidden = s["logits"] <= torch.finfo(s["logits"].dtype).min
    empty = hidden.all(-1, keepdim=True)
    if case["score"] == "sigmoid":
        p = torch.sigmoid(l).masked_fill(hidden, 0.0)
    else:
        p = torch.softmax(l.masked_fill(hidden & ~empty, -math.inf), -1).masked_fill(hidden, 0.0)
    # the choice, one expert after another
    with torch.no_grad():
        c = p.detach().clone() if s["bias"] is None else p.detach() + s["bias"].double()
        c[hidden] = -math.inf
        if case["groups"] > 1:
            each = c.view(T, case["groups"], -1)
            value = each.topk(case["group_top"], -1).values.sum(-1)
            last = value.topk(case["topk_groups"], -1).values[:, -1:]
            c = each.masked_fill((value < last)[..., None], -math.inf).view(T, E)
        chosen = []
        for _ in range(case["k"]):
            chosen.append(c.argmax(-1))
            c.scatter_(1, chosen[-1][:, None], -math.inf)
        idx = torch.stack(chosen, -1)
    w = p.gather(1, idx)
    if case["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    w = w * case["scale"]
    out = dict(idx=None, score=w.detach())
    if case["probs"]:
        out["probs"] = p.detach()
    if case["train"]:
        total = (w * s["grad_score"].double()).sum()
        if s["grad_probs"] is not None:
            total = total + (p * s["grad_probs"].double()).sum()
        out["grad_logits"] = torch.autograd.grad(total, l)[0]
    return out


def _exact_norm(case, s):
    names = [n for n in ("x", "h", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias") if s[n] is not None]
    v = {n: s[n].double().requires_grad_(case["train"]) for n in names}
    D = (case["width"],)

    def apply(t, which):
        if case[which] == "layer":
            return torch.nn.functional.layer_norm(t, D, v[which + "_weight"], v[which + "_bias"], 1e-5)
        if case[which] == "rms":
            return torch.nn.functional.rms_norm(t, D, v[which + "_weight"], 1e-5)
        return t

    branch = apply(v["h"], "post")
    if "gate" in v:
        branch = branch * (torch.sigmoid(v["gate"]) if case["act"] == "sigmoid" else v["gate"])
    y = v["x"] + branch * case["scale"]
    out = dict(y=y.detach())
    total = 0.0
    if case["pre"] != "none":
        z = apply(y, "pre")
        out["z"] = z.detach()
        if case["train"]:
            total = (z * s["grad_z"].double()).sum()
    if case["train"]:
        total = total + (y * s["grad_y"].double()).sum()
        out.update(("grad_" + n, d) for n, d in zip(names, torch.autograd.grad(total, [v[n] for n in names])))
    return out


def _exact_adapter(case, s):
    out = s["y"].double()
    for i in range(case["adapters"]):
        t = (s["adapter"] == i).nonzero()[:, 0]
        h = s["x"][t].double() @ s["a"][i].double().t()
        out[t] += s["scale"][i].double() * (h @ s["b"][i].double().t())
    return dict(out=out)


def exact(case, seed):
    s = prepare(case, seed)
    return {"route": _exact_route, "norm": _exact_norm, "adapter": _exact_adapter}[case["op"]](case, s)
