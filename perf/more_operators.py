"""Timed cases of three operators that an encoder's training and serving need beside the package's kernels:

* ``attention`` -- attention within packed users (documents): causal, a prefix that every query sees, scores capped by
                   a tanh, a bias that falls with distance, shared key/value heads; with gradients, and for a few
                   queries over long histories;
* ``embed``     -- embedding rows with a scale, and the table's gradient by sorted ids: of all rows, or of the touched
                   rows alone, ids by themselves or in bags;
* ``clip``      -- the norm of all gradients and the clipping by it, over many tensors of several types.

``own`` False: plain torch forms in 32 bits.  ``own`` True: the package's kernels.
"""

import math
import random

import torch

own = False


def listed():
    return [
        # one user's items through one attention layer of the encoder (8 heads of 64): a request by itself
        dict(name="attention one user", op="attention", segments=1, low=20, high=20, own_keys=False, key_low=0, key_high=0,
             heads=8, kv_heads=8, width=64, causal=True, prefix=0, cap=0.0, slopes=False, dtype="bfloat16", train=False),
        # a batch of 1024 users (100 items each on average) through one layer
        dict(name="attention 1024 users", op="attention", segments=1024, low=1, high=200, own_keys=False, key_low=0,
             key_high=0, heads=8, kv_heads=8, width=64, causal=True, prefix=0, cap=0.0, slopes=False, dtype="bfloat16",
             train=False),
        # a training step of the same layer on users of up to 1000 items, with a distance bias
        dict(name="attention train users", op="attention", segments=60, low=10, high=1000, own_keys=False, key_low=0,
             key_high=0, heads=8, kv_heads=8, width=64, causal=True, prefix=0, cap=0.0, slopes=True, dtype="float16",
             train=True),
        # two long documents in training: capped scores, a prefix seen by all, two key/value heads for eight
        dict(name="attention train long", op="attention", segments=2, low=4100, high=7001, own_keys=False, key_low=0,
             key_high=0, heads=8, kv_heads=2, width=128, causal=True, prefix=513, cap=30.0, slopes=False,
             dtype="bfloat16", train=True),
        # one new item for each of 64 users over their cached histories
        dict(name="attention 64 histories", op="attention", segments=64, low=1, high=1, own_keys=True, key_low=1000,
             key_high=16000, heads=16, kv_heads=4, width=128, causal=True, prefix=0, cap=0.0, slopes=False,
             dtype="bfloat16", train=False),
        # one item's ids, one in each of the 28 slots
        dict(name="embed 28 ids", op="embed", ids=28, rows=2800001, width=512, skew=1.0, bag=0, form="lookup", scale=1.0,
             dtype="bfloat16"),
        # a training step's ids of a table with a dense gradient, few rows being most of the ids
        dict(name="embed train 103k", op="embed", ids=103725, rows=50000, width=512, skew=3.0, bag=0, form="dense",
             scale=22.627417, dtype="bfloat16"),
        # the gradient of the encoder's bags for 256 users: 28 slots of two ids on average, of the touched rows alone
        dict(name="embed bags 1.4M", op="embed", ids=1450000, rows=2800001, width=512, skew=3.0, bag=2, form="sparse",
             scale=1.0, dtype="bfloat16"),
        # a narrow table in 32 bits, sizes off every tile
        dict(name="embed train ragged", op="embed", ids=40001, rows=9001, width=100, skew=2.0, bag=0, form="dense",
             scale=0.5, dtype="float32"),
        # the norms and biases of one layer
        dict(name="clip one layer", op="clip", count=12, low=512, high=1024, dtypes="float32", most=0.5),
        # all gradients of the encoder: 8 layers of 8 experts (512 to 1024), their attention, the first projection
        dict(name="clip encoder", op="clip", count=290, low=512, high=4194304, dtypes="bfloat16", most=1.0),
        # mixed types and odd sizes
        dict(name="clip mixed", op="clip", count=301, low=1, high=300001, dtypes="mixed", most=30.0),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("attention", "attention", "attention", "embed", "embed", "clip"))
    if op == "attention":
        train = rng.random() < 0.5
        kv = rng.choice((1, 2, 4, 8))
        heads = kv * rng.choice((1, 1, 2, 4))
        case = dict(op="attention", segments=_log(rng, 1, 1000), low=1, high=1, own_keys=False, key_low=0, key_high=0,
                    heads=heads, kv_heads=kv, width=rng.choice((32, 64, 64, 96, 128, 8 * rng.randint(1, 16))),
                    causal=rng.random() < 0.8, prefix=rng.choice((0, 0, _log(rng, 1, 300))), cap=rng.choice((0.0, 0.0, 20.0, 50.0)),
                    slopes=rng.random() < 0.3, dtype=rng.choice(("bfloat16", "bfloat16", "float16")), train=train)
        if not train and rng.random() < 0.4:  # a few queries over longer keys
            case.update(own_keys=True, high=_log(rng, 1, 16), segments=_log(rng, 1, 200))
            most = max(20, min(20000, 800000 // case["segments"], 200000000 // (case["segments"] * kv * case["width"])))
            case["key_high"] = _log(rng, 20, most)
            case["key_low"] = rng.randint(1, case["key_high"])
        else:
            most = int((3.0e8 / (heads * case["segments"])) ** 0.5)  # pairs of all heads
            most = max(1, min(most, 7000, 100000 // case["segments"], 50000000 // (case["segments"] * heads * case["width"])))
            case["high"] = _log(rng, 1, most)
            case["low"] = rng.randint(1, case["high"])
        return case
    if op == "embed":
        dtype = rng.choice(("bfloat16", "bfloat16", "float16", "float32"))
        width = rng.choice((512, 512, 64, 8 * rng.randint(1, 256), rng.randint(1, 1100)))
        form = rng.choice(("lookup", "dense", "dense", "sparse"))
        bag = rng.choice((0, 0, 2, 5)) if form != "lookup" else 0
        most = max(2, min(1450000, 370000000 // width))
        rows = _log(rng, 2 if dtype != "float16" else 100, 5000000)  # (sums that fp16 holds)
        if form != "sparse":
            rows = min(rows, 300000000 // width)
        return dict(op="embed", ids=_log(rng, 1, most), rows=rows, width=width, skew=rng.choice((1.0, 2.0, 3.0)), bag=bag,
                    form=form, scale=1.0 if dtype == "float16" else rng.choice((1.0, width ** 0.5)), dtype=dtype)
    count = _log(rng, 1, 400)
    high = _log(rng, 2, max(2, min(4000000, 80000000 // count)))
    return dict(op="clip", count=count, low=rng.randint(1, high), high=high,
                dtypes=rng.choice(("bfloat16", "float16", "float32", "mixed")), most=rng.choice((1.0, 1000.0, 1e9)))


# ------------------------------------------------------------------ inputs
def _lengths(case):
    """(query lengths, key lengths) of a case's segments: a user's program knows its batch on the host."""
    rng = random.Random(case["segments"] * 7919 + case["high"] * 31 + case["key_high"])
    n = [rng.randint(case["low"], case["high"]) for _ in range(case["segments"])]
    if not case["own_keys"]:
        return n, n
    return n, [rng.randint(case["key_low"], case["key_high"]) for _ in range(case["segments"])]


def _sizes(case):
    """Values of each gradient: matrices as a rule, and the vectors beside them."""
    rng = random.Random(case["count"] * 7919 + case["high"])
    if case["high"] == 4194304:  # an encoder: per layer 8 experts (two matrices, two biases), attention, two norms
        layer = [524288, 1024, 524288, 512] * 8 + [786432, 262144, 512, 512]
        return (layer * 8 + [7340032, 512])[: case["count"]]
    return [_log(rng, case["low"], case["high"]) if case["low"] < case["high"] else case["low"] for _ in range(case["count"])]


def _types(case):
    if case["dtypes"] != "mixed":
        return [getattr(torch, case["dtypes"])] * case["count"]
    return [(torch.bfloat16, torch.float32, torch.float16)[i % 3] for i in range(case["count"])]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, to=None):
        return torch.randn(shape, device="cuda", generator=g).mul_(std).to(dtype if to is None else to)

    s = dict(case=case)
    if case["op"] == "attention":
        dtype = getattr(torch, case["dtype"])
        H, K, D = case["heads"], case["kv_heads"], case["width"]
        nq, nk = _lengths(case)
        s["lengths"] = nq, nk
        Tq, Tk = sum(nq), sum(nk)

        def offsets(n):
            return torch.tensor([0] + n, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()

        s["offsets"] = offsets(nq)
        if case["own_keys"]:  # the histories' keys and values as a cache keeps them
            s["q"], s["k"], s["v"] = normal(Tq, H, D), normal(Tk, K, D), normal(Tk, K, D)
            s["k_offsets"] = offsets(nk)
        else:  # three parts of one projection
            fused = normal(Tq, H + 2 * K, D)
            s["q"], s["k"], s["v"] = fused[:, :H], fused[:, H:H + K], fused[:, H + K:]
            s["k_offsets"] = None
        s["prefix"] = None
        if case["prefix"]:
            s["prefix"] = torch.randint(0, case["prefix"] + 1, (case["segments"],), device="cuda", generator=g).to(torch.int32)
        s["slopes"] = None
        if case["slopes"]:
            s["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)]).cuda()
        if case["train"]:
            s["grad"] = normal(Tq, H, D)
    elif case["op"] == "embed":
        dtype = getattr(torch, case["dtype"])
        n, V, D = case["ids"], case["rows"], case["width"]
        # frequent ids are low numbers; an odd factor and a shift spread them over the table
        u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)
        ids = (u ** case["skew"] * V).long().clamp_(max=V - 1)
        s["ids"] = (ids * _odd_factor(V) + seed) % V
        s["bags"], B = None, n
        if case["bag"]:
            B = max(1, n // case["bag"])
            cuts = torch.randint(0, n + 1, (B - 1,), device="cuda", generator=g).sort().values
            s["bags"] = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), n)])
        if case["form"] != "sparse":
            s["table"] = normal(V, D, std=0.02)
        if case["form"] != "lookup":
            s["grad"] = normal(B, D)
        if case["form"] == "sparse":  # buffers that a program keeps: rows behind the last touched one stay as they are
            s["out_ids"] = torch.zeros(n, dtype=torch.int64, device="cuda")
            s["out_rows"] = torch.zeros(n, D, dtype=dtype, device="cuda")
    else:
        sizes, types = _sizes(case), _types(case)
        s["grads"] = [normal(n, std=0.003 * (1 + i % 5), to=t) for i, (n, t) in enumerate(zip(sizes, types))]
        s["flat"], s["out"] = _flat(s["grads"])  # what the optimiser reads
    return s


def _flat(tensors):
    """One buffer for each type, and every tensor's place in its type's buffer (on 16-byte boundaries)."""
    ends, spans = {}, []
    for t in tensors:
        at = ends.get(t.dtype, 0)
        spans.append((at, at + t.numel()))
        ends[t.dtype] = (at + t.numel() + 7) // 8 * 8
    flat = {d: torch.zeros(n, dtype=d, device="cuda") for d, n in ends.items()}
    return flat, [flat[t.dtype][a:b] for t, (a, b) in zip(tensors, spans)]


def _odd_factor(V):
    f = int(V * 0.6180339887) | 1
    while math.gcd(f, V) != 1:
        f += 2
    return f


# -------------------------------------------------------------- plain forms
def _batches(nq, nk, heads, width):
    """Runs of segments whose padded scores stay under 2^28 values (one segment at least)."""
    first = 0
    while first < len(nq):
        last, a, b = first, 0, 0
        while last < len(nq):
            a2, b2, count = max(a, nq[last]), max(b, nk[last]), last + 1 - first
            if last > first and count * max(heads * a2 * b2, b2 * heads * width) > 1 << 28:
                break
            a, b, last = a2, b2, last + 1
        yield first, last, a, b
        first = last


def _padded(offsets, first, last, longest, total):
    """Row numbers [segments, longest] of a run of segments, `total` where there is none."""
    start, end = offsets[first:last].long(), offsets[first + 1:last + 1].long()
    at = start[:, None] + torch.arange(longest, device=offsets.device)
    return torch.where(at < end[:, None], at, total), end - start


def _take(t, at):
    """Rows of t [T, heads, D] by number as [segments, heads, longest, D] in 32 bits; zeros behind a segment's end."""
    rows = t[at.clamp(max=t.shape[0] - 1)].float()
    return (rows * (at < t.shape[0])[..., None, None]).transpose(1, 2)


def _attention(s):
    case, q, k, v = s["case"], s["q"], s["k"], s["v"]
    (Tq, H, D), (Tk, K, _) = q.shape, k.shape
    G, scale, cap = H // K, D ** -0.5, case["cap"]
    q_off = s["offsets"]
    k_off = q_off if s["k_offsets"] is None else s["k_offsets"]
    device = q.device
    outs = [torch.zeros(Tq + 1, H, D, device=device)]  # the last row takes what is padded
    if case["train"]:
        outs += [torch.zeros(Tq + 1, H, D, device=device)] + [torch.zeros(Tk + 1, K, D, device=device) for _ in range(2)]
    for first, last, a, b in _batches(*s["lengths"], H, D):
        iq, nq = _padded(q_off, first, last, a, Tq)
        ik, nk = _padded(k_off, first, last, b, Tk)
        B = last - first
        Q = _take(q, iq).reshape(B, K, G * a, D)
        k32, v32 = _take(k, ik), _take(v, ik)
        t = (Q @ k32.transpose(-1, -2)).view(B, K, G, a, b) * scale
        if cap:
            th = torch.tanh(t / cap)
            t = cap * th
        i, j = torch.arange(a, device=device)[:, None], torch.arange(b, device=device)
        at = i + (nk - nq)[:, None, None]  # [B, a, 1]: the query's place among the keys
        if s["slopes"] is not None:
            t = t - s["slopes"].view(K, G, 1, 1) * (at - j).abs()[:, None, None].float()
        seen = (j < nk[:, None, None]) & (i < nq[:, None, None])
        if case["causal"]:
            near = j <= at
            if s["prefix"] is not None:
                near = near | (j < s["prefix"][first:last, None, None])
            seen = seen & near
        seen = seen[:, None, None]
        t = t.masked_fill(~seen, -math.inf)
        top = t.amax(-1, keepdim=True)
        e = torch.exp(t - torch.where(top == -math.inf, torch.zeros_like(top), top))
        total = e.sum(-1, keepdim=True)
        p = e / torch.where(total == 0, torch.ones_like(total), total)
        o = p.view(B, K, G * a, b) @ v32
        outs[0][iq] = o.view(B, H, a, D).transpose(1, 2)
        if case["train"]:
            dO = _take(s["grad"], iq).reshape(B, K, G * a, D)
            dp = (dO @ v32.transpose(-1, -2)).view(B, K, G, a, b)
            ds = p * (dp - (dO * o).sum(-1).view(B, K, G, a, 1))
            if cap:
                ds = ds * (1.0 - th * th)
            ds = ds.view(B, K, G * a, b) * scale
            outs[1][iq] = (ds @ k32).view(B, H, a, D).transpose(1, 2)
            outs[2][ik] = (ds.transpose(-1, -2) @ Q).transpose(1, 2)
            outs[3][ik] = (p.view(B, K, G * a, b).transpose(-1, -2) @ dO).transpose(1, 2)
    names = ("out", "grad_q", "grad_k", "grad_v")
    return {n: t[:-1].to(q.dtype) for n, t in zip(names, outs)}


def _embed(s):
    case, ids = s["case"], s["ids"]
    dtype = getattr(torch, case["dtype"])
    n, V, D = case["ids"], case["rows"], case["width"]
    out = {}
    if case["form"] != "sparse":
        out["out"] = (s["table"][ids].float() * case["scale"]).to(dtype)
    if case["form"] == "lookup":
        return out
    sorted_ids, order = torch.sort(ids, stable=True)
    if s["bags"] is not None:  # each id's bag
        order = torch.searchsorted(s["bags"], order, right=True) - 1
    new = torch.ones_like(sorted_ids, dtype=torch.bool)
    new[1:] = sorted_ids[1:] != sorted_ids[:-1]
    place = new.long().cumsum(0) - 1  # of each id among the distinct ones
    if case["form"] == "dense":
        total = torch.zeros(V, D, device=ids.device).index_add_(0, sorted_ids, s["grad"].float()[order])
        out["grad_table"] = (total * case["scale"]).to(dtype)
        return out
    total = torch.zeros(n, D, device=ids.device).index_add_(0, place, s["grad"].float()[order])
    out["ids"] = torch.zeros(n, dtype=torch.int64, device=ids.device).scatter_(0, place, sorted_ids)
    out["rows"] = (total * case["scale"]).to(dtype)
    out["count"] = place[-1:].to(torch.int32) + 1
    return out


def _clip(s):
    total = torch.stack([(t.float() * t.float()).sum() for t in s["grads"]]).sum()
    norm = torch.sqrt(total)
    factor = (s["case"]["most"] / (norm + 1e-6)).clamp(max=1.0)
    for t, o in zip(s["grads"], s["out"]):
        o.copy_(t.float() * factor)
    return dict(norm=norm, grads=list(s["flat"].values()))


# ------------------------------------------------------- the package's calls
def _own_attention(s):
    from baidu_cti_grab_b200 import device_ops

    case = s["case"]
    how = dict(causal=case["causal"], prefix=s["prefix"], slopes=s["slopes"], cap=case["cap"])
    where = s["offsets"], s["k_offsets"]
    out, lse = device_ops.segment_attention(s["q"], s["k"], s["v"], *where, want_lse=case["train"], **how)
    if not case["train"]:
        return dict(out=out)
    dq, dk, dv = device_ops.segment_attention_backward(s["grad"], s["q"], s["k"], s["v"], out, lse, *where, **how)
    return dict(out=out, grad_q=dq, grad_k=dk, grad_v=dv)


def _own_embed(s):
    from baidu_cti_grab_b200 import device_ops

    case = s["case"]
    out = {}
    if case["form"] != "sparse":
        out["out"] = device_ops.embed_rows(s["table"], s["ids"], scale=case["scale"])
    if case["form"] == "dense":
        out["grad_table"] = device_ops.embed_rows_backward(s["grad"], s["ids"], case["rows"], bags=s["bags"], scale=case["scale"])
    elif case["form"] == "sparse":
        ids, rows, count = device_ops.embed_rows_backward_sparse(s["grad"], s["ids"], case["rows"], bags=s["bags"],
                                                                 scale=case["scale"], out=(s["out_ids"], s["out_rows"]))
        out.update(ids=ids, rows=rows, count=count)
    return out


def _own_clip(s):
    from baidu_cti_grab_b200 import device_ops

    norm = device_ops.clip_grads(s["grads"], s["case"]["most"], out=s["out"])
    return dict(norm=norm, grads=list(s["flat"].values()))


def run(state):
    op = state["case"]["op"]
    if own:
        return {"attention": _own_attention, "embed": _own_embed, "clip": _own_clip}[op](state)
    return {"attention": _attention, "embed": _embed, "clip": _clip}[op](state)


# ---------------------------------------------------------------- the work
def _size(name):
    return 4 if name == "float32" else 2


def _pairs(case):
    """Scores that the mask leaves, of one head (a prefix at half of its bound)."""
    total = 0
    for n, m in zip(*_lengths(case)):
        if not case["causal"]:
            total += n * m
            continue
        x = min(case["prefix"] // 2, m)
        i = max(0, min(n, x - 1 - (m - n)))  # queries that the prefix gives all they see
        total += i * x
        a, b = max(i + m - n + 1, 0), m
        total += (a + b) * (b - a + 1) // 2 if b >= a else 0
    return total


def _distinct(n, V, skew):
    """How many different rows n ids are, on average: the sum over rows of 1 - (1 - p)^n."""
    total, steps = 0.0, 4000
    for i in range(steps):  # rows in runs that grow geometrically
        lo, hi = V ** (i / steps) - 1.0, V ** ((i + 1) / steps) - 1.0
        if hi <= lo:
            continue
        a, b = min(lo / V, 1.0), min(hi / V, 1.0)
        p = (b ** (1 / skew) - a ** (1 / skew)) / (hi - lo)
        total += (hi - lo) * (1.0 - math.exp(-n * p))
    return int(min(total, n, V))


def work(case):
    if case["op"] == "attention":
        nq, nk = (sum(n) for n in _lengths(case))
        H, K, D = case["heads"], case["kv_heads"], case["width"]
        e, pairs = _size(case["dtype"]), _pairs(case) * H
        n, f = e * D * (2 * nq * H + 2 * nk * K), 4 * D * pairs
        if case["train"]:  # q, k, v and out are read again for the gradients, the output's gradient once
            n += e * D * (3 * nq * H + 2 * nk * K) + e * D * (nq * H + 2 * nk * K)
            f += 10 * D * pairs
        return dict(bytes=n, flops=f)
    if case["op"] == "embed":
        n, V, D, e = case["ids"], case["rows"], case["width"], _size(case["dtype"])
        some = _distinct(n, V, case["skew"])
        b, f = 8 * n, 0
        if case["form"] != "sparse":
            b += some * D * e + n * D * e
            f += n * D
        if case["form"] != "lookup":
            bags = max(1, n // case["bag"]) if case["bag"] else n
            b += bags * D * e + (8 * bags if case["bag"] else 0)
            f += n * D
            b += V * D * e if case["form"] == "dense" else some * (D * e + 8)
        return dict(bytes=b, flops=f)
    b = sum(n * _size(str(t).split(".")[1]) for n, t in zip(_sizes(case), _types(case)))
    return dict(bytes=2 * b, flops=3 * sum(_sizes(case)))


# ------------------------------------------- the definitions, in 64 bits
def _exact_attention(case, s):
    H, K, D = case["heads"], case["kv_heads"], case["width"]
    nq, nk = _lengths(case)
    if max(nq) * max(nk) * H > 1 << 30:
        return None
    results, a, c = [], 0, 0
    for u, (n, m) in enumerate(zip(nq, nk)):
        leaves = [s["q"][a:a + n].double(), s["k"][c:c + m].double(), s["v"][c:c + m].double()]
        if case["train"]:
            leaves = [t.requires_grad_() for t in leaves]
        q, k, v = leaves
        place = torch.arange(m - n, m, device=q.device)[:, None]
        j = torch.arange(m, device=q.device)[None]
        hidden = torch.zeros(n, m, dtype=torch.bool, device=q.device)
        if case["causal"]:
            hidden = j > place
            if s["prefix"] is not None:
                hidden = hidden & (j >= s["prefix"][u])
        none = hidden.all(-1)
        heads = []
        for h in range(H):
            x = q[:, h] @ k[:, h * K // H].t() / math.sqrt(D)
            if case["cap"]:
                x = case["cap"] * torch.tanh(x / case["cap"])
            if s["slopes"] is not None:
                x = x - float(s["slopes"][h]) * (place - j).abs()
            x = x.masked_fill(hidden & ~none[:, None], -math.inf)
            heads.append(torch.softmax(x, -1).masked_fill(none[:, None], 0.0) @ v[:, h * K // H])
        out = torch.stack(heads, 1)
        each = [out.detach()]
        if case["train"]:
            each += torch.autograd.grad((out * s["grad"][a:a + n].double()).sum(), leaves)
        results.append(each)
        a, c = a + n, c + m
    return {name: torch.cat(parts) for name, parts in zip(("out", "grad_q", "grad_k", "grad_v"), zip(*results))}


def _exact_embed(case, s):
    n, V, D = case["ids"], case["rows"], case["width"]
    out = {}
    if case["form"] != "sparse":
        out["out"] = s["table"].index_select(0, s["ids"]).double() * case["scale"]
    if case["form"] == "lookup":
        return out
    each = s["grad"].double()
    if s["bags"] is not None:
        each = each.repeat_interleave(s["bags"].diff(), 0)
    if case["form"] == "dense":
        out["grad_table"] = torch.zeros(V, D, dtype=torch.float64, device="cuda").index_add_(0, s["ids"], each) * case["scale"]
        return out
    some, where = torch.unique(s["ids"], return_inverse=True)
    out["ids"] = out["count"] = None
    out["rows"] = torch.zeros(n, D, dtype=torch.float64, device="cuda").index_add_(0, where, each) * case["scale"]
    return out


def _exact_clip(case, s):
    norm = torch.linalg.vector_norm(torch.cat([t.double().flatten() for t in s["grads"]]))
    factor = min(1.0, case["most"] / (float(norm) + 1e-6))
    grads = [torch.zeros(f.shape, dtype=torch.float64, device="cuda") for f in s["flat"].values()]
    ends = [0] * len(grads)
    for t in s["grads"]:
        i = list(s["flat"]).index(t.dtype)
        grads[i][ends[i]:ends[i] + t.numel()] = t.double() * factor
        ends[i] += -(-t.numel() // 8) * 8
    return dict(norm=norm, grads=grads)


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "embed": _exact_embed, "clip": _exact_clip}[case["op"]](case, s)
