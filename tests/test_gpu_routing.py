"""Routing to experts (rb_route_topk, rb_route_topk_backward, routing.py) on the GPU against
the definition in float64.

The choice is exact: every index has to be the definition's, ties at the lowest index.
Tolerances of the computed numbers, u = 2^-24: a softmax score takes the rounding of l - max
(at most |l - max| u, under 32 u for these inputs), expf (2 u), a sum of positive terms over
V values a lane and up to five shuffles (21 u), its reciprocal and a product (2 u): under
62 u < 2^-18.  A sigmoid and a renormalised weight take fewer.  Each output is then rounded
once to its type: eps / 2, or half the smallest subnormal.  A gradient s (ds - sum ds s) with
ds = (g - sum(g s) / total) / total takes at most four such factors: 2^-16 of the magnitudes
it is summed from, and its rounding.
"""

import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _half_step(dtype):
    fi = torch.finfo(dtype)
    return fi.eps / 2, fi.smallest_normal * fi.eps / 2


def _scores(logits, kind):
    hidden = logits <= torch.finfo(logits.dtype).min
    v = logits.double()
    if kind == "sigmoid":
        return torch.sigmoid(v).masked_fill(hidden, 0.0), hidden
    s = torch.softmax(v.masked_fill(hidden, -math.inf), -1)
    return torch.where(hidden | hidden.all(-1, keepdim=True), torch.zeros_like(s), s), hidden


def _reference(logits, k, kind, bias, groups, topk_groups, group_top, renorm, scale):
    """(idx, weights, scores) in float64; equal scores by their logits, so that float64's own rounding
    of the scores orders nothing"""
    logits = logits.cpu()
    s, hidden = _scores(logits, kind)
    T, E = s.shape
    by_logit = bias is None and (groups == topk_groups or group_top == 1 or E == groups)
    c = logits.double() if by_logit else s if bias is None else s + bias.cpu().double()
    c = c.masked_fill(hidden, -math.inf)
    keep = torch.ones(T, groups, dtype=torch.bool)
    if groups > topk_groups:
        value = c.view(T, groups, -1).sort(dim=-1, descending=True).values[..., :group_top].sum(-1)
        keep.zero_().scatter_(1, value.sort(dim=-1, descending=True, stable=True).indices[:, :topk_groups], True)
    keep = keep.repeat_interleave(E // groups, 1)
    order = c.sort(dim=-1, descending=True, stable=True).indices
    order = order.gather(1, (~keep.gather(1, order)).to(torch.int8).sort(dim=-1, stable=True).indices)
    idx = order[:, :k]
    w = s.gather(1, idx)
    if renorm:
        total = w.sum(-1, keepdim=True)
        w = torch.where(total == 0, torch.zeros_like(w), w / total)
    return idx, w * scale, s


def _inputs(T, E, dtype, seed, spread=2.0, masked=False):
    gen = torch.Generator().manual_seed(seed)
    l = (torch.randn(T, E, generator=gen) * spread).clamp(-12, 12).to(dtype)
    if masked:
        l[torch.rand(T, E, generator=gen) < 0.3] = -math.inf
        l[0] = -math.inf                              # a token that may use no expert
        l[T // 2] = torch.finfo(dtype).min            # the same by the type's lowest value
        l[T - 1, 1:] = -math.inf                      # one expert only
    return l


def _close(got, want, dtype, extra, mag=None):
    rel, tiny = _half_step(dtype)
    off = (got.cpu().double() - want).abs()
    bound = rel * want.abs() + extra * (want.abs() if mag is None else mag) + tiny + 2.0 ** -126
    assert bool((off <= bound).all()), float((off - bound).max())


CASES = [
    # T, E, k, dtype, score, bias, groups, topk_groups, group_top, renorm, scale, masked
    (1, 8, 2, BF, "softmax", False, 1, 1, 2, False, 1.0, False),
    (1000, 8, 2, BF, "softmax", False, 1, 1, 2, False, 1.0, True),
    (4099, 8, 8, FP, "softmax", False, 1, 1, 2, True, 1.0, False),
    (33, 1, 1, FP, "sigmoid", False, 1, 1, 2, False, 2.0, False),
    (129, 2, 1, HF, "softmax", True, 1, 1, 2, False, 1.0, False),
    (77, 7, 3, HF, "sigmoid", True, 1, 1, 2, True, 2.5, True),
    (300, 16, 4, BF, "sigmoid", True, 4, 2, 2, True, 1.0, True),
    (301, 30, 6, FP, "softmax", False, 5, 2, 2, True, 1.0, False),
    (301, 30, 6, HF, "softmax", False, 5, 2, 1, True, 1.0, True),
    (513, 64, 6, BF, "softmax", False, 1, 1, 2, True, 1.0, True),
    (257, 65, 9, FP, "sigmoid", True, 1, 1, 2, False, 1.0, True),
    (100, 128, 32, BF, "softmax", True, 8, 3, 1, True, 1.0, False),
    (515, 256, 8, FP, "sigmoid", True, 8, 4, 2, True, 2.5, False),
    (515, 256, 8, BF, "sigmoid", True, 8, 4, 2, True, 2.5, True),
    (64, 256, 32, HF, "softmax", False, 256, 100, 2, False, 1.0, False),
    (90, 257, 5, BF, "softmax", True, 1, 1, 2, True, 1.0, False),
    (90, 512, 10, FP, "softmax", True, 16, 5, 2, True, 1.0, True),
    (41, 510, 32, BF, "sigmoid", False, 2, 1, 2, True, 1.0, False),
]


@pytest.mark.parametrize("T,E,k,dtype,score,has_bias,groups,topk_groups,group_top,renorm,scale,masked", CASES)
def test_choice_scores_and_counts(cuda_device, T, E, k, dtype, score, has_bias, groups, topk_groups, group_top, renorm,
                                  scale, masked):
    from baidu_cti_grab_b200 import device_ops

    logits = _inputs(T, E, dtype, 7 * T + E, masked=masked and T > 4)
    bias = 0.1 * torch.randn(E, generator=torch.Generator().manual_seed(E)) if has_bias else None
    idx, w, probs, counts = device_ops.route_topk(
        logits.to(cuda_device), k, score=score, bias=None if bias is None else bias.to(cuda_device), groups=groups,
        topk_groups=topk_groups, group_top=group_top, renormalize=renorm, scale=scale, want_probs=True, want_counts=True)
    want_idx, want_w, want_s = _reference(logits, k, score, bias, groups, topk_groups, group_top, renorm, scale)
    assert torch.equal(idx.cpu(), want_idx)
    assert w.dtype == probs.dtype == dtype
    _close(w, want_w, dtype, 2.0 ** -18)
    _close(probs, want_s, dtype, 2.0 ** -18)
    assert torch.equal(counts.cpu().long(), torch.bincount(want_idx.reshape(-1), minlength=E))


@pytest.mark.parametrize("dtype,E,spacing", [(BF, 64, 0.25), (FP, 256, 0.5), (HF, 8, 1.0), (FP, 500, 2.0)])
@pytest.mark.parametrize("bias", ["none", "zeros", "steps"])
def test_ties_go_to_the_lowest_index(cuda_device, dtype, E, spacing, bias):
    """Logits on a coarse grid and biases of few values: most choices are ties."""
    from baidu_cti_grab_b200 import device_ops

    gen = torch.Generator().manual_seed(E)
    logits = (torch.randn(400, E, generator=gen) / spacing).round().mul(spacing).to(dtype)
    logits[3] = 0.0
    logits[4] = -0.0
    logits[4, ::2] = 0.0
    b = {"none": None, "zeros": torch.zeros(E), "steps": torch.randint(-1, 2, (E,), generator=gen) * 0.125}[bias]
    for groups, keep in ((1, 1), (4, 2)):
        k = min(6, E // groups * keep)
        idx, _, _, _ = device_ops.route_topk(logits.to(cuda_device), k, bias=None if b is None else b.to(cuda_device),
                                             groups=groups, topk_groups=keep, group_top=1)
        assert torch.equal(idx.cpu(), _reference(logits, k, "softmax", b, groups, keep, 1, False, 1.0)[0])


def test_neighbours_below_fp32_resolution(cuda_device):
    """Choice values that fp32 cannot tell apart: sigmoids of logits one unit apart, and biases that
    undo the scores' differences to within an fp32 unit."""
    from baidu_cti_grab_b200 import device_ops

    gen = torch.Generator().manual_seed(5)
    base = torch.randn(600, 1, generator=gen)
    logits = (base + torch.randint(-3, 4, (600, 96), generator=gen) * 2.0 ** -24).float()
    bias = torch.randint(-1, 2, (96,), generator=gen) * 2.0 ** -25
    idx, _, _, _ = device_ops.route_topk(logits.to(cuda_device), 7, score="sigmoid", bias=bias.to(cuda_device))
    assert torch.equal(idx.cpu(), _reference(logits, 7, "sigmoid", bias, 1, 1, 1, False, 1.0)[0])
    s = torch.softmax(torch.randn(96, generator=gen).double(), -1)
    undo = (0.5 - s).float()                       # s + bias is 0.5 to within half a unit
    logits = s.log().float().repeat(5, 1)
    idx, _, _, _ = device_ops.route_topk(logits.to(cuda_device), 7, bias=undo.to(cuda_device), groups=8, topk_groups=3)
    assert torch.equal(idx.cpu(), _reference(logits, 7, "softmax", undo, 8, 3, 2, False, 1.0)[0])


def test_nan_infinity_and_masks_stay_in_their_rows(cuda_device):
    from baidu_cti_grab_b200 import device_ops

    logits = _inputs(70, 40, FP, 3)
    clean = device_ops.route_topk(logits.to(cuda_device), 4, want_probs=True)
    bad = logits.clone()
    bad[10, 5] = math.nan
    bad[11, 6] = math.inf
    bad[12] = math.nan
    bad[13] = -math.inf
    idx, w, probs, _ = device_ops.route_topk(bad.to(cuda_device), 4, want_probs=True)
    rows = [i for i in range(70) if i not in (10, 11, 12, 13)]
    for a, b in zip((idx, w, probs), clean):
        assert torch.equal(a[rows], b[rows])
    assert idx[10, 0] == 5 and idx[11, 0] == 6  # a NaN is above every number
    assert idx[12].tolist() == [0, 1, 2, 3] and bool(w[12].isnan().all())
    assert idx[13].tolist() == [0, 1, 2, 3] and bool((w[13] == 0).all()) and bool((probs[13] == 0).all())
    assert int(idx.min()) >= 0 and int(idx.max()) < 40


def test_sigmoids_of_very_negative_logits_keep_their_ratios(cuda_device):
    """Scores near fp32's smallest numbers: e^-85 is normal (1.2e-37), e^-95 subnormal (5.5e-42, in steps of 2^-149);
    renormalised weights of the former are as exact as any."""
    from baidu_cti_grab_b200 import device_ops

    logits = (-85.0 - torch.rand(64, 24, generator=torch.Generator().manual_seed(1))).float()
    idx, w, _, _ = device_ops.route_topk(logits.to(cuda_device), 4, score="sigmoid", renormalize=True)
    want_idx, want_w, _ = _reference(logits, 4, "sigmoid", None, 1, 1, 2, True, 1.0)
    assert torch.equal(idx.cpu(), want_idx)
    _close(w, want_w, FP, 2.0 ** -18)
    low = (logits - 10.0).to(cuda_device)
    _, _, probs, _ = device_ops.route_topk(low, 4, score="sigmoid", want_probs=True)
    assert bool(((probs.cpu().double() - torch.sigmoid(logits.double() - 10.0)).abs() <= 2.0 ** -148).all())


def test_strides_types_and_no_tokens(cuda_device):
    from baidu_cti_grab_b200 import device_ops

    wide = _inputs(50, 300, BF, 9).to(cuda_device)
    for view in (wide[:, 3:67], wide[:, 8:72], wide[::3, :64], wide.t()[:64], wide[:1, :64].expand(9, 64)):
        a = device_ops.route_topk(view, 3, want_probs=True, idx_dtype=torch.int32, score_dtype=FP)
        b = device_ops.route_topk(view.contiguous().float(), 3, want_probs=True)
        assert a[0].dtype == torch.int32 and a[1].dtype == a[2].dtype == FP
        assert torch.equal(a[0].long(), b[0])
        for x, y in zip(a[1:3], b[1:3]):  # each within 2^-18 of the definition; the order of the sum goes by the layout
            assert bool(((x - y).abs() <= 2.0 ** -17 * y).all())
    none = device_ops.route_topk(wide[:0, :64], 3, want_probs=True, want_counts=True)
    assert none[0].shape == (0, 3) and none[2].shape == (0, 64) and bool((none[3] == 0).all())
    assert device_ops.route_topk_backward(wide[:0, :64], none[0], none[1]).shape == (0, 64)


GRADS = [(1, 8, 2, BF, "softmax", False, True), (777, 8, 2, FP, "softmax", True, True),
         (130, 64, 6, BF, "softmax", True, True), (130, 65, 6, HF, "softmax", True, False),
         (99, 256, 8, FP, "sigmoid", True, True), (99, 300, 32, BF, "sigmoid", False, False),
         (64, 33, 1, FP, "softmax", True, True)]


@pytest.mark.parametrize("T,E,k,dtype,score,renorm,with_probs", GRADS)
def test_gradient_against_the_formula_and_differences(cuda_device, T, E, k, dtype, score, renorm, with_probs):
    from baidu_cti_grab_b200 import device_ops

    logits = _inputs(T, E, dtype, T + E, masked=T > 4)
    gen = torch.Generator().manual_seed(1)
    gs, gp = torch.randn(T, k, generator=gen).to(dtype), (0.1 * torch.randn(T, E, generator=gen)).to(dtype)
    idx = _reference(logits, k, score, None, 1, 1, 1, renorm, 2.0)[0]

    def loss(l64):
        hidden = logits <= torch.finfo(dtype).min
        if score == "sigmoid":
            s = torch.sigmoid(l64).masked_fill(hidden, 0.0)
        else:
            e = torch.exp(l64.masked_fill(hidden, 0.0)).masked_fill(hidden, 0.0)
            total = e.sum(-1, keepdim=True)
            s = e / torch.where(total == 0, torch.ones_like(total), total)
        w = s.gather(1, idx)
        if renorm:
            total = w.sum(-1, keepdim=True)
            w = w / torch.where(total == 0, torch.ones_like(total), total)
        out = 2.0 * (w * gs.double()).sum()
        return out + (s * gp.double()).sum() if with_probs else out

    l64 = logits.double().clamp_min(-1e4).requires_grad_()
    want, = torch.autograd.grad(loss(l64), l64)
    dev = [t.to(cuda_device) for t in (logits, idx, gs, gp)]
    for i in (dev[1], dev[1].int()):
        got = device_ops.route_topk_backward(dev[0], i, dev[2], dev[3] if with_probs else None, score=score,
                                             renormalize=renorm, scale=2.0)
        s, _ = _scores(logits, score)
        total = s.gather(1, idx).sum(-1, keepdim=True).clamp_min(1e-30) if renorm else torch.ones(T, 1)
        g = torch.zeros_like(s).scatter_(1, idx, 2.0 * gs.double().abs())
        ds = g / total
        if renorm:
            ds = ds + torch.zeros_like(s).scatter_(1, idx, 1.0) * (g * s).sum(-1, keepdim=True) / total ** 2
        if with_probs:
            ds = ds + gp.double().abs()
        mag = s * ds if score == "sigmoid" else s * (ds + (ds * s).sum(-1, keepdim=True))
        _close(got, want, dtype, 2.0 ** -16, mag)
        assert bool((got.cpu()[(logits <= torch.finfo(dtype).min)] == 0).all())
    # central differences of the definition along random directions: h^2 |f'''| / 6 is under 1e-7 of the terms' sizes
    for seed in range(3):
        v = torch.randn(T, E, generator=torch.Generator().manual_seed(seed)).double()
        with torch.no_grad():
            slope = (loss(l64 + 1e-4 * v) - loss(l64 - 1e-4 * v)) / 2e-4
        rel, tiny = _half_step(dtype)
        bound = float(((rel * want.abs() + 2.0 ** -16 * mag + tiny) * v.abs()).sum() + 1e-6 * (mag * v.abs()).sum() + 1e-9)
        assert abs(float((got.cpu().double() * v).sum()) - float(slope)) <= bound


def test_autograd_and_router_module(cuda_device):
    from baidu_cti_grab_b200 import device_ops, routing

    logits = _inputs(65, 12, FP, 2).to(cuda_device).requires_grad_()
    r = routing.route_topk(logits, 3, renormalize=True, want_probs=True, want_counts=True)
    (r.score.square().sum() + (r.probs * 0.3).sum()).backward()
    want = device_ops.route_topk_backward(logits.detach(), r.idx, 2 * r.score.detach(), torch.full_like(r.probs, 0.3),
                                          renormalize=True)
    assert torch.equal(logits.grad, want)
    assert not r.idx.requires_grad and not r.counts.requires_grad
    logits.grad = None
    routing.route_topk(logits, 3).score.sum().backward()  # probs not asked for
    assert logits.grad is not None
    gate = routing.TopKRouter(64, 12, 2, score="sigmoid", renormalize=True, balanced=True).to(cuda_device, BF)
    assert gate.balance_bias.dtype == FP and gate.balance_bias.device.type == "cuda"
    x = torch.randn(3, 20, 64, device=cuda_device).to(BF)
    idx, score, probs = gate(x)
    assert idx.shape == (3, 20, 2) and score.shape == (3, 20, 2) and probs.shape == (3, 20, 12)
    counts = gate.route(x, want_counts=True).counts
    gate.update_balance(counts, 0.5)
    assert torch.equal(gate.balance_bias.cpu(), 0.5 * torch.sign(10.0 - counts.cpu().float()))
    score.float().sum().backward()
    assert gate.w_g.weight.grad is not None


def test_streams_graphs_and_repeats(cuda_device):
    from baidu_cti_grab_b200 import device_ops

    logits = _inputs(2000, 96, BF, 4).to(cuda_device)
    bias = torch.zeros(96, device=cuda_device)
    want = device_ops.route_topk(logits, 4, bias=bias, want_counts=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = device_ops.route_topk(logits, 4, bias=bias, want_counts=True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = device_ops.route_topk(logits, 4, bias=bias, want_counts=True)
        grad = device_ops.route_topk_backward(logits, held[0], held[1])
    for _ in range(2):
        graph.replay()
        for a, b, c in zip(want, other, held):
            assert a is None or (torch.equal(a, b) and torch.equal(a, c))
    assert torch.equal(grad, device_ops.route_topk_backward(logits, want[0], want[1]))
    fresh = _inputs(2000, 96, BF, 5).to(cuda_device)
    logits.copy_(fresh)
    graph.replay()
    now = device_ops.route_topk(fresh, 4, bias=bias, want_counts=True)
    assert torch.equal(held[0], now[0]) and torch.equal(held[3], now[3])


@pytest.mark.parametrize("lead", [(0,), (0, 5), (3, 0)])
def test_empty_batch_through_the_router(cuda_device, lead):
    from baidu_cti_grab_b200 import routing

    gate = routing.TopKRouter(16, 8, 2, renormalize=True).to(cuda_device)
    x = torch.zeros(*lead, 16, device=cuda_device, requires_grad=True)
    idx, score, probs = gate(x)
    assert idx.shape == score.shape == (*lead, 2) and probs.shape == (*lead, 8)
    (score.sum() + probs.sum()).backward()
    assert x.grad.shape == x.shape and bool((gate.w_g.weight.grad == 0).all())


@pytest.mark.parametrize("E", [8, 100, 300])
def test_gradients_of_saturated_sigmoids(cuda_device, E):
    """s (1 - s) of logits from -60 to 60: exp within 2 units of 2^-23, the sum, quotient, difference and products half a unit or
    (the quotient) two each: under 2^-20 of the value, not of s."""
    from baidu_cti_grab_b200 import device_ops

    gen = torch.Generator().manual_seed(E)
    logits = (torch.rand(70, E, generator=gen) - 0.5) * 120
    logits[0, :4] = torch.tensor([0.0, 17.5, 40.0, -40.0])
    gp = torch.randn(70, E, generator=gen)
    idx = torch.zeros(70, 1, dtype=torch.int64)
    grad = device_ops.route_topk_backward(logits.to(cuda_device), idx.to(cuda_device), None, gp.to(cuda_device), score="sigmoid")
    l = logits.double()
    want = gp.double() / (1.0 + torch.exp(-l)) / (1.0 + torch.exp(l))
    assert bool(((grad.cpu().double() - want).abs() <= (2.0 ** -20 + 2.0 ** -24) * want.abs()).all())
