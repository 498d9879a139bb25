"""The seam between two blocks (rb_sandwich_norm and its backward, block_norm.py) on the GPU against
the definition and its gradients in float64.

Tolerances, u = 2^-24.  A row's mean and sum of squares are sums of at most 32 values a thread and up to
nine pairwise steps: 41 u of the sum of magnitudes, so a normalised value v^ is off by at most
48 u (1 + |v^|) (the mean's error against the deviation, half the square sum's, rsqrtf 2 u); weight, bias,
gate and residual add under 16 u: y is within 2^-18 of M = |x| + |s a| (|w| (1 + |v^|) + |b|).  z takes y's error over
its deviation and the same again: 2^-17 of |w| (1 + |y^| + M / dev) + |b|.  A gradient of a norm is r (d w - mean - v^ mean(d w
v^)), whose means are at most rms(d w): with v^ off as above it is within 2^-14 of
r (|d w| + 2 (1 + |v^|) rms(d w)) and, through the second norm, 2^-13.  Sums over rows: 2^-13 of
the summed magnitudes (their own additions, under 2^10 u for these rows, included).  Every output
is rounded once: half a step of its type on top.
"""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
NAMES = ("x", "h", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias")


def _half_step(dtype):
    fi = torch.finfo(dtype)
    return fi.eps / 2, fi.smallest_normal * fi.eps / 2 + 2.0 ** -120


def _inputs(N, D, dtype, wdtype, post, pre, gate, seed, affine=True):
    gen = torch.Generator().manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0, to=dtype):
        return (torch.randn(*shape, generator=gen) * std + mean).to(to)

    t = dict(x=normal(N, D, std=2.0), h=normal(N, D, std=0.7, mean=0.1))
    for name, kind in (("post", post), ("pre", pre)):
        t[name + "_weight"] = normal(D, std=0.2, mean=1.0, to=wdtype) if kind and affine else None
        t[name + "_bias"] = normal(D, std=0.1, to=wdtype) if kind == "layer" and affine else None
    shape = {"channel": (D,), "row": (N, 1), "full": (N, D), None: None}[gate]
    t["gate"] = normal(*shape, std=0.6, mean=0.3, to=wdtype if gate == "channel" else dtype) if shape else None
    return t, normal(N, D), normal(N, D) if pre else None


def _norm64(v, kind, w, b, eps):
    if kind is None:
        return v, torch.zeros_like(v), torch.ones_like(v[..., :1])
    c = v - v.mean(-1, keepdim=True) if kind == "layer" else v
    r = 1.0 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    out = c * r if w is None else c * r * w
    return (out if b is None else out + b), c * r, r


def _forward64(t, post, pre, act, scale, eps=1e-5):
    n, hh, rh = _norm64(t["h"], post, t["post_weight"], t["post_bias"], eps)
    g = t["gate"]
    a = torch.ones((), dtype=torch.float64) if g is None else torch.sigmoid(g) if act == "sigmoid" else g
    y = t["x"] + scale * a * n
    z, yh, ry = _norm64(y, pre, t["pre_weight"], t["pre_bias"], eps)
    return y, z, n, a, hh, rh, yh, ry


def _abs(w, like):
    return torch.ones_like(like) if w is None else w.abs()


def _check(got, want, dtype, bound, name):
    rel, tiny = _half_step(dtype)
    off = (got.cpu().double() - want).abs()
    limit = rel * want.abs() + bound + tiny
    assert bool((off <= limit).all()), (name, float((off - limit).max()), float(off.max()))


def _to(t, dev):
    return {k: None if v is None else v.to(dev) for k, v in t.items()}


CASES = [
    # N, D, dtype, weights, post, pre, gate, act, scale
    (1, 512, BF, BF, "layer", "layer", "channel", "none", 1.0),
    (1, 1, FP, FP, "layer", "rms", "row", "sigmoid", 0.5),
    (5, 7, HF, FP, "rms", "layer", "full", "sigmoid", 1.0),
    (9, 8, BF, FP, None, "layer", None, "none", 1.0),
    (33, 33, BF, BF, "layer", "layer", "row", "none", 2.0),
    (700, 256, HF, HF, "layer", None, "channel", "sigmoid", 0.5),
    (2500, 512, BF, BF, "layer", "layer", "channel", "none", 1.0),
    (1301, 512, HF, HF, "layer", "layer", "full", "sigmoid", 0.5),
    (77, 520, FP, FP, "rms", "rms", "full", "none", 1.0),
    (300, 1000, BF, FP, "layer", "rms", "channel", "none", 0.7),
    (300, 1023, HF, HF, "layer", "layer", "full", "none", 0.7),
    (129, 1032, BF, BF, "layer", "layer", "row", "sigmoid", 1.0),
    (401, 2048, BF, BF, None, None, "full", "sigmoid", 1.0),
    (65, 2056, FP, FP, "layer", "layer", "channel", "none", 1.0),
    (400, 4097, BF, FP, "rms", "layer", "channel", "sigmoid", 1.0),
    (310, 5000, BF, FP, "rms", "rms", "row", "none", 0.7),
    (20, 8191, HF, HF, "layer", "layer", "full", "none", 1.0),
    (170, 5120, BF, BF, "layer", "layer", "full", "sigmoid", 1.0),   # the widest with constants in registers
    (170, 5128, BF, BF, "layer", "layer", "channel", "none", 1.0),   # in shared memory
    (33, 6144, BF, FP, "rms", "rms", None, "none", 1.0),
    (33, 7200, FP, FP, "layer", "layer", "full", "none", 1.0),       # the widest fp32 of those
    (33, 7208, FP, FP, "rms", "layer", "full", "none", 1.0),         # made for each row
    (160, 8192, FP, FP, "layer", "layer", "full", "sigmoid", 1.0),
]


@pytest.mark.parametrize("N,D,dtype,wdtype,post,pre,gate,act,scale", CASES)
def test_forward_and_gradients_against_float64(cuda_device, N, D, dtype, wdtype, post, pre, gate, act, scale):
    from baidu_cti_grab_b200 import device_ops

    t, gy, gz = _inputs(N, D, dtype, wdtype, post, pre, gate, N + D)
    dev = _to(t, cuda_device)
    how = dict(post=post, pre=pre, gate_act=act, scale=scale)
    kw = {k: v for k, v in dev.items() if k not in ("x", "h")}
    y, z, stats = device_ops.sandwich_norm(dev["x"], dev["h"], want_stats=True, **kw, **how)
    t64 = {k: None if v is None else v.double().requires_grad_() for k, v in t.items()}
    y64, z64, n, a, hh, rh, yh, ry = _forward64(t64, post, pre, act, scale)
    loss = (y64 * gy.double()).sum() + ((z64 * gz.double()).sum() if pre else 0.0)
    used = [k for k in NAMES if t64[k] is not None]
    want = dict(zip(used, torch.autograd.grad(loss, [t64[k] for k in used])))
    with torch.no_grad():
        w1, b1 = _abs(t64["post_weight"], n), 0.0 if t64["post_bias"] is None else t64["post_bias"].abs()
        w2, b2 = _abs(t64["pre_weight"], n), 0.0 if t64["pre_bias"] is None else t64["pre_bias"].abs()
        nmag = w1 * (1 + hh.abs()) + b1 if post else n.abs()
        M = t64["x"].abs() + (scale * a).abs() * nmag
        _check(y, y64, dtype, 2.0 ** -18 * M, "y")
        mt = gy.double().abs()
        if pre:
            _check(z, z64, dtype, 2.0 ** -17 * (w2 * (1 + yh.abs() + M * ry) + b2), "z")
            u = gz.double().abs() * w2
            mt = mt + ry * (u + 2 * (1 + yh.abs() + M * ry) * u.square().mean(-1, keepdim=True).sqrt())
        got = dict(zip(NAMES, device_ops.sandwich_norm_backward(gy.to(cuda_device), None if gz is None else gz.to(cuda_device),
                                                                dev["x"], dev["h"], stats, **kw, **how)))
        _check(got["x"], want["x"], dtype, 2.0 ** -14 * mt, "dx")
        dn = (scale * a).abs() * mt
        mh = dn
        if post:
            v = w1 * dn
            mh = rh * (v + 2 * (1 + hh.abs()) * v.square().mean(-1, keepdim=True).sqrt())
        _check(got["h"], want["h"], dtype, 2.0 ** -13 * mh, "dh")
        if gate:
            mg = abs(scale) * nmag * mt
            mg = {"channel": mg.sum(0), "row": mg.sum(-1, keepdim=True), "full": mg}[gate]
            _check(got["gate"], want["gate"], t["gate"].dtype, 2.0 ** -13 * mg, "dgate")
        sums = dict(post_weight=dn * (1 + hh.abs()), post_bias=dn)
        if pre:
            sums.update(pre_weight=gz.double().abs() * (1 + yh.abs() + M * ry), pre_bias=gz.double().abs())
        for k, m in sums.items():
            if t[k] is not None:
                _check(got[k], want[k], wdtype, 2.0 ** -13 * m.sum(0), k)
            else:
                assert got[k] is None
    again = device_ops.sandwich_norm_backward(gy.to(cuda_device), None if gz is None else gz.to(cuda_device), dev["x"], dev["h"],
                                              stats, **kw, **how)
    for k, v in zip(NAMES, again):
        assert v is None or torch.equal(v, got[k])


@pytest.mark.parametrize("post,pre,gate,act", [("layer", "layer", "channel", "sigmoid"), ("rms", "rms", "full", "none"),
                                               ("layer", "rms", "row", "sigmoid")])
def test_gradients_against_differences(cuda_device, post, pre, gate, act):
    """Directional derivatives of the float64 definition by central differences (their h^2 error under 1e-6 of
    the terms) against the kernel's gradients in fp32 (each within 2^-13 of its magnitude, under 2^-9 of the sum)."""
    from baidu_cti_grab_b200 import device_ops

    t, gy, gz = _inputs(6, 40, FP, FP, post, pre, gate, 3)
    dev = _to(t, cuda_device)
    kw = {k: v for k, v in dev.items() if k not in ("x", "h")}
    how = dict(post=post, pre=pre, gate_act=act, scale=0.8)
    _, _, stats = device_ops.sandwich_norm(dev["x"], dev["h"], want_stats=True, **kw, **how)
    grads = device_ops.sandwich_norm_backward(gy.to(cuda_device), gz.to(cuda_device), dev["x"], dev["h"], stats, **kw, **how)

    def loss(t64):
        y, z, *_ = _forward64(t64, post, pre, act, 0.8)
        return float((y * gy.double()).sum() + (z * gz.double()).sum())

    t64 = {k: None if v is None else v.double() for k, v in t.items()}
    for name, grad in zip(NAMES, grads):
        if grad is None:
            continue
        for seed in range(2):
            v = torch.randn(t[name].shape, generator=torch.Generator().manual_seed(seed)).double()
            up, down = dict(t64), dict(t64)
            up[name], down[name] = t64[name] + 1e-5 * v, t64[name] - 1e-5 * v
            slope = (loss(up) - loss(down)) / 2e-5
            terms = grad.cpu().double() * v
            assert abs(float(terms.sum()) - slope) <= 2.0 ** -9 * float(terms.abs().sum()) + 1e-6, name


def test_strided_and_unaligned_rows_and_leading_dims(cuda_device):
    """Rows that bulk copies cannot fetch give the same bits."""
    from baidu_cti_grab_b200 import device_ops

    t, gy, gz = _inputs(60, 512, BF, BF, "layer", "layer", "full", 8)
    dev = _to(t, cuda_device)
    kw = {k: v for k, v in dev.items() if k not in ("x", "h")}
    how = dict(post="layer", pre="layer", gate_act="sigmoid", scale=0.5)
    want = device_ops.sandwich_norm(dev["x"], dev["h"], want_stats=True, **kw, **how)
    grads = device_ops.sandwich_norm_backward(gy.to(cuda_device), gz.to(cuda_device), dev["x"], dev["h"], want[2], **kw, **how)

    def odd(v, ld, off):
        room = torch.full((61 * ld + off,), float("nan"), dtype=v.dtype, device=cuda_device)
        view = room[off:off + 60 * ld].view(60, ld)[:, :512]
        view.copy_(v)
        return view

    for ld, off in ((512, 1), (515, 0), (640, 0), (1024, 8)):
        x, h, g = odd(t["x"], ld, off), odd(t["h"], ld, off), odd(t["gate"], ld, off)
        kw2 = dict(kw, gate=g)
        got = device_ops.sandwich_norm(x, h, want_stats=True, **kw2, **how)
        for p, q in zip(got, want):
            assert torch.equal(p, q)
        back = device_ops.sandwich_norm_backward(odd(gy, ld, off), odd(gz, ld, off), x, h, got[2], **kw2, **how)
        for p, q in zip(back, grads):
            assert torch.equal(p, q)
    lead = {k: v.view(3, 20, 512) for k, v in dict(x=dev["x"], h=dev["h"], gate=dev["gate"]).items()}
    y, z, _ = device_ops.sandwich_norm(lead["x"], lead["h"], **dict(kw, gate=lead["gate"]), **how)
    assert torch.equal(y.view(60, 512), want[0]) and torch.equal(z.view(60, 512), want[1])
    same = dev["x"][:1].expand(4, 512)  # one row read four times
    y4, _, _ = device_ops.sandwich_norm(same, same, post="rms")
    y1, _, _ = device_ops.sandwich_norm(dev["x"][:1], dev["x"][:1], post="rms")
    assert torch.equal(y4, y1.expand(4, 512))


def test_gradients_that_are_not_there_and_no_rows(cuda_device):
    from baidu_cti_grab_b200 import device_ops

    t, gy, gz = _inputs(50, 96, FP, FP, "layer", "layer", "channel", 4)
    dev = _to(t, cuda_device)
    kw = {k: v for k, v in dev.items() if k not in ("x", "h")}
    how = dict(post="layer", pre="layer", scale=1.0)
    gy, gz = gy.to(cuda_device), gz.to(cuda_device)
    _, _, stats = device_ops.sandwich_norm(dev["x"], dev["h"], want_stats=True, **kw, **how)
    zero = torch.zeros_like(gy)
    run = lambda a, b: device_ops.sandwich_norm_backward(a, b, dev["x"], dev["h"], stats, **kw, **how)  # noqa: E731
    for p, q in zip(run(None, gz), run(zero, gz)):
        assert torch.equal(p, q)
    for p, q in zip(run(gy, None), run(gy, zero)):
        assert torch.equal(p, q)
    assert torch.equal(run(gy, None)[0], gy)
    empty = {k: (v[:0] if k in ("x", "h") else v) for k, v in dev.items()}
    y, z, s = device_ops.sandwich_norm(empty["x"], empty["h"], want_stats=True, **kw, **how)
    assert y.shape == z.shape == (0, 96) and s.shape == (0, 4)
    grads = device_ops.sandwich_norm_backward(y, z, empty["x"], empty["h"], s, **kw, **how)
    assert grads[0].shape == (0, 96) and all(bool((v == 0).all()) for v in grads[2:])


def test_constant_rows_and_nan_stay_in_their_rows(cuda_device):
    from baidu_cti_grab_b200 import device_ops

    t, gy, gz = _inputs(40, 512, FP, FP, "layer", "layer", "row", 6)
    t["h"][7] = 3.0
    t["x"][7] = -1.0
    dev = _to(t, cuda_device)
    kw = {k: v for k, v in dev.items() if k not in ("x", "h")}
    how = dict(post="layer", pre="layer", scale=1.0)
    gy, gz = gy.to(cuda_device), gz.to(cuda_device)

    def run(h):
        y, z, s = device_ops.sandwich_norm(dev["x"], h, want_stats=True, **kw, **how)
        return (y, z, *device_ops.sandwich_norm_backward(gy, gz, dev["x"], h, s, **kw, **how)[:3])

    clean = run(dev["h"])
    assert all(bool(v.isfinite().all()) for v in clean)
    bad = dev["h"].clone()
    bad[11, 100], bad[12, 3] = float("nan"), float("inf")
    rows = [i for i in range(40) if i not in (11, 12)]
    for p, q in zip(run(bad), clean):
        assert torch.equal(p[rows], q[rows])
        assert bool(p[11].isnan().any()) and not bool(p[12].isfinite().all())


def test_autograd_module_streams_and_graphs(cuda_device):
    from baidu_cti_grab_b200 import block_norm, device_ops

    m = block_norm.SandwichNorm(128, post="rms", pre="layer", scale=0.5, channel_gate=True, gate_act="sigmoid").to(cuda_device)
    x = torch.randn(70, 128, device=cuda_device, requires_grad=True)
    h = torch.randn(70, 128, device=cuda_device, requires_grad=True)
    y, z = m(x, h)
    (y.sum() + z.square().sum()).backward()
    assert all(p.grad is not None for p in m.parameters()) and x.grad is not None and h.grad is not None
    how = dict(post="rms", pre="layer", scale=0.5, gate_act="sigmoid")
    kw = dict(gate=m.gate.detach(), post_weight=m.post_weight.detach(), pre_weight=m.pre_weight.detach(),
              pre_bias=m.pre_bias.detach())
    _, z0, stats = device_ops.sandwich_norm(x.detach(), h.detach(), want_stats=True, **kw, **how)
    run = lambda: device_ops.sandwich_norm_backward(torch.ones_like(z0), 2 * z0, x.detach(), h.detach(), stats, **kw, **how)  # noqa: E731
    want = run()
    for p, q in zip((x.grad, h.grad, m.gate.grad, m.post_weight.grad, None, m.pre_weight.grad, m.pre_bias.grad), want):
        assert q is None or torch.equal(p, q)
    m(x, h)[0].sum().backward()  # z not used
    with torch.no_grad():
        assert not m(x, h)[1].requires_grad
    with pytest.raises(ValueError):
        m(x, h, gate=torch.ones(128, device=cuda_device))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    torch.cuda.current_stream().wait_stream(side)
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    with torch.cuda.graph(graph2):
        held2 = run()
    for _ in range(2):
        graph.replay()
        graph2.replay()
        for p, q, s, e in zip(want, other, held, held2):
            assert p is None or (torch.equal(p, q) and torch.equal(p, s) and torch.equal(p, e))
    assert device_ops.device_error() == 0


AFFINE = ("post_weight", "post_bias", "pre_weight", "pre_bias")


@pytest.mark.parametrize("absent", [AFFINE[:1], AFFINE[1:2], AFFINE[2:3], AFFINE[3:], (AFFINE[0], AFFINE[2]), AFFINE],
                         ids="+".join)
@pytest.mark.parametrize("D,dtype", [(7, HF), (100, BF), (512, HF), (520, BF), (768, FP), (1023, HF), (5000, BF), (5121, FP),
                                     (5128, BF), (7208, FP)])
@pytest.mark.parametrize("gate,act", [("row", "none"), ("channel", "sigmoid"), ("full", "sigmoid"), (None, "none")])
def test_without_weights_or_biases(cuda_device, monkeypatch, D, dtype, gate, act, absent):
    """Each of the norms' weights and biases left out, on widths that fill their team of threads and that do not."""
    whole = _inputs

    def fewer(*args):
        t, gy, gz = whole(*args)
        t.update(dict.fromkeys(absent))
        return t, gy, gz

    monkeypatch.setitem(globals(), "_inputs", fewer)
    test_forward_and_gradients_against_float64(cuda_device, 37, D, dtype, dtype, "layer", "layer", gate, act, 0.7)
    if gate is None:
        test_forward_and_gradients_against_float64(cuda_device, 37, D, dtype, dtype, "rms", "layer", gate, act, 0.7)
        test_forward_and_gradients_against_float64(cuda_device, 37, D, dtype, dtype, "layer", "rms", gate, act, 0.7)


@pytest.mark.parametrize("gate,dtype", [("full", FP), ("row", FP), ("row", BF), ("channel", FP), ("channel", HF)])
def test_saturated_sigmoid_gates(cuda_device, gate, dtype):
    """Gates of -60 to 60 in fp32: the sigmoid and its derivative keep their own precision where they are small (y = a h without a
    residual or norms; one element of h is not 0 in each sum).  exp's argument is exact, exp within 2 units of 2^-23, the sum,
    quotient and up to four products half a unit each: under 2^-20 of the value.  16-bit rows are gated by the fast exponential,
    off by 2 + 1.2 |g| units of 2^-23, 74 at 60: under 2^-16.  y and dh take half a step of the rows' type on top."""
    from baidu_cti_grab_b200 import device_ops

    N, D = (200, 40) if gate != "channel" else (40, 200)
    gen = torch.Generator().manual_seed(5)
    g = (torch.rand(N, D, generator=gen) - 0.5) * 120
    one = torch.zeros(N, D)
    one[torch.arange(N), torch.arange(N) % D] = 1.0
    if gate == "channel":
        one = torch.zeros(N, D)
        one[torch.arange(D) % N, torch.arange(D)] = 1.0
    g = {"full": g, "row": g[:, :1].contiguous(), "channel": g[0].contiguous()}[gate]
    g.view(-1)[:5] = torch.tensor([0.0, -0.0, 20.0, -20.0, 60.0])
    h = (torch.randn(N, D, generator=gen) * (1.0 if gate == "full" else one)).to(dtype)
    gy = torch.randn(N, D, generator=gen).to(dtype)
    x = torch.zeros(N, D, dtype=dtype)
    a = 1.0 / (1.0 + torch.exp(-g.double()))
    d = a * (1.0 / (1.0 + torch.exp(g.double())))
    dev = {k: v.to(cuda_device) for k, v in dict(x=x, h=h, gate=g, gy=gy).items()}
    y, _, stats = device_ops.sandwich_norm(dev["x"], dev["h"], gate=dev["gate"], gate_act="sigmoid", want_stats=True)
    _, dh, dg, *_ = device_ops.sandwich_norm_backward(dev["gy"], None, dev["x"], dev["h"], stats, gate=dev["gate"],
                                                      gate_act="sigmoid")
    rows = 2.0 ** -20 if dtype == FP else 2.0 ** -16
    _check(y, a * h.double(), dtype, rows * (a * h.double()).abs(), "y")
    _check(dh, a * gy.double(), dtype, rows * (a * gy.double()).abs(), "dh")
    want = d * h.double() * gy.double()
    want = {"full": want, "row": want.sum(-1, keepdim=True), "channel": want.sum(0)}[gate]
    _check(dg, want, FP, 2.0 ** -20 * want.abs(), "dgate")
