"""Attention within packed segments (rb_segment_attention and its backward, attention.py) on the GPU against the
definition in float64.

Tolerance.  u = 2^-24, half = eps / 2 of the model type.
* A score is D products summed in fp32: off by at most 2 D u of scale sum |q| |k| (the factor 2: the tensor cores' adds may
  truncate).  tanh is 1 - 2 / (1 + e^2x) from approximations good to 2 u in e^2x and 1 u in the quotient: off by 4 u, so
  the capped score by 4 u cap.  Scaling, shifting and the distance add 4 u of the largest |score| and bias.  Together `ds`,
  and a weight is off by a factor within exp(2 ds) (its own score and the sum's) times 1 + 8 u.  `eta` is that, less 1.
* On the tensor cores a weight is rounded to the type before it meets v: half of itself, at least 2^-25 in fp16, of
  weights whose largest is 1 to 256.
  So out is within sum p |v| (half + eta) + 2^-25 sum |v| and, rounded once, half of itself.
* exp2's approximation has no subnormals: a weight under 2^-126 is 0, so every weight is off by up to that besides.
* delta = g . out takes out's error; dp is off by 2 D u of sum |g| |v|; e = p (dp - delta) slant is off by (half + eta + 8 u)
  of itself and p slant times these two (the slant 1 - tanh^2 by 8 u).  In fp16 an e below the type's normal range loses
  2^-25 of 2^15 / (2 max |g| max |v|), and p likewise 2^-25 of 2^15.
  dq, dk and dv are those errors times |k|, |q| and |g|, summed, plus n u for a sum of n terms, and half of themselves.
* `near`: rows of few keys have delta as the sum of p dp, off by (eta + n u) of sum p |dp| and 2 D u of sum p |g| |v|; and e
  is carried as two values of the type, off by half of half of itself, in fp16 by twice 2^-25.
"""

import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
U = 2.0 ** -24


def oracle(q, k, v, nq, nk, first=0, k_first=0, g=None, causal=True, prefix=None, slopes=None, cap=0.0, scale=None, half=0.0,
           fp16=False, near=False):
    """(values, bounds) by name in float64, from inputs of any type."""
    (Tq, H, D), (Tk, Hk, _) = q.shape, k.shape
    scale = D ** -0.5 if scale is None else scale
    G = H // Hk
    val = dict(out=torch.zeros(Tq, H, D, dtype=torch.float64, device=q.device),
               lse=torch.full((H, Tq), -math.inf, dtype=torch.float64, device=q.device))
    val.update(dq=torch.zeros_like(val["out"]), dk=torch.zeros(Tk, Hk, D, dtype=torch.float64, device=q.device))
    val["dv"] = torch.zeros_like(val["dk"])
    tol = {n: torch.zeros_like(t) for n, t in val.items()}
    tiny, flushed = (2.0 ** -25 if fp16 else 0.0), 2.0 ** -126
    peak = 1.0
    if g is not None and g.numel() and v.numel():
        peak = 2.0 * max(1e-30, float(g.double().nan_to_num(0, 0, 0).norm(dim=-1).max())) * max(
            1e-30, float(v.double().nan_to_num(0, 0, 0).norm(dim=-1).max()))
    a, c = first, k_first
    for s, (n, m) in enumerate(zip(nq, nk)):
        if n and m:
            i, j = torch.arange(n, device=q.device)[:, None], torch.arange(m, device=q.device)
            seen = torch.ones(n, m, dtype=torch.bool, device=q.device)
            if causal:
                seen = j <= i + m - n
                if prefix is not None:
                    seen = seen | (j < prefix[s])
            far = (i + m - n - j).abs().double()
            for h in range(H):
                Q, K, V = q[a:a + n, h].double(), k[c:c + m, h // G].double(), v[c:c + m, h // G].double()
                x = scale * (Q @ K.t())
                ds = 2 * D * U * scale * (Q.abs() @ K.abs().t())
                slant = torch.ones_like(x)
                if cap:
                    t = torch.tanh(x / cap)
                    x, slant = cap * t, 1 - t * t
                    ds = ds + 4 * U * cap
                bias = float(slopes[h]) * far if slopes is not None else torch.zeros_like(x)
                ds = ds + 4 * U * (x.abs() + bias)
                x = (x - bias).masked_fill(~seen, -math.inf)
                top = x.amax(-1, keepdim=True)
                none = top == -math.inf
                w = torch.exp(x - top.masked_fill(none, 0.0))
                total = w.sum(-1, keepdim=True)
                p = w / total.masked_fill(none, 1.0)
                ds = ds.masked_fill(~seen, 0.0).amax(-1, keepdim=True) + 4 * U * top.masked_fill(none, 0.0).abs()
                eta = torch.expm1(2 * ds) + 8 * U
                o = p @ V
                val["out"][a:a + n, h] = o
                val["lse"][h, a:a + n] = (top + torch.log(total))[:, 0]
                off = (half + eta + m * U) * (p @ V.abs()) + (tiny + flushed) * (seen.double() @ V.abs())
                tol["out"][a:a + n, h] = off + half * o.abs()
                tol["lse"][h, a:a + n] = (ds + eta + m * U + 2 * U * val["lse"][h, a:a + n, None].abs())[:, 0]
                if g is None:
                    continue
                g1 = g[a:a + n, h].double()
                dp, delta = g1 @ V.t(), (g1 * o).sum(-1, keepdim=True)
                e = p * (dp - delta) * slant
                d_delta = (g1.abs() * tol["out"][a:a + n, h]).sum(-1, keepdim=True) + 2 * D * U * (g1 * o).abs().sum(-1, keepdim=True)
                if near:
                    d_delta = (p * dp.abs()).sum(-1, keepdim=True) * (eta + m * U) + 2 * D * U * (p * (g1.abs() @ V.abs().t())).sum(-1, keepdim=True)
                d_e = e.abs() * ((half * half if near else half) + eta + 16 * U) + p * (slant + 8 * U) * (d_delta + 2 * D * U * (g1.abs() @ V.abs().t()))
                d_e = d_e + p * (dp - delta).abs() * 8 * U + ((2.0 if near else 1.0) * tiny * 2.0 ** -15 * peak + flushed * (dp - delta).abs()) * seen
                d_p = p * (half + eta) + (tiny * 2.0 ** -15 + flushed) * seen
                val["dq"][a:a + n, h] = scale * (e @ K)
                tol["dq"][a:a + n, h] = scale * ((d_e + m * U * e.abs()) @ K.abs())
                val["dk"][c:c + m, h // G] += scale * (e.t() @ Q)
                tol["dk"][c:c + m, h // G] += scale * ((d_e + n * G * U * e.abs()).t() @ Q.abs())
                val["dv"][c:c + m, h // G] += p.t() @ g1
                tol["dv"][c:c + m, h // G] += (d_p + n * G * U * p).t() @ g1.abs()
        a, c = a + n, c + m
    for name in ("dq", "dk", "dv"):
        tol[name] += half * val[name].abs()
    return val, tol


def _inputs(nq, nk, H, Hk, D, dtype, seed, device, tail=0):
    gen = torch.Generator().manual_seed(seed)
    T, M = sum(nq) + 2 * tail, sum(nk) + 2 * tail
    q, g = (torch.randn(T, H, D, generator=gen).to(dtype).to(device) for _ in range(2))
    k, v = (torch.randn(M, Hk, D, generator=gen).to(dtype).to(device) for _ in range(2))
    return q, k, v, g


def _offsets(n, dtype, device, first=0):
    return torch.tensor([first, *n]).cumsum(0).to(dtype).to(device)


def _close(got, val, tol, dtype):
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2 if dtype is not torch.float32 else 0.0
    none = torch.isneginf(val)
    assert torch.equal(torch.isneginf(got) & none, none)
    off = (got.double() - val).abs()[~none]
    limit = 1.01 * tol[~none] + tiny
    assert bool((off <= limit).all()), (float((off - limit).max()), int((~(off <= limit)).sum()), off.numel())


def run(nq, nk, H, Hk, D, dtype, device, causal=True, prefix=None, slopes=False, cap=0.0, scale=None, idx=torch.int32, tail=0,
        seed=0):
    from baidu_cti_grab_b200 import device_ops

    q, k, v, g = _inputs(nq, nq if nk is None else nk, H, Hk, D, dtype, seed, device, tail)
    off = _offsets(nq, idx, device, tail)
    k_off = None if nk is None else _offsets(nk, idx, device, tail)
    pre = None if prefix is None else torch.tensor(prefix, dtype=idx, device=device)
    slp = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device=device) if slopes else None
    how = dict(causal=causal, prefix=pre, slopes=slp, cap=cap, scale=scale)
    out, lse = device_ops.segment_attention(q, k, v, off, k_off, want_lse=True, **how)
    grads = device_ops.segment_attention_backward(g, q, k, v, out, lse, off, k_off, **how)
    half = torch.finfo(dtype).eps / 2
    val, tol = oracle(q, k, v, nq, nq if nk is None else nk, tail, tail, g, causal, prefix, slp, cap, scale, half, dtype is HF)
    _close(out, val["out"], tol["out"], dtype)
    _close(lse, val["lse"], tol["lse"], torch.float32)
    for name, got in zip(("dq", "dk", "dv"), grads):
        _close(got, val[name], tol[name], dtype)
    again = device_ops.segment_attention_backward(g, q, k, v, out, lse, off, k_off, **how)
    assert all(torch.equal(x, y) for x, y in zip(grads, again))  # the same bits again
    torch.cuda.synchronize()
    assert device_ops.device_error() == 0


CASES = [
    # query lengths, key lengths (None: the same), H, Hk, D, dtype, mask
    ([1], None, 1, 1, 64, BF, {}),
    ([1], [1000], 4, 4, 64, BF, {}),
    ([1], [0], 2, 1, 64, BF, {}),
    ([0, 0], None, 2, 2, 64, BF, {}),
    ([3, 1, 0, 5, 2], None, 2, 2, 8, HF, {}),
    ([64, 63, 65, 1, 127, 128, 129], None, 2, 1, 64, BF, {}),
    ([300], None, 1, 1, 128, BF, dict(causal=False)),
    ([129, 200, 31], None, 4, 2, 128, HF, dict(cap=20.0)),
    ([129, 200, 31], None, 3, 1, 64, HF, dict(cap=5.0, slopes=True)),
    ([100, 30, 77], [40, 30, 200], 2, 2, 64, BF, {}),               # more queries than keys: the first see nothing
    ([100, 30, 77], [40, 0, 200], 4, 1, 96, HF, dict(prefix=[7, 3, 300])),
    ([90, 140, 1], None, 2, 2, 64, BF, dict(prefix=[0, 60, 5], slopes=True)),
    ([513], None, 2, 2, 72, BF, dict(prefix=[100], cap=30.0)),
    ([4] * 70, None, 8, 2, 32, BF, {}),
    ([1] * 300, [3] * 300, 2, 2, 40, HF, {}),
    ([2] * 9, [700, 1, 64, 65, 900, 0, 128, 63, 300], 8, 2, 128, BF, {}),
    ([60, 40], None, 4, 2, 64, BF, {}),                             # fewer keys than a tile: heads that share them in one CTA
    ([60, 40], None, 6, 2, 128, HF, dict(prefix=[50, 0])),
    ([17, 16, 1], [1500, 40, 2000], 16, 1, 64, HF, dict(causal=False, slopes=True)),
    ([1, 1, 1], [5000, 1, 3001], 6, 2, 128, BF, dict(cap=15.0, slopes=True)),
    ([1000, 37], None, 1, 1, 16, BF, dict(scale=0.9)),
    ([257, 300], None, 5, 5, 120, BF, dict(slopes=True)),
    ([70, 41], None, 2, 1, 20, BF, dict(prefix=[9, 0], cap=8.0)),   # D off 8: row by row
    ([33, 64], None, 2, 2, 136, HF, dict(slopes=True)),             # D above the tiles'
    ([40], [90], 1, 1, 256, BF, {}),
]


@pytest.mark.parametrize("nq,nk,H,Hk,D,dtype,mask", CASES)
def test_against_float64(cuda_device, nq, nk, H, Hk, D, dtype, mask):
    run(nq, nk, H, Hk, D, dtype, cuda_device, seed=len(nq) + D, **mask)


@pytest.mark.parametrize("H,Hk,D,mask", [(2, 2, 64, {}), (4, 1, 128, dict(slopes=True)), (2, 1, 96, dict(cap=8.0)),
                                         (1, 1, 20, {}), (2, 2, 200, dict(prefix=[3] * 72)), (3, 3, 32, dict(causal=False))])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_gradients_of_few_keys(cuda_device, dtype, H, Hk, D, mask):
    """Where dp - delta is a small difference: dq and dk as near as their own rounding."""
    from baidu_cti_grab_b200 import device_ops

    nq = [4, 5, 0, 7, 8, 1, 2, 3] * 9
    q, k, v, g = _inputs(nq, nq, H, Hk, D, dtype, D, cuda_device)
    off = _offsets(nq, torch.int64, cuda_device)
    how = dict(mask, slopes=torch.full((H,), 0.25, device=cuda_device) if mask.get("slopes") else None)
    if "prefix" in mask:
        how["prefix"] = torch.tensor(mask["prefix"], device=cuda_device)
    out, lse = device_ops.segment_attention(q, k, v, off, want_lse=True, **how)
    grads = device_ops.segment_attention_backward(g, q, k, v, out, lse, off, **how)
    if "prefix" in mask:
        how["prefix"] = mask["prefix"]
    val, tol = oracle(q, k, v, nq, nq, g=g, half=torch.finfo(dtype).eps / 2, fp16=dtype is HF, near=True, **how)
    for name, got in zip(("dq", "dk", "dv"), grads):
        _close(got, val[name], tol[name], dtype)


@pytest.mark.parametrize("nq,nk,H,Hk,D,dtype", [
    ([300], [3000], 1, 1, 64, BF),                  # many queries of few heads: 16 rows a CTA, keys in parts
    ([33, 1, 20], [900, 2600, 4000], 8, 1, 64, HF),
    ([31] * 12, [700, 3, 129, 400] * 3, 8, 2, 128, BF),
    ([0, 0, 1, 0, 3] * 8, [900, 30, 700, 5, 2000] * 8, 8, 2, 64, HF),  # segments without queries among them
    ([1] * 200, [16] * 200, 8, 8, 64, BF),          # tiles of single queries by segment
    ([30] * 100, [130] * 100, 8, 8, 64, HF),        # tiles rather than 16 rows a CTA
    ([700, 900], None, 8, 2, 64, HF),               # few tiles of keys: heads that share them apart
    ([70] * 40, None, 8, 2, 64, BF),                # and together
])
def test_either_side_of_the_choices(cuda_device, nq, nk, H, Hk, D, dtype):
    run(nq, nk, H, Hk, D, dtype, cuda_device, seed=len(nq) + H)


@pytest.mark.parametrize("idx", [torch.int32, torch.int64])
@pytest.mark.parametrize("D", [64, 128, 20])
def test_rows_outside_every_segment(cuda_device, idx, D):
    """Rows before the first offset and behind the last see nothing: zeros, and no gradient."""
    run([50, 0, 170], None, 2, 1, D, BF, cuda_device, idx=idx, tail=37)
    run([1, 3], [900, 200], 4, 2, D, BF, cuda_device, idx=idx, tail=150)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_long_rows_and_large_scores(cuda_device, dtype):
    run([2100], None, 2, 2, 64, dtype, cuda_device, scale=1.0, seed=3)
    run([1100], None, 2, 1, 128, dtype, cuda_device, scale=0.7, cap=50.0, seed=4)


def test_oracle_against_differences():
    """The formulas' gradients against differences of the formula itself, in float64 on the CPU: with a step of 1e-5 the
    difference is off by about 1e-10 of third derivatives and 1e-16 / 1e-5 of rounding."""
    torch.manual_seed(0)
    nq, nk = [5, 3], [9, 2]
    q, g = (torch.randn(8, 4, 6, dtype=torch.float64) for _ in range(2))
    k, v = (torch.randn(11, 2, 6, dtype=torch.float64) for _ in range(2))
    how = dict(prefix=[4, 0], slopes=torch.tensor([0.5, 0.25, 0.1, 0.0]), cap=3.0)
    val, _ = oracle(q, k, v, nq, nk, g=g, **how)
    f = lambda *t: float((oracle(*t, nq, nk, **how)[0]["out"] * g).sum())  # noqa: E731
    for name, at in (("dq", 0), ("dk", 1), ("dv", 2)):
        d = torch.randn_like((q, k, v)[at])
        plus, minus = [q, k, v], [q, k, v]
        plus[at], minus[at] = plus[at] + 1e-5 * d, minus[at] - 1e-5 * d
        assert abs((f(*plus) - f(*minus)) / 2e-5 - float((val[name] * d).sum())) < 1e-6


@pytest.mark.parametrize("D", [64, 128, 24])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_is_not_seen_stays_out(cuda_device, D, bad):
    """NaN and infinities in other segments, behind the last one, and in keys that a query does not see."""
    from baidu_cti_grab_b200 import device_ops

    nq = [70, 90, 50]
    q, k, v, g = _inputs(nq, nq, 2, 1, D, BF, 11, cuda_device, 9)
    off = _offsets(nq, torch.int32, cuda_device, 9)
    want, lse = device_ops.segment_attention(q, k, v, off, want_lse=True)
    grads = device_ops.segment_attention_backward(g, q, k, v, want, lse, off)
    val, tol = oracle(q, k, v, nq, nq, 9, 9, g, half=2.0 ** -8)
    poisoned = [t.clone() for t in (q, k, v, g)]
    for t in poisoned:
        t[:9] = bad
        t[79:169] = bad  # the second segment
        t[219:] = bad
    for t in poisoned[1:3]:
        t[218] = bad     # the last key of the third: only its last query sees it
    q2, k2, v2, g2 = poisoned
    out, lse2 = device_ops.segment_attention(q2, k2, v2, off, want_lse=True)
    clean = torch.cat([torch.arange(9, 79), torch.arange(169, 218)]).to(cuda_device)
    _close(out[clean], val["out"][clean], tol["out"][clean], BF)
    assert torch.equal(out[:9], torch.zeros_like(out[:9])) and torch.equal(out[219:], torch.zeros_like(out[219:]))
    # gradients: the last query of the third segment is given none, so that its weights reach nothing
    g2[218] = 0
    _, tol3 = oracle(q, k, v, nq, nq, 9, 9, g, half=2.0 ** -8)
    dq, dk, dv = device_ops.segment_attention_backward(g2, q2, k2, v2, out, lse2, off)
    first = torch.arange(9, 79).to(cuda_device)
    for name, got in (("dq", dq), ("dk", dk), ("dv", dv)):
        _close(got[first], val[name][first], tol3[name][first], BF)
        assert torch.equal(got[:9], torch.zeros_like(got[:9])) and torch.equal(got[219:], torch.zeros_like(got[219:]))
    third = torch.arange(169, 218).to(cuda_device)
    _close(dq[third], val["dq"][third], tol3["dq"][third], BF)
    assert all(bool(t.isfinite().all()) for t in grads)
    torch.cuda.synchronize()
    assert device_ops.device_error() == 0


@pytest.mark.parametrize("splits", [1, 4])
def test_what_few_queries_do_not_see_stays_out(cuda_device, splits):
    """The same where few queries meet many keys: another segment's NaN, and the keys behind a query's own."""
    from baidu_cti_grab_b200 import device_ops

    nq, nk = [2, 1, 2], [300 * splits, 70, 299 * splits]
    q, k, v, _ = _inputs(nq, nk, 4, 2, 128, BF, 13, cuda_device, 5)
    off, k_off = _offsets(nq, torch.int32, cuda_device, 5), _offsets(nk, torch.int32, cuda_device, 5)
    val, tol = oracle(q, k, v, nq, nk, 5, 5, half=2.0 ** -8)
    out, lse = device_ops.segment_attention(q, k, v, off, k_off, want_lse=True)
    _close(out, val["out"], tol["out"], BF)
    _close(lse, val["lse"], tol["lse"], torch.float32)
    for t in (k, v):
        t[:5] = math.nan
        t[5 + nk[0]:5 + nk[0] + nk[1]] = math.inf
        t[5 + sum(nk) - 1:] = math.nan  # the last key of the third segment: only its last query sees it
    q[:5] = math.nan
    out, _ = device_ops.segment_attention(q, k, v, off, k_off)
    clean = torch.tensor([5, 6, 8], device=cuda_device)
    _close(out[clean], val["out"][clean], tol["out"][clean], BF)
    assert torch.equal(out[:5], torch.zeros_like(out[:5])) and torch.equal(out[10:], torch.zeros_like(out[10:]))


def test_no_segments_and_no_keys(cuda_device):
    """No segment at all, segments without keys, no query: zeros, and shapes."""
    from baidu_cti_grab_b200 import device_ops

    q, k, v, g = _inputs([40], [70], 2, 1, 64, BF, 3, cuda_device)
    none = torch.zeros(1, dtype=torch.int64, device=cuda_device)
    for off, k_off, keys in ((none, none, 70), (torch.tensor([0, 40], device=cuda_device), torch.tensor([0, 0], device=cuda_device), 70),
                             (torch.tensor([0, 40], device=cuda_device), torch.tensor([0, 0], device=cuda_device), 0)):
        out, lse = device_ops.segment_attention(q, k[:keys], v[:keys], off, k_off, want_lse=True)
        assert not out.any() and bool(torch.isneginf(lse).all())
        grads = device_ops.segment_attention_backward(g, q, k[:keys], v[:keys], out, lse, off, k_off)
        assert not any(bool(t.any()) for t in grads)
    off = torch.zeros(2, dtype=torch.int64, device=cuda_device)
    out, lse = device_ops.segment_attention(q[:0], k, v, off, torch.tensor([0, 70], device=cuda_device), want_lse=True)
    assert out.shape == (0, 2, 64) and lse.shape == (2, 0)
    dq, dk, dv = device_ops.segment_attention_backward(g[:0], q[:0], k, v, out, lse, off, torch.tensor([0, 70], device=cuda_device))
    assert dq.shape == (0, 2, 64) and not dk.any() and not dv.any()


def test_gradients_of_any_size_in_fp16(cuda_device):
    """fp16 gradients over the type's whole range: weights and their gradients are scaled into it."""
    from baidu_cti_grab_b200 import device_ops

    nq = [200, 600]
    for up in (2.0 ** -14, 1.0, 2.0 ** 11):
        q, k, v, g = _inputs(nq, nq, 2, 2, 64, HF, 5, cuda_device)
        g = (g.float() * up).to(HF)
        off = _offsets(nq, torch.int32, cuda_device)
        out, lse = device_ops.segment_attention(q, k, v, off, want_lse=True)
        grads = device_ops.segment_attention_backward(g, q, k, v, out, lse, off)
        val, tol = oracle(q, k, v, nq, nq, g=g, half=2.0 ** -11, fp16=True)
        for name, got in zip(("dq", "dk", "dv"), grads):
            _close(got, val[name], tol[name], HF)


@pytest.mark.parametrize("D", [64, 128])
def test_strides_streams_and_graphs(cuda_device, D):
    from baidu_cti_grab_b200 import device_ops

    nq, H, Hk = [40, 300, 1, 90], 4, 2
    q, k, v, g = _inputs(nq, nq, H, Hk, D, BF, 21, cuda_device)
    off = _offsets(nq, torch.int64, cuda_device)
    out, lse = device_ops.segment_attention(q, k, v, off, want_lse=True)
    grads = device_ops.segment_attention_backward(g, q, k, v, out, lse, off)
    # parts of one projection, heads first, and odd rows that no tensor map takes
    fused = torch.cat([q, k, v], 1)
    parts = fused[:, :H], fused[:, H:H + Hk], fused[:, H + Hk:]
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v, g)]
    odd = [torch.empty(t.numel() + 1, dtype=BF, device=cuda_device)[1:].view(t.shape).copy_(t) for t in (q, k, v, g)]
    wide = [torch.cat([t, t], -1)[..., ::2] for t in (q.repeat_interleave(2, -1)[..., :D * 2],)]
    assert wide[0].stride(-1) == 2
    for a, b, c, d in ((*parts, g), tuple(turned), tuple(odd)):
        o2, l2 = device_ops.segment_attention(a, b, c, off, want_lse=True)
        assert torch.equal(o2, out) and torch.equal(l2, lse)
        for x, y in zip(device_ops.segment_attention_backward(d, a, b, c, o2, l2, off), grads):
            assert torch.equal(x, y)
    shared = k[:, :1].expand(-1, Hk, -1)  # a key head given twice
    o2, _ = device_ops.segment_attention(q, shared, v, off)
    o3, _ = device_ops.segment_attention(q, shared.contiguous(), v, off)
    assert torch.equal(o2, o3)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o2, l2 = device_ops.segment_attention(q, k, v, off, want_lse=True)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o2, out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o2, l2 = device_ops.segment_attention(q, k, v, off, want_lse=True)
        g2 = device_ops.segment_attention_backward(g, q, k, v, o2, l2, off)
    for _ in range(2):
        for t in (o2, l2, *g2):
            t.zero_()
        graph.replay()
        assert torch.equal(o2, out) and torch.equal(l2, lse) and all(torch.equal(x, y) for x, y in zip(g2, grads))
    # other segments in the same offsets array: what a captured call reads is the array, not what it held
    off.copy_(_offsets([100, 100, 100, 131], torch.int64, cuda_device))
    graph.replay()
    o4, _ = device_ops.segment_attention(q, k, v, off)
    assert torch.equal(o2, o4) and not torch.equal(o4, out)


def test_offsets_outside_the_rows_name_none(cuda_device):
    """Offsets below 0 or past the rows are taken as the nearest row."""
    from baidu_cti_grab_b200 import device_ops

    q, k, v, _ = _inputs([100], [100], 2, 2, 64, BF, 2, cuda_device)
    wild = torch.tensor([-5, 40, 1 << 40], device=cuda_device)
    tame = torch.tensor([0, 40, 100], device=cuda_device)
    for off in (wild, tame):
        out, _ = device_ops.segment_attention(q, k, v, off)
        if off is wild:
            first = out
    assert torch.equal(first, out)


def test_module_trains_and_reads_a_cache(cuda_device):
    """A layer's gradients through autograd against torch's own operations in float64, and new items over a cache
    against all items at once: two roundings to bf16 more or less on either side, under 2^-6 in relative L2."""
    from baidu_cti_grab_b200 import attention

    torch.manual_seed(1)
    D, H, n = 64, 4, [30, 1, 77]
    layer = attention.SegmentAttention(D, H, 2, cap=10.0, distance=True).to(cuda_device, BF)
    assert layer.slopes.dtype == torch.float32
    off = _offsets(n, torch.int64, cuda_device)
    x = torch.randn(sum(n), D, device=cuda_device, dtype=BF, requires_grad=True)
    g = torch.randn(sum(n), D, device=cuda_device, dtype=BF)
    y = layer(x, off)
    y.backward(g)
    w = {name: p.detach().double().requires_grad_() for name, p in layer.named_parameters()}
    x64 = x.detach().double().requires_grad_()
    lin = torch.nn.functional.linear
    q, k, v = lin(x64, w["qkv.weight"], w["qkv.bias"]).view(-1, 2 * H, D // H).split((H, 2, 2), 1)
    rows = []
    for a, b in zip(off[:-1], off[1:]):
        i = torch.arange(int(b - a), device=cuda_device)
        far = i[:, None] - i
        s = torch.einsum("ihd,jhd->hij", q[a:b], k[a:b].repeat_interleave(2, 1)) / (D // H) ** 0.5
        s = 10.0 * torch.tanh(s / 10.0) - layer.slopes.double()[:, None, None] * far.abs()
        s = s.masked_fill(far < 0, -math.inf)
        rows.append(torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v[a:b].repeat_interleave(2, 1)).flatten(1))
    y64 = lin(torch.cat(rows), w["out.weight"], w["out.bias"])
    y64.backward(g.double())
    rel = lambda got, want: float((got.double() - want).norm() / want.norm())  # noqa: E731
    assert rel(y, y64.detach()) < 2.0 ** -6 and rel(x.grad, x64.grad) < 2.0 ** -6
    for name, p in layer.named_parameters():
        assert rel(p.grad, w[name].grad) < 2.0 ** -6, name
    with torch.no_grad():
        k, v = layer.keys_and_values(x)
        last = off[1:] - 1
        new = layer(x[last], torch.arange(len(n) + 1, device=cuda_device), cache=(k, v, off))
        assert rel(new, y[last].double()) < 2.0 ** -6
    with pytest.raises(RuntimeError):
        attention.segment_attention(q.bfloat16(), k, v, off, slopes=layer.slopes.clone().requires_grad_())


@pytest.mark.parametrize("D", [64, 128])
def test_rows_that_are_taken_again_hold_nobody_up(cuda_device, D):
    """A NaN among a long segment's values: a tile that meets it takes its rows again one by one, seconds of work for 32
    rows of 120,000 keys, and the tiles behind it in the same CTA have waits of bounded time.  All rows are written, other
    users' and those before the last tile with the same bits as without the NaN.

    The last tile's rows: either result is within half + eta + n u of sum p |v| and half of itself, with
    eta < 2^-10 (scale sum |q| |k| is under 2^5 here, so ds under 2 D u 2^5 = 2^-11)."""
    from baidu_cti_grab_b200 import device_ops

    n = [120_000, 300]
    q, k, v, _ = _inputs(n, n, 1, 1, D, BF, D, cuda_device)
    off = _offsets(n, torch.int32, cuda_device)
    want, _ = device_ops.segment_attention(q, k, v, off)
    spread, _ = device_ops.segment_attention(q, k, v.abs(), off)
    v[n[0] - 1] = math.nan  # which the segment's last query alone sees
    got, _ = device_ops.segment_attention(q, k, v, off)
    assert device_ops.device_error() == 0
    assert torch.equal(got[:n[0] - 128], want[:n[0] - 128]) and torch.equal(got[n[0] + 128:], want[n[0] + 128:])
    rest = [i for i in range(n[0] - 128, n[0] + 128) if i != n[0] - 1]
    off_by = (got[rest].double() - want[rest].double()).abs()
    half = torch.finfo(BF).eps / 2
    assert bool((off_by <= 2 * ((half + 2.0 ** -10 + n[0] * U) * spread[rest].double() * (1 + half) + half * want[rest].double().abs() * (1 + half))).all())
    assert bool(got[n[0] - 1].isnan().all())


def _few_bits(dtype, exact, spread, loose):
    """A value rounded once: half of itself, and sums of weights as two values (half of half of them, in fp16 2^-32 of the
    largest of up to 3000) beside `loose`, the bound without any of these."""
    half = torch.finfo(dtype).eps / 2
    return half * exact.abs() + (half * half + (3000 * 2.0 ** -32 if dtype is HF else 0.0)) * spread + loose * (1 + half)


@pytest.mark.parametrize("nq,nk,H,Hk,D,mask", [
    ([300, 41], None, 2, 2, 64, {}), ([257, 130], None, 4, 1, 128, dict(cap=20.0)), ([90] * 8, None, 2, 2, 40, dict(causal=False)),
    ([2, 1, 3], [1500, 40, 2700], 8, 2, 64, {}), ([5], [2900], 4, 1, 128, dict(causal=False)),
])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_weights_keep_their_bits(cuda_device, dtype, nq, nk, H, Hk, D, mask):
    """`out` is as near as its own rounding: the weights meet the values with twice the type's bits."""
    from baidu_cti_grab_b200 import device_ops

    nk = nq if nk is None else nk
    q, k, v, _ = _inputs(nq, nk, H, Hk, D, dtype, D, cuda_device)
    off, k_off = _offsets(nq, torch.int32, cuda_device), _offsets(nk, torch.int32, cuda_device)
    out, _ = device_ops.segment_attention(q, k, v, off, k_off, **mask)
    val, loose = oracle(q, k, v, nq, nk, **mask)
    spread, _ = oracle(q, k, v.abs(), nq, nk, **mask)
    _close(out, val["out"], _few_bits(dtype, val["out"], spread["out"], loose["out"]), dtype)


def test_many_small_weights_in_fp16(cuda_device):
    """One key of a score 17 above 20,000 others, whose weights of 2^-24.5 fp16 by itself rounds to 2^-24: what a weight is
    rounded to is 2^-32 of the largest, and each sum is off by m u.  Either form of the kernels."""
    from baidu_cti_grab_b200 import device_ops

    m = 20_000
    for Tq in (1, 6000):
        q, k, v = (torch.zeros(n, 1, 64, device=cuda_device, dtype=HF) for n in (Tq, m, m))
        q[..., 0], k[0, :, 0], v[1:] = 8.0, 17.0, 1.0
        off, k_off = _offsets([Tq], torch.int32, cuda_device), _offsets([m], torch.int32, cuda_device)
        out, lse = device_ops.segment_attention(q, k, v, off, k_off, causal=False, want_lse=True)
        w = (m - 1) * math.exp(-17.0)
        assert bool((out.double() - w / (1 + w)).abs().max() <= w / (1 + w) * (2.0 ** -11 + 2.0 ** -17 + 2 * m * U) + m * 2.0 ** -32)
        assert bool((lse.double() - 17.0 - math.log1p(w)).abs().max() <= 2.0 ** -17 + m * U)


@pytest.mark.parametrize("nq,nk,H,Hk,D,mask", [
    ([300, 41], None, 2, 2, 64, {}), ([700], None, 4, 1, 64, dict(causal=False)), ([257, 130], None, 4, 2, 128, dict(cap=20.0)),
    ([90] * 8, [200] * 8, 2, 2, 40, {}),
])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_value_gradients_keep_their_bits(cuda_device, dtype, nq, nk, H, Hk, D, mask):
    """dv is as near as its own rounding: p meets the output's gradient with twice the type's bits (in fp16 p is brought
    up by 2^15 and loses 2^-40 of at most 3000 rows)."""
    from baidu_cti_grab_b200 import device_ops

    nk = nq if nk is None else nk
    q, k, v, g = _inputs(nq, nk, H, Hk, D, dtype, D, cuda_device)
    off, k_off = _offsets(nq, torch.int32, cuda_device), _offsets(nk, torch.int32, cuda_device)
    out, lse = device_ops.segment_attention(q, k, v, off, k_off, want_lse=True, **mask)
    dv = device_ops.segment_attention_backward(g, q, k, v, out, lse, off, k_off, **mask)[2]
    val, loose = oracle(q, k, v, nq, nk, g=g, **mask)
    spread, _ = oracle(q, k, v, nq, nk, g=g.abs(), **mask)
    _close(dv, val["dv"], _few_bits(dtype, val["dv"], spread["dv"], loose["dv"]), dtype)


@pytest.mark.parametrize("D,mask", [(64, {}), (64, dict(cap=50.0)), (128, {}), (128, dict(cap=40.0, causal=False)), (24, {}), (20, {}), (200, {})])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_gradients_where_one_key_has_the_weight(cuda_device, dtype, D, mask):
    """Long rows whose weight lies on one key: dp - delta is a small difference there as in short rows, and dq and dk are as
    near as their own rounding.  Beside `near`'s bound: the first delta is off by half of out at most, and that times
    sum p |k|, whose p is rounded once, is what the correction of dq is off by."""
    from baidu_cti_grab_b200 import device_ops

    nq, H = [300, 41, 700], 2
    q, k, v, g = _inputs(nq, nq, H, H, D, dtype, D, cuda_device)
    q = (1.5 * (64 / D) ** 0.25 * k.float()).to(dtype)
    off = _offsets(nq, torch.int32, cuda_device)
    out, lse = device_ops.segment_attention(q, k, v, off, want_lse=True, **mask)
    grads = device_ops.segment_attention_backward(g, q, k, v, out, lse, off, **mask)
    half = torch.finfo(dtype).eps / 2
    val, tol = oracle(q, k, v, nq, nq, g=g, half=half, fp16=dtype is HF, near=True, **mask)
    reach, _ = oracle(q, k, k.abs(), nq, nq, **mask)
    first = (g.double().abs() * val["out"].abs()).sum(-1, keepdim=True) * half * (1 + 2.0 ** -6)
    tol["dq"] += D ** -0.5 * half * first * reach["out"]
    for name, got in zip(("dq", "dk", "dv"), grads):
        _close(got, val[name], tol[name], dtype)


def test_prefix_of_another_type_than_the_offsets(cuda_device):
    """A prefix beyond int32 is all of a segment's keys, whatever the offsets' type; one below 0 is none."""
    from baidu_cti_grab_b200 import device_ops

    nq = [40, 30, 50]
    q, k, v, _ = _inputs(nq, nq, 2, 2, 64, BF, 3, cuda_device)
    all_of = torch.tensor([1 << 32, (1 << 40) + 1, -(1 << 33) + 5], device=cuda_device)
    want, _ = device_ops.segment_attention(q, k, v, _offsets(nq, torch.int64, cuda_device), prefix=all_of)
    got, _ = device_ops.segment_attention(q, k, v, _offsets(nq, torch.int32, cuda_device), prefix=all_of)
    small, _ = device_ops.segment_attention(q, k, v, _offsets(nq, torch.int32, cuda_device), prefix=torch.tensor([40, 30, 0], device=cuda_device))
    assert torch.equal(got, want) and torch.equal(got, small)
    val, tol = oracle(q, k, v, nq, nq, prefix=[40, 30, 0], half=2.0 ** -8)
    _close(got, val["out"], tol["out"], BF)


@pytest.mark.parametrize("D", [16, 20, 72])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_gradients_of_saturated_scores(cuda_device, dtype, D):
    """Scores of 4.5 to 8 caps: dk and dq follow 1 - tanh^2, 5e-4 to 5e-7, which has to keep its own precision.

    1 - tanh(y)^2 changes by 2 of what y is off by; the rest as at the head of this file, delta as in `near`."""
    from baidu_cti_grab_b200 import device_ops

    n, m, cap = 96, 130, 0.5
    gen = torch.Generator().manual_seed(D)
    q, k, v, g = (torch.randn(r, 1, D, generator=gen) for r in (n, m, m, n))
    q, k = 0.01 * q, 0.01 * k
    q[..., 0] = 1.0
    k[:, 0, 0] = torch.linspace(4.5, 8.0, m) * cap * (1 - 2 * (torch.arange(m) % 2))
    q, k, v, g = (t.to(dtype).to(cuda_device) for t in (q, k, v, g))
    off, k_off = _offsets([n], torch.int32, cuda_device), _offsets([m], torch.int32, cuda_device)
    how = dict(causal=False, cap=cap, scale=1.0)
    out, lse = device_ops.segment_attention(q, k, v, off, k_off, want_lse=True, **how)
    dq, dk, _ = device_ops.segment_attention_backward(g, q, k, v, out, lse, off, k_off, **how)
    Q, K, V, G = (t[:, 0].double() for t in (q, k, v, g))
    x = Q @ K.t()
    ds = 2 * D * U * (Q.abs() @ K.abs().t())
    slant = 1 / torch.cosh(x / cap) ** 2
    p = torch.softmax(cap * torch.tanh(x / cap), -1)
    dp = G @ V.t()
    delta = (p * dp).sum(-1, keepdim=True)
    e = p * (dp - delta) * slant
    half = torch.finfo(dtype).eps / 2
    eta = torch.expm1(2 * (ds.amax(-1, keepdim=True) + 8 * U * cap)) + 8 * U
    d_dp = 2 * D * U * (G.abs() @ V.abs().t())
    first = half * (G.abs() * (p @ V).abs()).sum(-1, keepdim=True)  # the delta that dq is corrected from, p rounded once
    d_delta = (p * dp.abs()).sum(-1, keepdim=True) * (eta + m * U) + (p * d_dp).sum(-1, keepdim=True)
    d_e = e.abs() * (half * half + eta + 2 * (ds / cap + 4 * U * (x / cap).abs()) + 16 * U) + p * slant * (d_delta + d_dp)
    if dtype is HF:
        d_e = d_e + 2 * 2.0 ** -40 * 2 * G.norm(dim=-1).max() * V.norm(dim=-1).max()
    for got, want, tol in ((dq, e @ K, (d_e + half * first * p * slant) @ K.abs() + m * U * (e.abs() @ K.abs())),
                           (dk, e.t() @ Q, (d_e + n * U * e.abs()).t() @ Q.abs())):
        _close(got[:, 0], want, tol + half * want.abs(), dtype)


@pytest.mark.parametrize("nq,nk,H,Hk,D", [([200, 65], None, 2, 1, 64), ([130], None, 2, 2, 128), ([2, 1], [900, 1500], 4, 1, 64),
                                          ([60], None, 1, 1, 20)])
@pytest.mark.parametrize("cap", [300.0, 1e5, 1e30])
def test_caps_far_above_the_scores(cuda_device, cap, nq, nk, H, Hk, D):
    """A cap that no score comes near changes nothing: a score is off by 16 u of itself, however large the cap is (and by
    x^3 / 3 cap^2 from x, which the definition has too)."""
    from baidu_cti_grab_b200 import device_ops

    nk = nq if nk is None else nk
    q, k, v, g = _inputs(nq, nk, H, Hk, D, HF, D, cuda_device)
    off, k_off = _offsets(nq, torch.int32, cuda_device), _offsets(nk, torch.int32, cuda_device)
    out, lse = device_ops.segment_attention(q, k, v, off, k_off, want_lse=True, cap=cap)
    grads = device_ops.segment_attention_backward(g, q, k, v, out, lse, off, k_off, cap=cap)
    val, _ = oracle(q, k, v, nq, nk, g=g, cap=cap)
    spread, _ = oracle(q, k, v.abs(), nq, nk, cap=cap)
    _, loose = oracle(q, k, v, nq, nk, g=g, half=2.0 ** -11, fp16=True)
    _, bare = oracle(q, k, v, nq, nk)
    more = 2.0 ** -18  # 2 (16 u) |x|, of scores under 8: exp's argument and the sum's
    assert float(val["lse"].abs().max()) < 16
    _close(out, val["out"], _few_bits(HF, val["out"], spread["out"], bare["out"] + more * spread["out"]), HF)
    _close(lse, val["lse"], bare["lse"] + more, torch.float32)
    for name, got in zip(("dq", "dk", "dv"), grads):
        _close(got, val[name], loose[name], HF)


@pytest.mark.parametrize("H,Hk,D", [(2, 2, 64), (4, 2, 128), (6, 1, 32), (2, 1, 20)])
def test_other_users_take_no_bits_in_fp16(cuda_device, H, Hk, D):
    """The gradients of one segment in fp16 are the same bits whatever the size of another segment's rows and of the rows
    behind the last, and as near as their own rounding (e is scaled by the segment's own largest rows)."""
    from baidu_cti_grab_b200 import device_ops

    nq = [100, 90, 170]
    q, k, v, g = _inputs(nq, nq, H, Hk, D, HF, D, cuda_device, 40)
    off = _offsets(nq, torch.int32, cuda_device, 40)
    g = (g.float() * 2.0 ** -6).to(HF)
    grads = {}
    for up in (1.0, 2.0 ** 9):
        g2, v2 = g.clone(), v.clone()
        for t in (g2, v2):
            for rows in (slice(0, 40), slice(140, 230), slice(400, None)):
                t[rows] = (t[rows].float() * up).to(HF)
        g2[140:230] = (g2[140:230].float() * up ** 0.5).to(HF)
        out, lse = device_ops.segment_attention(q, k, v2, off, want_lse=True)
        grads[up] = device_ops.segment_attention_backward(g2, q, k, v2, out, lse, off)
    for a, b in zip(*grads.values()):
        assert torch.equal(a[40:140], b[40:140]) and torch.equal(a[230:400], b[230:400])
    for first, n in ((40, 100), (230, 170)):
        mine = slice(first, first + n)
        val, tol = oracle(q[mine], k[mine], v[mine], [n], [n], g=g[mine], half=2.0 ** -11, fp16=True, near=True)
        reach, _ = oracle(q[mine], k[mine], k[mine].abs(), [n], [n])
        near = (g[mine].double().abs() * val["out"].abs()).sum(-1, keepdim=True) * 2.0 ** -11 * (1 + 2.0 ** -6)
        tol["dq"] += D ** -0.5 * 2.0 ** -11 * near * reach["out"]
        for name, got in zip(("dq", "dk", "dv"), grads[2.0 ** 9]):
            _close(got[mine], val[name], tol[name], HF)


@pytest.mark.parametrize("nq,H,Hk,D,dtype,mask", [
    ([300] * 60, 4, 2, 128, BF, {}), ([260, 700, 130, 1, 515] * 12, 4, 4, 96, HF, dict(cap=15.0)),
    ([2500, 2300], 16, 4, 128, BF, dict(causal=False)), ([400] * 150, 6, 6, 64, HF, {}),
])
def test_tiles_behind_one_another(cuda_device, nq, H, Hk, D, dtype, mask):
    """More tiles of several blocks than the GPU holds CTAs: each takes several of them in turn, the next tile's copies and
    scores begun before the last one's rows are done."""
    run(nq, None, H, Hk, D, dtype, cuda_device, seed=D, **mask)


@pytest.mark.parametrize("D", [64, 128, 20])
def test_columns_apart(cuda_device, D):
    """Heads whose columns lie two elements apart, in any of the operands: the same bits as contiguous ones."""
    from baidu_cti_grab_b200 import device_ops

    nq = [40, 300, 1, 90]
    operands = _inputs(nq, nq, 4, 2, D, BF, 22, cuda_device)
    q, k, v, g = operands
    off = _offsets(nq, torch.int64, cuda_device)
    out, lse = device_ops.segment_attention(q, k, v, off, want_lse=True)
    grads = device_ops.segment_attention_backward(g, q, k, v, out, lse, off)
    apart = [torch.stack([t, -t], -1)[..., 0] for t in operands]
    assert all(t.stride(-1) == 2 and torch.equal(t, o) for t, o in zip(apart, operands))
    for which in ((0,), (1,), (2,), (3,), (0, 1, 2, 3)):
        a, b, c, d = (apart[i] if i in which else operands[i] for i in range(4))
        o2, l2 = device_ops.segment_attention(a, b, c, off, want_lse=True)
        assert torch.equal(o2, out) and torch.equal(l2, lse)
        for x, y in zip(device_ops.segment_attention_backward(d, a, b, c, o2, l2, off), grads):
            assert torch.equal(x, y)


@pytest.mark.parametrize("D", [64, 128, 24])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_is_not_seen_stays_out_in_fp16(cuda_device, D, bad):
    """In fp16 too, whose gradients are scaled by the largest finite rows: another segment's NaN and infinities, and those
    of the rows outside, change no bit of the first and third segment's."""
    from baidu_cti_grab_b200 import device_ops

    nq = [70, 90, 50]
    clean = _inputs(nq, nq, 2, 1, D, HF, 11, cuda_device, 9)
    off = _offsets(nq, torch.int32, cuda_device, 9)
    half = 2.0 ** -11
    val, tol = oracle(*clean[:3], nq, nq, 9, 9, clean[3], half=half, fp16=True)
    q, k, v, g = (t.clone() for t in clean)
    for t in (q, k, v, g):
        t[:9] = bad
        t[79:169] = bad
        t[219:] = bad
    out, lse = device_ops.segment_attention(q, k, v, off, want_lse=True)
    grads = device_ops.segment_attention_backward(g, q, k, v, out, lse, off)
    mine = torch.cat([torch.arange(9, 79), torch.arange(169, 219)]).to(cuda_device)
    for name, got in (("out", out), *zip(("dq", "dk", "dv"), grads)):
        _close(got[mine], val[name][mine], tol[name][mine], HF)
        assert not got[:9].any() and not got[219:].any()
    _close(lse[:, mine], val["lse"][:, mine], tol["lse"][:, mine], torch.float32)
    # a NaN of its own makes a row of the gradients NaN, and the keys that it sees, and nothing else
    q, k, v, g = (t.clone() for t in clean)
    g[9 + 40] = bad
    out, lse = device_ops.segment_attention(q, k, v, off, want_lse=True)
    dq, dk, dv = device_ops.segment_attention_backward(g, q, k, v, out, lse, off)
    assert bool((~dq[49].isfinite()).any(-1).all()) and bool((~dv[9:50].isfinite()).any(-1).all())
    rest = torch.tensor([i for i in range(9, 79) if i != 49] + list(range(79, 219)), device=cuda_device)
    _close(dq[rest], val["dq"][rest], tol["dq"][rest], HF)
    for name, got in (("dk", dk), ("dv", dv)):
        _close(got[50:], val[name][50:], tol[name][50:], HF)
    torch.cuda.synchronize()
    assert device_ops.device_error() == 0
