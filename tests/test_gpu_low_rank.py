"""Low-rank adapters beside a shared projection (rb_low_rank_add, adapters.py) on the GPU against the
definition in float64.

Tolerance: h = A x is a sum of K products in fp32, off by at most K u of sum |a| |x| (u = 2^-24); on the
tensor-core path it is rounded to the model type (half a step of |h|, or of its smallest subnormal).  B h adds rank u of
sum |B| |h|.  So out is within  sum_j |B_j| |s| (eps / 2 |h_j| + tiny + (K + rank) u sum |a| |x|)  and, rounded once, half a
step of itself (the fp32 sum with y adds u of the terms, inside the same bound's factor 1.01).
"""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _inputs(T, K, N, rank, R, dtype, run, seed):
    gen = torch.Generator().manual_seed(seed)
    x, y = torch.randn(T, K, generator=gen).to(dtype), torch.randn(T, N, generator=gen).to(dtype)
    a = (torch.randn(R, rank, K, generator=gen) * K ** -0.5).to(dtype)
    b = (torch.randn(R, N, rank, generator=gen) * rank ** -0.5).to(dtype)
    scale = torch.rand(R, generator=gen) + 0.5
    starts = torch.rand(T, generator=gen) < 1.0 / run
    chosen = torch.randint(-1, R, (T + 1,), generator=gen)
    return y, x, a, b, chosen[starts.long().cumsum(0)], scale


def _check(got, y, x, a, b, adapter, scale):
    dev = got.device
    y, x, a, b, adapter = (t.to(dev) for t in (y, x, a, b, adapter))
    scale = torch.ones(a.shape[0], device=dev) if scale is None else scale.to(dev)
    rank, K = a.shape[1:]
    fi = torch.finfo(y.dtype)
    want, bound = y.double(), torch.zeros_like(y, dtype=torch.float64)
    tiny = fi.smallest_normal * fi.eps / 2
    for i in range(a.shape[0]):
        t = (adapter == i).nonzero()[:, 0]
        if not len(t):
            continue
        xi, ai, bi, s = x[t].double(), a[i].double(), b[i].double(), scale[i].double()
        h = xi @ ai.t()
        want[t] += s * (h @ bi.t())
        off = fi.eps / 2 * h.abs() + tiny + (K + rank) * 2.0 ** -24 * (xi.abs() @ ai.abs().t())
        bound[t] = 1.01 * s.abs() * (off @ bi.abs().t()) + 2.0 ** -23 * y[t].double().abs()
    off = (got.double() - want).abs()
    limit = fi.eps / 2 * want.abs() + bound + tiny
    assert bool((off <= limit).all()), (float((off - limit).max()), int((off > limit).sum()))
    none = (adapter < 0) | (adapter >= a.shape[0])
    assert torch.equal(got[none], y[none])


SHAPES = [
    # T, K, N, rank, R, dtype, run
    (1, 512, 1536, 16, 4, BF, 1),
    (1, 14336, 512, 32, 2, BF, 1),
    (7, 40, 24, 8, 3, HF, 2),
    (64, 512, 1536, 16, 32, BF, 1),
    (96, 512, 513, 16, 5, BF, 4),
    (97, 512, 512, 16, 5, BF, 30),
    (128, 64, 64, 16, 1, BF, 10),
    (129, 8, 16, 8, 2, HF, 10),
    (300, 72, 200, 8, 7, BF, 9),
    (300, 512, 512, 32, 3, HF, 25),
    (700, 200, 100, 64, 3, BF, 50),
    (700, 200, 101, 24, 5, HF, 20),
    (515, 1000, 1544, 8, 24, HF, 7),
    (513, 512, 640, 40, 9, BF, 3),
    (1000, 4096, 512, 48, 4, BF, 80),
    (2049, 14336, 512, 32, 6, BF, 100),
    (256, 512, 512, 16, 300, BF, 1),        # every row of a tile its own adapter
    (19000, 128, 192, 16, 11, BF, 60),      # enough tiles for one fused kernel
    (19001, 256, 72, 8, 130, HF, 2),
    (60000, 72, 136, 16, 9, BF, 40),        # several tiles a CTA, of one group and of more
    (60001, 64, 72, 64, 5, HF, 30),
    (200, 100, 64, 16, 3, BF, 9),           # K not a multiple of 8: token kernel
    (200, 96, 64, 12, 3, HF, 9),            # rank not a multiple of 8
    (130, 96, 64, 128, 3, BF, 9),           # rank above the tensor path's
]


@pytest.mark.parametrize("T,K,N,rank,R,dtype,run", SHAPES)
def test_against_float64(cuda_device, T, K, N, rank, R, dtype, run):
    from baidu_cti_grab_b200 import device_ops

    args = _inputs(T, K, N, rank, R, dtype, run, T + K)
    y, x, a, b, adapter, scale = (t.to(cuda_device) for t in args)
    got = device_ops.low_rank_add(y, x, a, b, adapter, scale)
    _check(got, *args)
    assert torch.equal(device_ops.low_rank_add(y, x, a, b, adapter.int(), scale), got)  # and the same bits again
    _check(device_ops.low_rank_add(y, x, a, b, adapter), *args[:5], None)
    place = y.clone()
    assert device_ops.low_rank_add(place, x, a, b, adapter, scale, out=place) is place
    assert torch.equal(place, got)
    torch.cuda.synchronize()
    assert device_ops.device_error() == 0


@pytest.mark.parametrize("T", [50, 600, 19500])
def test_strides_odd_offsets_and_rows_left_alone(cuda_device, T):
    from baidu_cti_grab_b200 import device_ops

    K, N = 128, 96
    args = _inputs(T, K, N, 16, 6, BF, 12, 5)
    y, x, a, b, adapter, scale = (t.to(cuda_device) for t in args)
    want = device_ops.low_rank_add(y, x, a, b, adapter, scale)
    for ldx, offx, ld, off in ((K + 8, 0, N + 16, 0), (K + 8, 8, N + 8, 8), (K, 1, N + 3, 1)):
        rx = torch.zeros(T * ldx + offx, dtype=BF, device=cuda_device)
        xv = rx[offx:].view(T, ldx)[:, :K]
        xv.copy_(x)
        ry, ro = (torch.full((T * ld + off,), 7.0, dtype=BF, device=cuda_device) for _ in range(2))
        yv, ov = ry[off:].view(T, ld)[:, :N], ro[off:].view(T, ld)
        yv.copy_(y)
        got = device_ops.low_rank_add(yv, xv, a, b, adapter, scale, out=ov[:, :N])
        if offx % 8 == 0:
            assert torch.equal(got, want)
        else:
            _check(got, *args)  # unaligned rows: the token kernel, which does not round h
        assert bool((ov[:, N:] == 7.0).all()) and bool((ro[:off] == 7.0).all())


def test_no_adapter_none_of_a_tile_and_nan(cuda_device):
    from baidu_cti_grab_b200 import device_ops

    for T in (40, 400, 20000):
        y, x, a, b, adapter, scale = (t.to(cuda_device) for t in _inputs(T, 64, 80, 16, 5, HF, 10, 2))
        none = torch.full_like(adapter, -1)
        assert torch.equal(device_ops.low_rank_add(y, x, a, b, none, scale), y)
        none[::2] = 5  # past the bank
        assert torch.equal(device_ops.low_rank_add(y, x, a, b, none, scale), y)
        clean = device_ops.low_rank_add(y, x, a, b, adapter, scale)
        bad = x.clone()
        bad[3] = float("nan")
        a2 = a.clone()
        a2[4] = float("inf")  # an adapter that is not sound reaches its own tokens only
        adapter[3] = 0
        got = device_ops.low_rank_add(y, bad, a2, b, adapter, scale)
        b2 = b.clone()
        b2[4] = float("nan")
        b2[4, ::3] = float("inf")
        sick = device_ops.low_rank_add(y, x, a, b2, adapter, scale)
        well = (adapter != 4) & (torch.arange(T, device=cuda_device) != 3)
        # those of the others that shared a product with it are summed again, in another order: each within the
        # rank's 16 rounded products of the other, then half a step of either
        assert bool(sick[well].isfinite().all())
        step = torch.finfo(HF).eps * clean[well].double().abs() + 16 * 2.0 ** -22
        assert bool(((sick[well].double() - clean[well].double()).abs() <= step).all())
        assert bool((~sick[adapter == 4].isfinite()).any(-1).all())
        rows = adapter != 4
        rows[3] = False
        assert torch.equal(got[rows], clean[rows])
        assert bool(got[3].isnan().all())
    y0 = device_ops.low_rank_add(y[:0], x[:0], a, b, adapter[:0], scale)
    assert y0.shape == (0, 80)


@pytest.mark.parametrize("T,K,N,rank,R,dtype,run", [
    (1024, 512, 512, 16, 5, BF, 30),        # the last that is taken token by token: 2^24 products
    (1025, 512, 512, 16, 5, BF, 30),        # and tiles from there on
    (1024, 512, 520, 16, 5, BF, 30),
    (97, 14336, 512, 32, 3, BF, 1),         # few tokens, many products: tiles
    (1025, 8, 16, 8, 2, HF, 10),
    (1409, 72, 200, 8, 7, BF, 9),
    (1100, 200, 100, 64, 3, BF, 50),
    (1100, 200, 101, 24, 5, HF, 20),
    (1026, 1000, 1544, 8, 24, HF, 7),
    (1100, 512, 640, 40, 9, BF, 3),
    (1152, 512, 512, 16, 300, BF, 1),       # every row of a tile its own adapter
    (10000, 512, 1536, 16, 32, BF, 1),      # above half of the SMs in tiles: still H and out apart
    (10001, 1000, 200, 32, 6, HF, 40),
    (18900, 256, 192, 8, 11, BF, 60),
])
def test_tiles_above_the_token_kernels_share(cuda_device, T, K, N, rank, R, dtype, run):
    test_against_float64(cuda_device, T, K, N, rank, R, dtype, run)


@pytest.mark.parametrize("T,rank", [(1500, 16), (1500, 64), (12000, 8)])
def test_tiles_apart_strides_none_and_what_is_not_finite(cuda_device, T, rank):
    """H and out apart: rows at odd places, tokens without an adapter, adapters that are not sound."""
    from baidu_cti_grab_b200 import _lib, device_ops

    K, N = 640, 200
    args = _inputs(T, K, N, rank, 6, BF, 12, T + rank)
    y, x, a, b, adapter, scale = (t.to(cuda_device) for t in args)
    assert _lib.load().rb_low_rank_workspace_size(T, K, N, rank) > 0
    want = device_ops.low_rank_add(y, x, a, b, adapter, scale)
    _check(want, *args)
    for ldx, ld, off in ((K + 8, N + 8, 8), (K + 16, N + 3, 1)):
        xv = torch.zeros(T, ldx, dtype=BF, device=cuda_device)[:, :K]
        xv.copy_(x)
        ry, ro = (torch.full((T * ld + off,), 7.0, dtype=BF, device=cuda_device) for _ in range(2))
        yv, ov = ry[off:].view(T, ld)[:, :N], ro[off:].view(T, ld)
        yv.copy_(y)
        assert torch.equal(device_ops.low_rank_add(yv, xv, a, b, adapter, scale, out=ov[:, :N]), want)
        assert bool((ov[:, N:] == 7.0).all()) and bool((ro[:off] == 7.0).all())
    none = torch.full_like(adapter, -1)
    none[::2] = 6  # past the bank
    assert torch.equal(device_ops.low_rank_add(y, x, a, b, none, scale), y)
    a2, b2 = a.clone(), b.clone()
    a2[4] = float("inf")
    b2[4] = float("nan")
    rows = adapter != 4
    assert torch.equal(device_ops.low_rank_add(y, x, a2, b, adapter, scale)[rows], want[rows])
    sick = device_ops.low_rank_add(y, x, a, b2, adapter, scale)
    assert bool(sick[rows].isfinite().all()) and bool((~sick[~rows].isfinite()).all())


@pytest.mark.parametrize("T", [30, 3000, 20000])
def test_out_over_another_input_is_refused(cuda_device, T):
    from baidu_cti_grab_b200 import device_ops

    y, x, a, b, adapter, scale = (t.to(cuda_device) for t in _inputs(T, 64, 64, 8, 3, BF, 5, 1))
    rows = torch.zeros(T + 1, 160, dtype=BF, device=cuda_device)
    yv, xv, ov = rows[:T, :64], rows[:T, 64:128], rows[1:, :64]
    yv.copy_(y)
    xv.copy_(x)
    before = rows.clone()
    for bad in (ov, xv, rows[:T, 96:160], rows[:T, 8:72], rows.view(-1)[: T * 64].view(T, 64)):
        with pytest.raises(ValueError, match="overlap"):
            device_ops.low_rank_add(yv, xv, a, b, adapter, scale, out=bad)
    assert torch.equal(rows, before)
    want = device_ops.low_rank_add(y, x, a, b, adapter, scale)
    assert torch.equal(device_ops.low_rank_add(yv, xv, a, b, adapter, scale, out=yv), want)  # beside x in one buffer
    assert torch.equal(xv, x)


def test_bank_streams_and_graphs(cuda_device):
    from baidu_cti_grab_b200 import adapters, device_ops

    gen = torch.Generator().manual_seed(3)
    parts = [((torch.randn(r, 256, generator=gen) / 16).to(BF), (torch.randn(320, r, generator=gen) / 4).to(BF), 0.5 + i)
             for i, r in enumerate((8, 16, 4))]
    bank = adapters.AdapterBank.stack(parts).to(cuda_device)
    assert bank.a.shape == (3, 16, 256) and bank.to(torch.bfloat16).scale.dtype == torch.float32
    offsets = torch.tensor([0, 100, 100, 350, 700], device=cuda_device)
    who = adapters.AdapterBank.per_token(torch.tensor([2, 0, -1, 1], device=cuda_device), offsets, 700)
    y, x = (torch.randn(700, n, generator=gen).to(BF).to(cuda_device) for n in (320, 256))
    got = bank(y, x, who)
    _check(got, y, x, bank.a, bank.b, who, bank.scale)
    assert torch.equal(bank(y.view(7, 100, 320), x.view(7, 100, 256), who.view(7, 100)).view(700, 320), got)
    with pytest.raises(RuntimeError):
        device_ops.low_rank_add(y, x.clone().requires_grad_(), bank.a, bank.b, who)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = bank(y, x, who)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, got)
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    held = []
    for g in graphs:
        with torch.cuda.graph(g):
            held.append(bank(y, x, who))
    for g in graphs * 2:
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(h, got) for h in held)


# tiles: fused (19k and more; one tile of one chunk), H and out apart (with and without a split of K)
H_SHAPES = [
    # T, K, N, rank, R, run
    (60, 64, 128, 16, 5, 3),        # token by token
    (1100, 64, 64, 16, 5, 40),
    (1100, 64, 256, 8, 5, 40),
    (1101, 640, 200, 24, 9, 7),
    (1500, 1024, 264, 40, 7, 5),
    (1300, 128, 520, 64, 4, 30),
    (1026, 1000, 1544, 8, 24, 7),
    (19500, 64, 136, 8, 20, 9),
    (19500, 128, 72, 24, 9, 2),
    (19501, 64, 101, 48, 5, 30),
    (20000, 192, 128, 64, 3, 50),
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T,K,N,rank,R,run", H_SHAPES)
def test_h_keeps_more_bits_than_the_type(cuda_device, T, K, N, rank, R, run, dtype):
    """One nonzero in a row of x: h is a product of two values of the type (16 or 22 bits, exact in fp32).  B passes h on and y
    takes h's leading bits off, so what is left is the second half of h: exact in the type, and in every sum on the way."""
    from baidu_cti_grab_b200 import device_ops

    gen = torch.Generator().manual_seed(T + rank)
    _, _, a, _, adapter, _ = _inputs(T, K, N, rank, R, dtype, run, T)
    x = torch.zeros(T, K, dtype=dtype)
    at = torch.randint(0, K, (T,), generator=gen)
    # magnitudes of 4 to 8: the products' last bits are far above fp16's subnormals
    def some(*shape):
        sign = torch.randint(0, 2, shape, generator=gen) * 2.0 - 1.0
        return (sign * (4 + 4 * torch.rand(*shape, generator=gen))).to(dtype)

    x[torch.arange(T), at] = some(T)
    a = some(R, rank, K)
    b = torch.zeros(R, N, rank, dtype=dtype)
    b[:, torch.arange(N), torch.arange(N) % rank] = torch.where(torch.arange(N) // rank % 2 == 0, 1.0, -1.0).to(dtype)
    own = adapter.clamp(min=0)
    h = a[own, :, at].double() * x.double().gather(1, at[:, None])
    passed = (b[own[0]].double() @ h.t()).t()  # B is the same in every adapter
    y = (-passed).to(dtype)
    want = torch.where((adapter >= 0)[:, None], y.double() + passed, y.double())
    assert torch.equal(want.to(dtype).double(), want)
    got = device_ops.low_rank_add(*(t.to(cuda_device) for t in (y, x, a, b, adapter)))
    assert torch.equal(got.double().cpu(), want)
    assert device_ops.device_error() == 0


def _check_close(got, y, x, a, b, adapter, scale):
    """The bound above with h not rounded to the type, but held as two of its values: off by 2^-22 of it and, its row brought
    to 2^14 .. 2^15 before, by the subnormals' half step 2^-25, 2^-39 of the row's largest.  Sums on the tensor cores may
    truncate: a whole step 2^-23 an addition."""
    dev = got.device
    y, x, a, b, adapter, scale = (t.to(dev) for t in (y, x, a, b, adapter, scale))
    rank, K = a.shape[1:]
    fi = torch.finfo(y.dtype)
    tiny = fi.smallest_normal * fi.eps / 2
    for i in range(a.shape[0]):
        t = (adapter == i).nonzero()[:, 0]
        xi, ai, bi, s = x[t].double(), a[i].double(), b[i].double(), scale[i].double()
        h = xi @ ai.t()
        want = y[t].double() + s * (h @ bi.t())
        off = 2.0 ** -22 * h.abs() + 2.0 ** -39 * h.abs().amax(-1, keepdim=True) + (K + rank) * 2.0 ** -23 * (xi.abs() @ ai.abs().t())
        limit = 1.01 * s.abs() * (off @ bi.abs().t()) + 2.0 ** -23 * y[t].double().abs() + fi.eps / 2 * want.abs() + tiny
        over = (got[t].double() - want).abs() - limit
        assert bool((over <= 0).all()), (i, float(over.max()), int((over > 0).sum()), int((~got[t].isfinite()).sum()))


@pytest.mark.parametrize("grow,scale", [(4000.0, 1e-6), (2.0 ** -14, 1000.0)])
@pytest.mark.parametrize("T,K,N,rank,R,run", H_SHAPES)
def test_fp16_h_outside_the_type(cuda_device, T, K, N, rank, R, run, grow, scale):
    """h above fp16's 65504 or among its subnormals, under an adapter scale that brings the sum back."""
    from baidu_cti_grab_b200 import device_ops

    y, x, a, b, adapter, _ = _inputs(T, K, N, rank, R, HF, run, T + 1)
    x = (x.float().clamp(-4, 4) * grow).to(HF)
    if grow > 1:
        a = (a.float() * 100).to(HF)
        assert float((x.float() @ a[0].float().t()).abs().max()) > 2e5
    else:
        a = (a.float() * 2.0 ** -7).to(HF)
        y.zero_()
        assert float((x.float() @ a[0].float().t()).abs().max()) < 2e-5
    s = torch.full((R,), scale)
    args = tuple(t.to(cuda_device) for t in (y, x, a, b, adapter, s))
    got = device_ops.low_rank_add(*args)
    _check_close(got, *args)
    place = args[0].clone()
    device_ops.low_rank_add(place, *args[1:], out=place)
    assert torch.equal(place, got)


@pytest.mark.parametrize("T", [1500, 20000])
def test_infinite_own_b_under_an_exact_h(cuda_device, T):
    """h without a second half (powers of two): an infinity in the token's own B times that zero is no NaN in the result."""
    from baidu_cti_grab_b200 import device_ops

    for dtype in (BF, HF):
        y, x, a, b, adapter, scale = _inputs(T, 64, 200, 16, 6, dtype, 12, T)
        x.zero_()
        x[:, 5] = 2.0
        a = torch.where(a < 0, -0.5, 0.5).to(dtype)
        b[4, ::3, 2] = float("inf")
        args = tuple(t.to(cuda_device) for t in (y, x, a, b, adapter, scale))
        got = device_ops.low_rank_add(*args)
        rows = args[4] == 4
        sign = torch.sign(args[2][4, 2, 5].float())
        assert bool((got[rows][:, ::3].float() == sign * float("inf")).all())
        keep = torch.ones(200, dtype=torch.bool, device=cuda_device)
        keep[::3] = False
        assert bool(got[rows][:, keep].isfinite().all()) and bool(got[~rows].isfinite().all())


@pytest.mark.parametrize("T,K", [(60, 64), (1100, 64), (1500, 640), (20000, 64)])
@pytest.mark.parametrize("N", [1, 7, 97, 101, 127])
def test_odd_widths_in_padded_rows(cuda_device, T, K, N):
    """Rows on 16 bytes whose last columns are no whole 16 bytes: what follows them is neither read into them nor written."""
    from baidu_cti_grab_b200 import device_ops

    args = _inputs(T, K, N, 16, 6, BF, 12, N)
    y, x, a, b, adapter, scale = (t.to(cuda_device) for t in args)
    ld = (N + 8) // 8 * 8
    ry, ro = (torch.full((T, ld), v, dtype=BF, device=cuda_device) for v in (float("nan"), 7.0))
    ry[:, :N].copy_(y)
    device_ops.low_rank_add(ry[:, :N], x, a, b, adapter, scale, out=ro[:, :N])
    _check(ro[:, :N], *args)
    assert bool((ro[:, N:] == 7.0).all())
    ry[:, N:] = 7.0
    device_ops.low_rank_add(ry[:, :N], x, a, b, adapter, scale, out=ry[:, :N])
    assert torch.equal(ry, ro)


@pytest.mark.parametrize("shapes", [((1500, 640), (12000, 512)), ((20000, 128), (1500, 640))])
def test_tiles_on_two_streams_and_in_graphs(cuda_device, shapes):
    """Two calls at once, each in one kernel or in two of which the second starts early, eager and replayed in any order."""
    from baidu_cti_grab_b200 import device_ops

    sets = [[t.to(cuda_device) for t in _inputs(T, K, 200, 16, 6, BF, 12, T)] for T, K in shapes]
    want = [device_ops.low_rank_add(*s) for s in sets]
    for s, w in zip(sets, want):
        _check(w, *s)
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(device_ops.low_rank_add(*sets[i]))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in (0, 1) for g in got[i])
    graphs, held = [torch.cuda.CUDAGraph() for _ in sets], []
    for g, s in zip(graphs, sets):
        with torch.cuda.graph(g):
            # the second call reads what the first wrote
            one = device_ops.low_rank_add(*s)
            held.append((one, device_ops.low_rank_add(one, *s[1:])))
    twice = [device_ops.low_rank_add(w, *s[1:]) for w, s in zip(want, sets)]
    for order in ((0, 1), (1, 0), (0, 1)):
        for t in held:
            t[0].zero_(), t[1].zero_()
        torch.cuda.synchronize()
        for i in order:
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in order:
            assert torch.equal(held[i][0], want[i]) and torch.equal(held[i][1], twice[i])
    assert device_ops.device_error() == 0
