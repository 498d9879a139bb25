"""The norm of many gradients and the clipping by it (rb_clip_grads, grad_clip.py) on the GPU against float64.

Tolerance, u = 2^-24: a thread's 32 squares are summed in fp32 (each square and each of 10 adds in a row off by u), the
rest is fp64: the sum is within 12 u of itself, the norm within 6 u and its rounding, 7 u.  The factor takes two fp32
operations more and the product with a loss scale one: 10 u; a gradient's product one more, then half a step of its type.
"""

import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24


def _norm(grads, scale=1.0):
    return scale * math.sqrt(sum(float(t.double().square().sum()) for t in grads))


def _check(got, grads, norm, most, scale=1.0):
    f = scale * min(1.0, most / (norm + 1e-6))
    for o, t in zip(got, grads):
        want = t.double() * f
        fi = torch.finfo(t.dtype)
        limit = 11 * U * want.abs() + fi.eps / 2 * want.abs() + fi.smallest_normal * fi.eps / 2
        assert bool(((o.double() - want).abs() <= limit).all())


def _some(shapes, dtypes, device, std=0.1, seed=0):
    gen = torch.Generator(device=device).manual_seed(seed)
    return [(torch.randn(s, device=device, generator=gen) * std).to(dtypes[i % len(dtypes)]) for i, s in enumerate(shapes)]


SHAPES = {
    "one value": [(1,)],
    "scalars and empties": [(), (0,), (3, 0), (5,)],
    "a piece and around it": [(8191,), (8192,), (8193,), (16384,), (7,)],
    "a layer": [(512, 512), (512,), (1024, 512), (1024,), (512, 1024)],
    "odd": [(77, 3), (1001,), (13, 17, 5), (1,), (30001,)],
    "few": [(40,)] * 24,
    "more than few": [(40 + i,) for i in range(25)],
    "many": [(i % 50 + 1,) for i in range(1000)],
    "large": [(3000, 1001), (5000001,)],
}


@pytest.mark.parametrize("which", sorted(SHAPES))
@pytest.mark.parametrize("dtypes", [(BF,), (F32,), (HF, F32, BF)])
def test_against_float64(cuda_device, which, dtypes):
    from baidu_cti_grab_b200 import device_ops

    grads = _some(SHAPES[which], dtypes, cuda_device)
    norm = _norm(grads)
    got = device_ops.grad_norm(grads)
    assert got.shape == () and got.dtype is F32 and abs(float(got) - norm) <= 7 * U * norm
    assert abs(float(device_ops.grad_norm(grads, scale=0.125)) - norm / 8) <= 7 * U * norm / 8
    for most, scale in ((norm * 0.3, 1.0), (norm * 2, 1.0), (0.0, 1.0), (norm * 0.3, 0.5), (norm * 3, 0.5)):
        out = [torch.full_like(t, 3.0) for t in grads]
        n = device_ops.clip_grads(grads, most, out=out, scale=scale)
        assert abs(float(n) - scale * norm) <= 7 * U * scale * norm
        _check(out, grads, scale * norm, most, scale)
        place = [t.clone() for t in grads]
        assert torch.equal(device_ops.clip_grads(place, most, scale=scale), n)  # the same bits again
        assert all(torch.equal(a, b) for a, b in zip(place, out))


def test_values_whose_squares_leave_fp32(cuda_device):
    from baidu_cti_grab_b200 import device_ops

    for up in (1e30, 1e-30, 3e-38, 1e19, 1e-23):
        for dtype in (F32, BF):
            grads = [(t * up).to(dtype) for t in _some([(10000,), (33,)], (F32,), cuda_device, 1.0)]
            norm = _norm(grads)
            assert abs(float(device_ops.grad_norm(grads)) - norm) <= 7 * U * norm + 2.0 ** -149
            if up > 1:
                place = [t.clone() for t in grads]
                device_ops.clip_grads(place, norm / 8)
                _check(place, grads, norm, norm / 8)
    both = torch.tensor([3e30, 4e-30, 1.0], device=cuda_device)
    assert abs(float(device_ops.grad_norm([both])) - 3e30) <= 7 * U * 3e30
    assert float(device_ops.grad_norm([torch.zeros(50, device=cuda_device)])) == 0.0
    top = torch.full((2,), 3e38, device=cuda_device)
    assert float(device_ops.grad_norm([top])) == math.inf  # above fp32: the norm's own type


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_values_that_are_not_finite(cuda_device, bad):
    """As the formula has them: NaN reaches every gradient, an infinite norm takes finite ones to zero."""
    from baidu_cti_grab_b200 import device_ops

    grads = _some([(100,), (9000,)], (BF, F32), cuda_device)
    grads[1][5000] = bad
    n = device_ops.clip_grads(grads, 1.0)
    assert math.isnan(float(n)) if math.isnan(bad) else float(n) == math.inf
    assert bool(grads[0].isnan().all()) if math.isnan(bad) else not grads[0].any()
    assert math.isnan(float(grads[1][5000]))


def test_layouts_offsets_and_rows_that_count(cuda_device):
    from baidu_cti_grab_b200 import device_ops

    base = torch.randn(60, 90, device=cuda_device)
    turned, strided = base.t(), torch.randn(50, 40, device=cuda_device)[:, ::2]
    odd = torch.randn(1001, device=cuda_device).to(BF)[1:]
    images = torch.randn(2, 3, 4, 5, device=cuda_device).contiguous(memory_format=torch.channels_last)
    rows = torch.randn(100, 24, device=cuda_device).to(BF)
    rows[37:] = math.nan  # behind what counts
    grads = [turned, strided, odd, images]
    for count in (0, 1, 37):
        c = torch.tensor([count], dtype=torch.int32, device=cuda_device)
        counted = [*grads, rows[:count]]
        norm = _norm(counted)
        assert abs(float(device_ops.grad_norm([*grads, (rows, c)])) - norm) <= 7 * U * norm
        keep = [t.clone() for t in grads]
        mine = [t.as_strided(t.size(), t.stride()) for t in keep]
        room = strided._base.clone() if strided._base is not None else None
        place = [keep[0], strided.clone() if room is None else room[:, ::2], keep[2], keep[3]]
        r2 = rows.clone()
        device_ops.clip_grads([*place, (r2, c)], norm / 3)
        _check([*place, r2[:count]], counted, norm, norm / 3)
        assert bool(r2[37:].isnan().all()) and len(mine) == 4
        if room is not None:
            assert torch.equal(room[:, 1::2], strided._base[:, 1::2])


def test_streams_graphs_and_training(cuda_device):
    """A captured clipping on replay, another stream, and the call between backward and the optimiser with the touched
    rows of a table beside the parameters."""
    from baidu_cti_grab_b200 import device_ops, embedding, grad_clip

    grads = _some([(1000,), (513, 7)], (BF, F32), cuda_device)
    held = [t.clone() for t in grads]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n = device_ops.clip_grads(held, 0.5)
    for up in (1.0, 4.0):
        now = [(t * up).to(t.dtype) for t in grads]
        for h, t in zip(held, now):
            h.copy_(t)
        graph.replay()
        norm = _norm(now)
        assert abs(float(n) - norm) <= 7 * U * norm
        _check(held, now, norm, 0.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        n2 = device_ops.grad_norm(now)
    torch.cuda.current_stream().wait_stream(side)
    assert abs(float(n2) - norm) <= 7 * U * norm

    layer = torch.nn.Linear(32, 8).to(cuda_device)
    unused = torch.nn.Parameter(torch.zeros(3, device=cuda_device))
    x = torch.randn(20, 32, device=cuda_device)
    layer(x).square().sum().backward()
    ids = torch.randint(0, 50, (20,), device=cuda_device)
    sparse = embedding.SparseRows(*device_ops.embed_rows_backward_sparse(x, ids, 50))
    m = int(sparse.count)
    before = [layer.weight.grad.clone(), layer.bias.grad.clone(), sparse.rows[:m].clone()]
    norm = _norm(before)
    params = [*layer.parameters(), unused]
    assert abs(float(grad_clip.grad_norm(params, sparse=[sparse])) - norm) <= 7 * U * norm
    n = grad_clip.clip_grad_norm(params, 0.1 * norm, sparse=[sparse])
    assert abs(float(n) - norm) <= 7 * U * norm
    _check([layer.weight.grad, layer.bias.grad, sparse.rows[:m]], before, norm, 0.1 * norm)
    assert float(grad_clip.clip_grad_norm([unused], 1.0)) == 0.0


def test_clipped_tensors_count_as_modified(cuda_device):
    """Autograd refuses a backward pass over a saved tensor that was clipped since; the norm alone modifies nothing."""
    from baidu_cti_grab_b200 import device_ops

    w = torch.ones(40, device=cuda_device, requires_grad=True)
    saved = torch.ones(40, device=cuda_device)
    y = (w * saved).sum()
    device_ops.grad_norm([saved])
    assert saved._version == 0
    device_ops.clip_grads([saved], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    out = [torch.empty_like(saved)]
    device_ops.clip_grads([saved], 1.0, out=out)
    assert out[0]._version == 1 and saved._version == 1
    rows, count = torch.ones(6, 4, device=cuda_device), torch.tensor([3], dtype=torch.int32, device=cuda_device)
    device_ops.clip_grads([(rows, count)], 1.0)
    assert rows._version == 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("at", [0, 777, 9000])
def test_zeros_and_what_hides_among_them(cuda_device, dtype, at):
    """Zeros alone are a norm of 0; one value among them is the norm, however small its square, and a NaN is NaN."""
    from baidu_cti_grab_b200 import device_ops

    x = torch.zeros(10_001, dtype=dtype, device=cuda_device)
    assert float(device_ops.grad_norm([x])) == 0.0
    for value in (1e-38, 3e-23, 2.0, -5e30, math.nan):
        x[at] = value
        got, want = float(device_ops.grad_norm([x])), abs(float(x[at]))
        assert (math.isnan(got) and math.isnan(want)) or abs(got - want) <= 2.0 ** -22 * want
