"""Embedding rows and the table's gradient (rb_embed_rows and its backward forms, embedding.py) on the GPU against the
definition in float64.

Tolerance, u = 2^-24: a looked-up row is one product in fp32, rounded once: half a step of itself (and u for the
product).  A gradient of m ids is a sum of m fp32 terms in some order, off by at most m u of the sum of their magnitudes,
times the scale (u more), rounded once to the type (half a step, or of its smallest subnormal).
"""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24


def _ids(n, V, seed, skew=2.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.rand(n, generator=gen, dtype=torch.float64) ** skew * V).long().clamp(max=max(V - 1, 0))


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def _oracle(grad, ids, V, rows=None, scale=1.0, skip=None):
    """(gradient, its bound before rounding) in float64; rows: each id's row of grad; skip: ids that add nothing."""
    g = grad.double().reshape(-1, grad.shape[-1])
    ids = ids.reshape(-1).long().clamp(0, V - 1)
    rows = torch.arange(len(ids), device=ids.device) if rows is None else rows
    keep = torch.ones_like(ids, dtype=torch.bool) if skip is None else ~skip
    ids, g = ids[keep], g[rows[keep]]
    zero = torch.zeros(V, grad.shape[-1], dtype=torch.float64, device=grad.device)
    count = torch.bincount(ids, minlength=V)[:, None]
    total = zero.index_add(0, ids, g) * scale
    return total, (count + 2) * U * abs(scale) * zero.index_add(0, ids, g.abs()), count[:, 0] > 0


def _close(got, want, bound):
    limit = bound * 1.01 + _half(got.dtype) * want.abs() + _tiny(got.dtype)
    off = (got.double() - want).abs()
    assert bool((off <= limit).all()), (float((off - limit).max()), int((off > limit).sum()))


SIZES = [
    # ids, rows, width, type
    (1, 1, 1, F32),
    (1, 5, 512, BF),
    (28, 2801, 512, BF),
    (300, 7, 40, HF),
    (4096, 100000, 64, BF),
    (4097, 100000, 64, BF),          # one above what a CTA sorts by itself
    (5000, 1, 24, F32),              # one row for all
    (9001, 70000, 100, F32),
    (20000, 300, 513, BF),           # rows off 16 bytes
    (30001, 3, 1100, HF),
    (70000, 1 << 20, 8, BF),
    (270000, 40000, 32, BF),         # above what tiles add up by themselves
    (300000, 17, 48, F32),
]


@pytest.mark.parametrize("n,V,D,dtype", SIZES)
def test_against_float64(cuda_device, n, V, D, dtype):
    from baidu_cti_grab_b200 import device_ops

    gen = torch.Generator(device=cuda_device).manual_seed(n + D)
    table = torch.randn(V, D, device=cuda_device, generator=gen).to(dtype)
    grad = torch.randn(n, D, device=cuda_device, generator=gen).to(dtype)
    ids = _ids(n, V, n).to(cuda_device)
    out = device_ops.embed_rows(table, ids, scale=1.25)
    want = table[ids].double() * 1.25
    _close(out, want, 2 * U * want.abs())
    assert torch.equal(device_ops.embed_rows(table, ids.int()), table[ids])  # a scale of 1 copies
    want, bound, touched = _oracle(grad, ids, V, scale=0.75)
    got = device_ops.embed_rows_backward(grad, ids, V, scale=0.75)
    _close(got, want, bound)
    assert torch.equal(got, device_ops.embed_rows_backward(grad, ids.int(), V, scale=0.75))  # and the same bits again
    where, rows, count = device_ops.embed_rows_backward_sparse(grad, ids, V, scale=0.75)
    m = int(count)
    assert torch.equal(where[:m], touched.nonzero()[:, 0])
    assert torch.equal(rows[:m], got[where[:m]])
    # added to what is there, in fp32; rows that no id names stay
    base = torch.randn(V, D, device=cuda_device, generator=gen)
    total = base.clone()
    assert device_ops.embed_rows_backward(grad, ids, V, scale=0.75, out=total) is total
    _close(total, base.double() + want, bound + U * base.abs())
    assert torch.equal(total[~touched], base[~touched])


@pytest.mark.parametrize("D,step", [(46, 46), (100, 100), (100, 101), (48, 50), (770, 772), (1022, 1022)])
@pytest.mark.parametrize("dtype", [F32, BF, HF])
def test_widths_and_strides_of_fewer_bytes(cuda_device, D, step, dtype):
    """Rows that are whole multiples of 8, 4 or 2 bytes only, by their width or their stride."""
    from baidu_cti_grab_b200 import device_ops

    gen = torch.Generator(device=cuda_device).manual_seed(D)
    n, V = 3000, 500
    table = torch.randn(V, step, device=cuda_device, generator=gen).to(dtype)[:, :D]
    grad = torch.randn(n, step, device=cuda_device, generator=gen).to(dtype)[:, :D]
    ids = _ids(n, V, D).to(cuda_device)
    assert torch.equal(device_ops.embed_rows(table, ids), table[ids])
    want, bound, touched = _oracle(grad, ids, V)
    got = device_ops.embed_rows_backward(grad, ids, V)
    _close(got, want, bound)
    where, rows, count = device_ops.embed_rows_backward_sparse(grad, ids, V)
    m = int(count)
    assert torch.equal(rows[:m], got[where[:m]])
    total = torch.ones(V, step, device=cuda_device)[:, :D]
    device_ops.embed_rows_backward(grad, ids, V, out=total)
    _close(total, want + 1.0, bound + U)


def test_ids_outside_the_table_and_padding(cuda_device):
    """Ids are clamped in both directions; those of the padding row add nothing (clamped ones among them)."""
    from baidu_cti_grab_b200 import device_ops

    V, D = 50, 16
    ids = torch.tensor([[-3, 0, 49], [50, 1 << 40, 7], [7, 0, -1]], device=cuda_device)
    table = torch.randn(V, D, device=cuda_device)
    assert torch.equal(device_ops.embed_rows(table, ids), table[ids.clamp(0, V - 1)])
    grad = torch.randn(3, 3, D, device=cuda_device)
    for padding in (None, 0, 7, 49):
        flat = ids.reshape(-1).clamp(0, V - 1)
        want, bound, touched = _oracle(grad, ids, V, skip=None if padding is None else flat == padding)
        _close(device_ops.embed_rows_backward(grad, ids, V, padding_idx=padding), want, bound)
        where, rows, count = device_ops.embed_rows_backward_sparse(grad, ids, V, padding_idx=padding)
        assert torch.equal(where[:int(count)], touched.nonzero()[:, 0])
        _close(rows[:int(count)], want[touched], bound[touched])
    everything = torch.full((9,), 7, device=cuda_device)
    assert not device_ops.embed_rows_backward(grad.view(9, D), everything, V, padding_idx=7).any()
    assert int(device_ops.embed_rows_backward_sparse(grad.view(9, D), everything, V, padding_idx=7)[2]) == 0


@pytest.mark.parametrize("n,V", [(60, 9), (5001, 3000), (280000, 2000)])
@pytest.mark.parametrize("idx", [torch.int32, torch.int64])
def test_bags(cuda_device, n, V, idx):
    """Empty bags, ids before the first bag and behind the last, bags of one id and of many."""
    from baidu_cti_grab_b200 import device_ops, embedding

    gen = torch.Generator().manual_seed(n)
    B, D = max(n // 3, 4), 40
    inner = torch.randint(2, n - 3, (B - 1,), generator=gen).sort().values
    bags = torch.cat([torch.tensor([2]), inner, torch.tensor([n - 3])])
    bags[B // 2] = bags[B // 2 - 1]  # an empty one for certain
    ids = _ids(n, V, n + 1)
    at = torch.arange(n)
    row = torch.searchsorted(bags, at, right=True) - 1
    skip = (at < 2) | (at >= n - 3) | (ids == 0)
    grad = torch.randn(B, D, generator=gen).to(BF).to(cuda_device)
    args = ids.to(idx).to(cuda_device), bags.to(idx).to(cuda_device)
    want, bound, touched = _oracle(grad, ids.to(cuda_device), V, row.clamp(0, B - 1).to(cuda_device), 1.0, skip.to(cuda_device))
    got = embedding.bag_gradient(grad, *args, V)
    _close(got, want, bound)
    s = embedding.bag_gradient(grad, *args, V, sparse=True)
    m = int(s.count)
    assert torch.equal(s.ids[:m], touched.nonzero()[:, 0]) and torch.equal(s.rows[:m], got[s.ids[:m]])
    none = device_ops.embed_rows_backward(grad[:0], args[0], V, bags=args[1][:1])
    assert not none.any()


def test_gradient_of_pooled_bags(cuda_device):
    """The gradient of rep_gather_pool's rows: the sum over the slots' bags, against torch's own embedding_bag in
    float64 on the same ids."""
    from baidu_cti_grab_b200 import device_ops, embedding

    S, N, V, D = 3, 40, 500, 512
    gen = torch.Generator().manual_seed(2)
    sizes = torch.randint(0, 4, (S, N), generator=gen)
    values = [_ids(int(sizes[s].sum()), V, 10 + s).to(cuda_device) for s in range(S)]
    offsets = [torch.cat([torch.zeros(1, dtype=torch.long), sizes[s].cumsum(0)]).to(cuda_device) for s in range(S)]
    table = torch.randn(V, D, generator=gen).to(BF).to(cuda_device)
    grad = torch.randn(N, S * D, generator=gen).to(BF).to(cuda_device)
    pooled = device_ops.rep_gather_pool(table, values, offsets, list(range(S)), S)
    assert pooled.numel() == N * S * D
    t64 = table.double().requires_grad_()
    out = torch.cat([torch.nn.functional.embedding_bag(v, t64, o[:-1], mode="sum", padding_idx=0) for v, o in zip(values, offsets)], 1)
    out.backward(grad.double())
    starts = torch.tensor([0] + [len(v) for v in values]).cumsum(0)
    bags = torch.cat([o[:-1] + a for o, a in zip(offsets, starts[:-1].tolist())] + [torch.tensor([int(starts[-1])], device=cuda_device)])
    by_slot = grad.view(N, S, D).transpose(0, 1).reshape(S * N, D)
    got = embedding.bag_gradient(by_slot, torch.cat(values), bags, V)
    rows = torch.repeat_interleave(torch.arange(S * N, device=cuda_device), bags.diff())
    ids = torch.cat(values)
    want, bound, _ = _oracle(by_slot, ids, V, rows, 1.0, ids == 0)
    assert torch.allclose(want, t64.grad, rtol=1e-12, atol=1e-12)
    _close(got, want, bound)


def test_rows_and_buffers_that_are_left_alone(cuda_device):
    """Padded rows of grad, table and out; entries behind the count; NaN in a row stays in its own table row."""
    from baidu_cti_grab_b200 import device_ops

    n, V, D = 5000, 700, 64
    ids = _ids(n, V, 3).to(cuda_device)
    grad = torch.randn(n, D, device=cuda_device).to(BF)
    want = device_ops.embed_rows_backward(grad, ids, V)
    for pad, odd in ((8, 0), (3, 0), (0, 1)):
        room = torch.empty(n * (D + pad) + odd, dtype=BF, device=cuda_device)
        view = room[odd:].view(n, D + pad)[:, :D]
        view.copy_(grad)
        assert torch.equal(device_ops.embed_rows_backward(view, ids, V), want)
        table = torch.full((V, D + pad), 7.0, device=cuda_device)
        device_ops.embed_rows_backward(grad, ids, V, out=table[:, :D].zero_())
        assert torch.equal(table[:, :D].to(BF), want) and (pad == 0 or bool((table[:, D:] == 7).all()))
    out = torch.full((n,), -9, device=cuda_device), torch.full((n, D), 5.0, dtype=BF, device=cuda_device)
    where, rows, count = device_ops.embed_rows_backward_sparse(grad, ids, V, out=out)
    m = int(count)
    assert where is out[0] and m < n and bool((where[m:] == -9).all()) and bool((rows[m:] == 5).all())
    bad = grad.clone()
    bad[17] = float("nan")
    got = device_ops.embed_rows_backward(bad, ids, V)
    others = torch.arange(V, device=cuda_device) != ids[17]
    assert torch.equal(got[others], want[others]) and bool(got[ids[17]].isnan().all())
    empty = torch.zeros(0, dtype=torch.long, device=cuda_device)
    assert device_ops.embed_rows(table[:, :D], empty).shape == (0, D)
    assert not device_ops.embed_rows_backward(grad[:0], empty, V).any()
    assert int(device_ops.embed_rows_backward_sparse(grad[:0], empty, V)[2]) == 0
    assert device_ops.embed_rows_backward(grad[:0], empty, 0).shape == (0, D)


def test_streams_and_graphs(cuda_device):
    """Two captured calls of one graph, other ids on replay, and another stream."""
    from baidu_cti_grab_b200 import device_ops

    for n in (900, 9000):
        V, D = 400, 72
        ids, other = _ids(n, V, 1).to(cuda_device), _ids(n, V, 2).to(cuda_device)
        grad = torch.randn(n, D, device=cuda_device)
        held = ids.clone()
        want = [device_ops.embed_rows_backward(grad, i, V) for i in (ids, other)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a = device_ops.embed_rows_backward(grad, held, V)
            b = device_ops.embed_rows_backward_sparse(grad, ids, V)
        for i, w in ((other, want[1]), (ids, want[0])):
            held.copy_(i)
            graph.replay()
            assert torch.equal(a, w)
            m = int(b[2])
            assert torch.equal(b[1][:m], want[0][b[0][:m]])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            c = device_ops.embed_rows_backward(grad, ids, V)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(c, want[0])


def test_module_gradients(cuda_device):
    from baidu_cti_grab_b200 import embedding

    torch.manual_seed(0)
    m = embedding.RowEmbedding(30, 16, scale=4.0, padding_idx=2).to(cuda_device)
    ids = torch.randint(0, 30, (5, 7), device=cuda_device)
    out = m(ids)
    assert torch.equal(out, m.weight[ids] * 4.0)
    g = torch.randn_like(out)
    out.backward(g)
    want, bound, _ = _oracle(g, ids, 30, scale=4.0, skip=ids.reshape(-1) == 2)
    _close(m.weight.grad, want, bound)
    with torch.no_grad():
        assert not m(ids).requires_grad


@pytest.mark.parametrize("out_dtype", [BF, HF])
@pytest.mark.parametrize("dtype,D", [(F32, 100), (BF, 512), (HF, 46), (BF, 7)])
def test_results_of_another_type(cuda_device, dtype, D, out_dtype):
    """Sums added to a bf16 or fp16 tensor (rounded once, from fp32), and touched rows in another type than grad's."""
    from baidu_cti_grab_b200 import device_ops

    n, V = 3000, 700
    gen = torch.Generator(device=cuda_device).manual_seed(D)
    grad = torch.randn(n, D, device=cuda_device, generator=gen).to(dtype)
    ids = _ids(n, V, D).to(cuda_device)
    want, bound, touched = _oracle(grad, ids, V)
    base = torch.randn(V, D, device=cuda_device, generator=gen).to(out_dtype)
    total = base.clone()
    device_ops.embed_rows_backward(grad, ids, V, out=total)
    exact = want + base.double()
    _close(total, exact, bound + U * exact.abs())
    assert torch.equal(total[~touched], base[~touched])
    out = torch.full((n,), -7, dtype=torch.int64, device=cuda_device), torch.full((n, D), 9.0, dtype=out_dtype, device=cuda_device)
    where, rows, count = device_ops.embed_rows_backward_sparse(grad, ids, V, out=out)
    m = int(count)
    assert where is out[0] and rows is out[1] and torch.equal(where[:m], touched.nonzero()[:, 0])
    _close(rows[:m], want[where[:m]], bound[where[:m]])
    assert bool((where[m:] == -7).all()) and bool((rows[m:] == 9.0).all())


@pytest.mark.parametrize("n", [3000, 50_000])
def test_tables_above_2_to_the_24_rows(cuda_device, n):
    """Four passes of the sort: ids that differ in their highest byte alone, and the last rows of the table."""
    from baidu_cti_grab_b200 import device_ops

    V, D = (1 << 24) + 70_000, 8
    gen = torch.Generator().manual_seed(n)
    ids = torch.randint(0, V, (n,), generator=gen)
    ids[::5] = torch.randint(0, 4, (len(ids[::5]),), generator=gen)
    ids[1::5] = (1 << 24) + torch.randint(0, 4, (len(ids[1::5]),), generator=gen)
    ids[2] = V - 1
    ids = ids.to(cuda_device)
    grad = torch.randn(n, D, generator=gen).to(cuda_device)
    distinct, place = torch.unique(ids, return_inverse=True)
    want, bound, _ = _oracle(grad, place, len(distinct))
    where, rows, count = device_ops.embed_rows_backward_sparse(grad, ids, V)
    m = int(count)
    assert torch.equal(where[:m], distinct)
    _close(rows[:m], want, bound)
    dense = device_ops.embed_rows_backward(grad, ids, V)
    assert torch.equal(dense[distinct], rows[:m])
    dense[distinct] = 0.0
    assert not dense.any()
