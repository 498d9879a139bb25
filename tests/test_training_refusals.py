"""What the embedding's gradient and the clipping of gradients refuse, before any kernel runs (no GPU needed)."""

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture
def calls(monkeypatch):
    from baidu_cti_grab_b200 import device_ops

    names = []
    monkeypatch.setattr(device_ops, "_device_of", lambda name, first, *others: first.device)
    monkeypatch.setattr(device_ops, "_plan_bytes", lambda *a: 0)
    monkeypatch.setattr(device_ops, "_call_on", lambda dev, name, *a: names.append(name))
    return names


IDS = torch.tensor([1, 2, 2])


def test_embedding_arguments(calls):
    from baidu_cti_grab_b200 import device_ops as d

    table, grad = torch.zeros(5, 8), torch.zeros(3, 8)
    bags = torch.tensor([0, 2, 3])
    assert d.embed_rows(table, IDS.view(1, 3)).shape == (1, 3, 8)
    assert d.embed_rows_backward(grad, IDS, 5, padding_idx=4).shape == (5, 8)
    d.embed_rows_backward(grad[:2], IDS, 5, bags=bags.int(), out=torch.zeros(5, 8, dtype=torch.bfloat16))
    ids, rows, count = d.embed_rows_backward_sparse(grad[:2], IDS, 5, bags=bags)
    assert ids.shape == (3,) and rows.shape == (3, 8) and count.shape == (1,)
    assert calls == ["rb_embed_rows", "rb_embed_rows_backward", "rb_embed_rows_backward", "rb_embed_rows_backward_sparse"]
    for bad in (
        lambda: d.embed_rows(table.double(), IDS),
        lambda: d.embed_rows(table[0], IDS),
        lambda: d.embed_rows(table, IDS.float()),
        lambda: d.embed_rows_backward(grad.long(), IDS, 5),
        lambda: d.embed_rows_backward(grad[:2], IDS, 5),
        lambda: d.embed_rows_backward(grad, IDS.short(), 5),
        lambda: d.embed_rows_backward(grad, IDS, -1),
        lambda: d.embed_rows_backward(grad, IDS, 5, bags=bags),
        lambda: d.embed_rows_backward(grad[:2], IDS, 5, bags=bags.float()),
        lambda: d.embed_rows_backward(grad[:2], IDS.view(1, 3), 5, bags=bags),
        lambda: d.embed_rows_backward(grad, IDS, 5, padding_idx=5),
        lambda: d.embed_rows_backward(grad, IDS, 5, padding_idx=-1),
        lambda: d.embed_rows_backward(grad, IDS, 5, out=torch.zeros(4, 8)),
        lambda: d.embed_rows_backward(grad, IDS, 5, out=torch.zeros(8, 5).t()),
        lambda: d.embed_rows_backward(grad, IDS, 5, out=torch.zeros(5, 8, dtype=torch.int32)),
        lambda: d.embed_rows_backward_sparse(grad, IDS, 5, out=(torch.zeros(2, dtype=torch.int64), torch.zeros(3, 8))),
        lambda: d.embed_rows_backward_sparse(grad, IDS, 5, out=(torch.zeros(3, dtype=torch.int32), torch.zeros(3, 8))),
        lambda: d.embed_rows_backward_sparse(grad, IDS, 5, out=(torch.zeros(3, dtype=torch.int64), torch.zeros(3, 7))),
    ):
        with pytest.raises(ValueError):
            bad()
    assert len(calls) == 4


def test_cpu_tensors_are_refused():
    from baidu_cti_grab_b200 import device_ops as d

    for call in (lambda: d.embed_rows(torch.zeros(5, 8), IDS), lambda: d.embed_rows_backward(torch.zeros(3, 8), IDS, 5),
                 lambda: d.grad_norm([torch.zeros(3)]), lambda: d.clip_grads([torch.zeros(3)], 1.0)):
        with pytest.raises(RuntimeError):
            call()


def test_clipping_arguments():
    from baidu_cti_grab_b200 import device_ops as d

    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            d.clip_grads([torch.zeros(3)], bad)
    for empty in ([], ()):
        with pytest.raises(ValueError):
            d.grad_norm(empty)
    for pair in ((torch.zeros(3, 2).t(), torch.zeros(1, dtype=torch.int32)), (torch.zeros(3), torch.zeros(1, dtype=torch.int32)),
                 (torch.zeros(3, 2), torch.zeros(1)), (torch.zeros(3, 2), torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(ValueError):
            d.grad_norm([pair])


def test_c_entries_refuse():
    """Bad sizes and null operands come back as a status with a message, without a device."""
    import ctypes

    from baidu_cti_grab_b200 import _lib as L

    lib = L.load()
    one = ctypes.c_void_p(1 << 20)  # never read: the arguments are refused first

    def rows(V=5, D=8, n=3, dtype=L.RB_F32, idx=L.RB_I64, ld=8, table=one):
        return lib.rb_embed_rows(table, dtype, ld, V, D, one, idx, n, 1.0, one, 8, None)

    def back(V=5, D=8, n=3, dtype=L.RB_F32, idx=L.RB_I64, ld=8, bags=None, n_bags=0, ws=0, out=one):
        return lib.rb_embed_rows_backward(one, dtype, 8, D, one, idx, n, V, bags, n_bags, -1, 1.0, 0, one, ws, out, L.RB_F32, ld,
                                          None)

    def clip(n=1, values=3, dtype=L.RB_F32, scale=1.0, most=1.0, ws=1 << 20, norm=one, counted=None, width=1):
        ptr = (ctypes.c_void_p * 1)(1 << 20)
        return lib.rb_clip_grads(ptr, ptr, (ctypes.c_int64 * 1)(values), (ctypes.c_int * 1)(dtype), counted,
                                 (ctypes.c_int64 * 1)(width), n, scale, most, one, ws, norm, None)

    refused = (L.RB_ERR_VALUE, L.RB_ERR_UNSUPPORTED)
    for call in (lambda: rows(V=-1), lambda: rows(V=0), lambda: rows(D=0), lambda: rows(dtype=L.RB_I8), lambda: rows(idx=L.RB_F32),
                 lambda: rows(ld=7), lambda: rows(table=None), lambda: rows(V=1 << 31), lambda: rows(n=1 << 31),
                 lambda: back(n=-1), lambda: back(ld=7), lambda: back(out=None), lambda: back(ws=16),
                 lambda: back(bags=one, n_bags=-1), lambda: back(dtype=L.RB_I64),
                 lambda: clip(n=-1), lambda: clip(values=-1), lambda: clip(dtype=L.RB_I32), lambda: clip(scale=-1.0),
                 lambda: clip(scale=float("nan")), lambda: clip(most=float("nan")), lambda: clip(ws=8), lambda: clip(norm=None),
                 lambda: clip(counted=(ctypes.c_void_p * 1)(1 << 20), width=0)):
        assert call() in refused
        assert L.last_error()
    assert lib.rb_embed_rows_backward_workspace_size(-1, 8) == -1
    assert lib.rb_embed_rows_backward_workspace_size(0, 8) == 0
    assert lib.rb_grad_norm_workspace_size(-1) == -1


def test_what_a_kernel_writes_counts_as_modified(calls):
    """Autograd refuses a backward pass over a saved tensor that was written since: by torch, or by these calls."""
    from baidu_cti_grab_b200 import device_ops as d

    out, grad = torch.zeros(5, 8, dtype=torch.bfloat16), torch.zeros(3, 8)
    d.embed_rows_backward(grad, IDS, 5, out=out)
    assert out._version == 1
    pair = torch.zeros(3, dtype=torch.int64), torch.zeros(3, 8)
    d.embed_rows_backward_sparse(grad, IDS, 5, out=pair)
    assert [t._version for t in pair] == [1, 1]
