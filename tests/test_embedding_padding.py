"""The padding row of embedding.py: given from the table's end, and refused in the forward call where it is none of its rows."""

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture
def seen(monkeypatch):
    from baidu_cti_grab_b200 import device_ops

    given = []
    monkeypatch.setattr(device_ops, "embed_rows", lambda table, ids, scale=1.0: table[ids] * scale)

    def dense(grad, ids, rows, padding_idx=None, **how):
        given.append(padding_idx)
        return torch.zeros(rows, grad.shape[-1])

    def sparse(grad, ids, rows, padding_idx=None, **how):
        given.append(padding_idx)
        return ids, grad, ids[:1]

    monkeypatch.setattr(device_ops, "embed_rows_backward", dense)
    monkeypatch.setattr(device_ops, "embed_rows_backward_sparse", sparse)
    return given


@pytest.mark.parametrize("padding,row", [(None, None), (0, 0), (4, 4), (-1, 4), (-5, 0)])
def test_rows_from_the_end(seen, padding, row):
    from baidu_cti_grab_b200 import embedding

    ids = torch.tensor([1, 4, 4])
    table = torch.ones(5, 8, requires_grad=True)
    embedding.embed(table, ids, padding_idx=padding).sum().backward()
    layer = embedding.RowEmbedding(5, 8, padding_idx=padding)
    assert layer.padding_idx == row and (row is None or not layer.weight[row].any())
    layer(ids).sum().backward()
    embedding.bag_gradient(torch.ones(1, 8), ids, torch.tensor([0, 3]), 5, padding_idx=padding)
    embedding.bag_gradient(torch.ones(1, 8), ids, torch.tensor([0, 3]), 5, padding_idx=padding, sparse=True)
    assert seen == [row] * 4


@pytest.mark.parametrize("padding", [5, -6])
def test_no_row_of_the_table(seen, padding):
    from baidu_cti_grab_b200 import embedding

    ids, table = torch.tensor([1]), torch.ones(5, 8)
    for call in (lambda: embedding.embed(table.requires_grad_(), ids, padding_idx=padding),
                 lambda: embedding.embed(table.detach(), ids, padding_idx=padding),
                 lambda: embedding.RowEmbedding(5, 8, padding_idx=padding),
                 lambda: embedding.bag_gradient(torch.ones(1, 8), ids, torch.tensor([0, 1]), 5, padding_idx=padding)):
        with pytest.raises(ValueError):
            call()
    assert seen == []
