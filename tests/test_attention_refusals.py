"""What attention within segments refuses, before any kernel runs (no GPU needed)."""

import pytest

torch = pytest.importorskip("torch")

BF = torch.bfloat16


@pytest.fixture
def args(monkeypatch):
    from baidu_cti_grab_b200 import device_ops

    monkeypatch.setattr(device_ops, "_device_of", lambda name, first, *others: first.device)
    monkeypatch.setattr(device_ops, "_plan_bytes", lambda *a: 0)
    calls = []
    monkeypatch.setattr(device_ops, "_call_on", lambda dev, name, *a: calls.append(name))
    q, k, v = torch.zeros(10, 4, 16, dtype=BF), torch.zeros(10, 2, 16, dtype=BF), torch.zeros(10, 2, 16, dtype=BF)
    return dict(q=q, k=k, v=v, offsets=torch.tensor([0, 4, 10])), calls


def _call(a, **more):
    from baidu_cti_grab_b200 import device_ops

    a = {**a, **more}
    return device_ops.segment_attention(a.pop("q"), a.pop("k"), a.pop("v"), a.pop("offsets"), **a)


def test_what_is_taken(args):
    a, calls = args
    _call(a)
    _call(a, prefix=torch.tensor([1, 2], dtype=torch.int32), slopes=torch.zeros(4), cap=3.0, scale=0.1, causal=False)
    _call(a, k=torch.zeros(30, 1, 16, dtype=BF), v=torch.zeros(30, 1, 16, dtype=BF), k_offsets=torch.tensor([0, 20, 30]))
    assert calls == ["rb_segment_attention"] * 3


@pytest.mark.parametrize("more", [
    dict(q=torch.zeros(10, 64, dtype=BF)),
    dict(q=torch.zeros(10, 4, 16)),
    dict(q=torch.zeros(10, 4, 16, dtype=torch.float16)),
    dict(q=torch.zeros(10, 3, 16, dtype=BF)),
    dict(q=torch.zeros(10, 4, 8, dtype=BF)),
    dict(q=torch.zeros(9, 4, 16, dtype=BF)),
    dict(v=torch.zeros(10, 2, 8, dtype=BF)),
    dict(offsets=torch.tensor([0.0, 10.0])),
    dict(offsets=torch.tensor([[0, 10]])),
    dict(offsets=torch.zeros(0, dtype=torch.int64)),
    dict(k_offsets=torch.tensor([0, 10])),
    dict(k_offsets=torch.tensor([0, 4, 10], dtype=torch.int32)),
    dict(prefix=torch.tensor([1])),
    dict(prefix=torch.tensor([1.0, 2.0])),
    dict(slopes=torch.zeros(2)),
    dict(slopes=torch.zeros(4, dtype=BF)),
])
def test_what_is_refused(args, more):
    a, calls = args
    with pytest.raises(ValueError):
        _call(a, **more)
    assert calls == []


@pytest.mark.parametrize("more", [dict(lse=torch.zeros(10, 4)), dict(lse=torch.zeros(4, 10, dtype=torch.float64)),
                                  dict(grad=torch.zeros(10, 4, 16)), dict(out=torch.zeros(10, 4, 8, dtype=BF))])
def test_backward_refuses(args, more):
    from baidu_cti_grab_b200 import device_ops

    a, calls = args
    t = dict(grad=torch.zeros(10, 4, 16, dtype=BF), out=torch.zeros(10, 4, 16, dtype=BF), lse=torch.zeros(4, 10), **{})
    device_ops.segment_attention_backward(t["grad"], a["q"], a["k"], a["v"], t["out"], t["lse"], a["offsets"])
    t.update(more)
    with pytest.raises(ValueError):
        device_ops.segment_attention_backward(t["grad"], a["q"], a["k"], a["v"], t["out"], t["lse"], a["offsets"])
    assert calls == ["rb_segment_attention_backward"]


def test_c_entry_refuses():
    """Bad sizes and null operands come back as a status with a message, without a device."""
    from baidu_cti_grab_b200 import _lib as L

    lib = L.load()

    def call(Tq=4, Tk=4, H=2, Hk=2, D=64, dtype=L.RB_BF16, idx=L.RB_I32, cap=0.0, scale=1.0, q=None):
        return lib.rb_segment_attention(q, H * D, D, q, Hk * D, D, q, Hk * D, D, dtype, Tq, Tk, H, Hk, D, q, q, None, idx, 1, 1,
                                        None, cap, scale, None, 0, q, None, None)

    for bad in (dict(Tq=-1), dict(H=0), dict(H=3), dict(D=257), dict(dtype=L.RB_F32), dict(idx=L.RB_F32), dict(cap=-1.0),
                dict(cap=float("nan")), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(Tq=1 << 31), {}):
        assert call(**bad) in (L.RB_ERR_VALUE, L.RB_ERR_UNSUPPORTED), bad
        assert L.last_error()
    assert lib.rb_segment_attention_workspace_size(-1, 0, 0, 1, 1, 64) == -1
    assert lib.rb_segment_attention_backward_workspace_size(4, 4, 1, 0, 1, 64) == -1


def test_module_refuses_heads_that_do_not_share():
    from baidu_cti_grab_b200.attention import SegmentAttention

    with pytest.raises(ValueError):
        SegmentAttention(64, 4, 3)
    with pytest.raises(ValueError):
        SegmentAttention(65, 4)
    assert SegmentAttention(65, 4, head_dim=16).width == 16
