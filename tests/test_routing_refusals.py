"""What rb_route_topk and its Python wrappers refuse, before any device work (no GPU)."""

import pytest

torch = pytest.importorskip("torch")

FAKE = 1 << 20  # an address that no call reaches: every one below fails a host check


def _route(T=4, E=8, k=2, dtype=1, kind=0, groups=1, topk_groups=1, group_top=2, idx_dtype=5, score_dtype=1, ld=None,
           logits=FAKE, idx=FAKE, score=FAKE):
    from baidu_cti_grab_b200 import _lib

    lib = _lib.load()
    rc = lib.rb_route_topk(logits, dtype, E if ld is None else ld, T, E, None, k, kind, groups, topk_groups, group_top, 0,
                           1.0, idx, idx_dtype, score, score_dtype, None, None, None)
    return rc, _lib.last_error()


@pytest.mark.parametrize("bad,word", [
    (dict(T=-1), "negative"), (dict(E=0), "empty"), (dict(E=513), "512"), (dict(k=0), "k must"), (dict(k=33, E=64), "k must"),
    (dict(k=9), "k must"), (dict(groups=3), "groups"), (dict(groups=0), "groups"), (dict(groups=4, topk_groups=5), "topk_groups"),
    (dict(groups=4, topk_groups=1, k=3), "k must"), (dict(group_top=3), "group_top"), (dict(kind=2), "score function"),
    (dict(idx_dtype=0), "idx"), (dict(dtype=4), "fp32"), (dict(score_dtype=3), "fp32"), (dict(ld=7), "leading"),
    (dict(logits=None), "null"), (dict(idx=None), "null"), (dict(score=None), "null")])
def test_route_topk_refuses_on_the_host(bad, word):
    from baidu_cti_grab_b200 import _lib

    rc, msg = _route(**bad)
    assert rc in (_lib.RB_ERR_VALUE, _lib.RB_ERR_UNSUPPORTED) and word in msg, (rc, msg)


def test_route_backward_refuses_on_the_host():
    from baidu_cti_grab_b200 import _lib

    lib = _lib.load()

    def call(T=4, E=8, k=2, dtype=1, kind=0, ld=8, logits=FAKE, out=FAKE, idx=FAKE, idx_dtype=5, gdt=1):
        return lib.rb_route_topk_backward(logits, dtype, ld, T, E, idx, idx_dtype, k, FAKE, gdt, None, 0, kind, 0, 1.0, out,
                                          dtype, None)

    for bad in (dict(T=-1), dict(E=0), dict(E=600, ld=600), dict(k=0), dict(k=9), dict(kind=7), dict(ld=3), dict(logits=None),
                dict(out=None), dict(idx=None), dict(idx_dtype=1), dict(dtype=3), dict(gdt=4)):
        assert call(**bad) in (_lib.RB_ERR_VALUE, _lib.RB_ERR_UNSUPPORTED), bad


def test_cpu_tensors_are_refused():
    from baidu_cti_grab_b200 import device_ops, routing

    with pytest.raises(RuntimeError):
        device_ops.route_topk(torch.zeros(3, 8), 2)
    with pytest.raises(RuntimeError):
        routing.route_topk(torch.zeros(3, 8, requires_grad=True), 2)
    with pytest.raises(RuntimeError):
        device_ops.route_topk_backward(torch.zeros(3, 8), torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2))
    with pytest.raises(ValueError):
        routing.TopKRouter(16, 8, 2).update_balance(torch.zeros(8))


@pytest.mark.parametrize("lead", [(0,), (0, 5), (3, 0), (2, 4), ()])
def test_router_keeps_the_leading_shape(monkeypatch, lead):
    """An empty batch too: its shapes do not follow from the number of values."""
    from baidu_cti_grab_b200 import routing

    def choose(logits, k, **_):
        T, E = logits.shape
        return routing.Routing(torch.zeros(T, k, dtype=torch.int64), torch.zeros(T, k), torch.zeros(T, E), None)

    monkeypatch.setattr(routing, "route_topk", choose)
    idx, score, probs = routing.TopKRouter(16, 8, 2)(torch.zeros(*lead, 16))
    assert idx.shape == score.shape == (*lead, 2) and probs.shape == (*lead, 8)
