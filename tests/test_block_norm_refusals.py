"""What rb_sandwich_norm and its Python wrappers refuse, before any device work (no GPU)."""

import pytest

torch = pytest.importorskip("torch")

FAKE = 1 << 20  # an address that no call reaches: every one below fails a host check


def _forward(x=FAKE, ldx=512, h=FAKE, ldh=512, dtype=1, N=4, D=512, post=1, w1=FAKE, b1=None, w1t=0, gk=0, gate=None, gt=0, ldg=0,
             act=0, pre=1, w2=None, b2=None, w2t=0, y=FAKE, z=FAKE, stats=None):
    from baidu_cti_grab_b200 import _lib

    lib = _lib.load()
    rc = lib.rb_sandwich_norm(x, ldx, h, ldh, dtype, N, D, post, w1, b1, w1t, 1e-5, gk, gate, gt, ldg, act, 1.0, pre, w2, b2,
                              w2t, 1e-5, y, z, stats, None)
    return rc, _lib.last_error()


@pytest.mark.parametrize("bad,word", [
    (dict(N=-1), "negative"), (dict(D=0), "empty"), (dict(D=8193, ldx=9000, ldh=9000), "wider"), (dict(dtype=4), "rows are"),
    (dict(post=3), "norm kind"), (dict(pre=-1), "norm kind"), (dict(gk=4), "gate kind"), (dict(act=2), "activation"),
    (dict(gk=1), "gate"), (dict(gate=FAKE), "gate"), (dict(gk=3, gate=FAKE, gt=0, ldg=512), "rows' type"),
    (dict(gk=1, gate=FAKE, gt=4), "gate is"), (dict(gk=3, gate=FAKE, gt=1, ldg=100), "leading"), (dict(w1t=3), "weights"),
    (dict(post=0), "without their norm"), (dict(ldx=511), "leading"), (dict(ldh=1), "leading"), (dict(x=None), "null"),
    (dict(h=None), "null"), (dict(y=None), "null"), (dict(z=None), "null"), (dict(stats=FAKE + 4), "misaligned")])
def test_forward_refuses_on_the_host(bad, word):
    from baidu_cti_grab_b200 import _lib

    rc, msg = _forward(**bad)
    assert rc in (_lib.RB_ERR_VALUE, _lib.RB_ERR_UNSUPPORTED) and word in msg, (rc, msg)


def test_backward_refuses_on_the_host():
    from baidu_cti_grab_b200 import _lib

    lib = _lib.load()
    need = lib.rb_sandwich_norm_workspace_size(4, 512, 1)
    assert need > 0 and need % (4 * 512 * 4) == 0
    assert lib.rb_sandwich_norm_workspace_size(4, 8193, 1) == -1 and lib.rb_sandwich_norm_workspace_size(-1, 8, 1) == -1

    def call(dy=FAKE, ldy=512, dz=FAKE, ldz=512, x=FAKE, stats=FAKE, D=512, gk=0, gate=None, pre=1, ws=FAKE, size=need, dx=FAKE,
             dgate=None):
        rc = lib.rb_sandwich_norm_backward(dy, ldy, dz, ldz, x, 512, FAKE, 512, stats, 1, 4, D, 1, None, None, 0, gk, gate, 1, 0, 0,
                                           1.0, pre, None, None, 0, ws, size, dx, FAKE, dgate, None, None, None, None, None)
        return rc, _lib.last_error()

    for bad, word in ((dict(ldy=1), "leading"), (dict(ldz=1), "leading"), (dict(x=None), "null"), (dict(stats=None), "null"),
                      (dict(gk=1, gate=FAKE), "null"), (dict(pre=0), "without its norm"), (dict(ws=None), "null"),
                      (dict(size=need - 1), "workspace"), (dict(dx=None), "null"), (dict(ws=FAKE + 8), "misaligned")):
        rc, msg = call(**bad)
        assert rc in (_lib.RB_ERR_VALUE, _lib.RB_ERR_UNSUPPORTED) and word in msg, (bad, rc, msg)


def test_cpu_tensors_are_refused():
    from baidu_cti_grab_b200 import block_norm, device_ops

    x = torch.zeros(3, 8)
    with pytest.raises(RuntimeError):
        device_ops.sandwich_norm(x, x, post="rms")
    with pytest.raises(RuntimeError):
        block_norm.SandwichNorm(8)(x, x)
    with pytest.raises(RuntimeError):
        device_ops.sandwich_norm_backward(x, None, x, x, torch.zeros(3, 4), post="rms")
