"""What rb_low_rank_add and its Python wrappers refuse, before any device work (no GPU)."""

import pytest

torch = pytest.importorskip("torch")

FAKE = 1 << 20  # an address that no call reaches: every one below fails a host check


def _call(y=FAKE, ldy=512, x=FAKE, ldx=256, dtype=1, T=4, K=256, N=512, a=FAKE, b=FAKE, R=3, rank=16, idx=FAKE, it=5, ws=None,
          size=0, out=FAKE, ldo=512):
    from baidu_cti_grab_b200 import _lib

    lib = _lib.load()
    rc = lib.rb_low_rank_add(y, ldy, x, ldx, dtype, T, K, N, a, b, R, rank, idx, it, None, ws, size, out, ldo, None)
    return rc, _lib.last_error()


@pytest.mark.parametrize("bad,word", [
    (dict(T=-1), "negative"), (dict(K=0), "empty"), (dict(N=0), "empty"), (dict(R=0), "empty"), (dict(rank=0), "empty"),
    (dict(rank=129), "ranks"), (dict(dtype=0), "bf16"), (dict(it=1), "adapter ids"), (dict(T=1 << 29), "tokens"),
    (dict(R=1 << 24), "rows of all"), (dict(ldy=511), "leading"), (dict(ldo=1), "leading"), (dict(ldx=255), "leading"),
    (dict(y=None), "null"), (dict(x=None), "null"), (dict(a=None), "null"), (dict(b=None), "null"), (dict(idx=None), "null"),
    (dict(out=None), "null"), (dict(T=2000), "workspace"), (dict(T=2000, ws=FAKE, size=16), "workspace"),
    (dict(T=2000, ws=FAKE + 4, size=1 << 30), "workspace")])
def test_refuses_on_the_host(bad, word):
    from baidu_cti_grab_b200 import _lib

    rc, msg = _call(**bad)
    assert rc in (_lib.RB_ERR_VALUE, _lib.RB_ERR_UNSUPPORTED) and word in msg, (rc, msg)


def test_workspace_sizes():
    """Few tokens and many tiles need none; tiles that are too few for the SMs hold partial h, fp32."""
    from baidu_cti_grab_b200 import _lib

    size = _lib.load().rb_low_rank_workspace_size
    assert size(96, 512, 512, 16) == 0 and size(100000, 512, 512, 16) == 0 and size(0, 512, 512, 16) == 0
    assert size(4099, 14336, 512, 32) % (4099 * 32 * 4) == 0 and size(4099, 14336, 512, 32) > 0
    assert size(1000, 100, 512, 16) == 0 and size(1000, 512, 512, 12) == 0 and size(1000, 512, 512, 72) == 0
    assert size(-1, 512, 512, 16) == -1 and size(10, 0, 512, 16) == -1 and size(10, 512, 512, 129) == -1


def test_wrappers_refuse():
    from baidu_cti_grab_b200 import adapters, device_ops

    t = torch.zeros(4, 8, dtype=torch.bfloat16)
    a, b = torch.zeros(2, 8, 8, dtype=torch.bfloat16), torch.zeros(2, 8, 8, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        device_ops.low_rank_add(t, t, a, b, torch.zeros(4, dtype=torch.int32))
    with pytest.raises(RuntimeError):
        adapters.AdapterBank(a, b)(t, t, torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError):
        adapters.AdapterBank(a, b[:1])
    with pytest.raises(ValueError):
        adapters.AdapterBank.stack([])


def test_per_token_of_padded_and_empty_requests():
    """Tokens outside every request have no adapter, whatever the batch's length."""
    from baidu_cti_grab_b200.adapters import AdapterBank

    who = torch.tensor([2, 0, -1, 1])
    offsets = torch.tensor([1, 3, 3, 5, 6])
    for dtype in (torch.int64, torch.int32):
        got = AdapterBank.per_token(who, offsets.to(dtype), 9)
        assert got.dtype == torch.int32 and got.tolist() == [-1, 2, 2, -1, -1, 1, -1, -1, -1]
        assert AdapterBank.per_token(who, offsets.to(dtype), 4).tolist() == [-1, 2, 2, -1]
        assert AdapterBank.per_token(who[:0], offsets[:1].to(dtype), 3).tolist() == [-1, -1, -1]
        assert AdapterBank.per_token(who, offsets.to(dtype), 0).shape == (0,)


def test_overlapping_rows_are_seen():
    from baidu_cti_grab_b200.device_ops import _rows_overlap

    g = torch.Generator().manual_seed(0)
    both = [0, 0]
    for _ in range(2000):
        T, wa, wb, lda, same, off = (int(torch.randint(lo, hi, (1,), generator=g))
                                     for lo, hi in ((1, 5), (1, 6), (1, 6), (6, 12), (0, 4), (-40, 41)))
        ldb = lda if same else lda + 1
        buf = torch.zeros(200, dtype=torch.bfloat16)
        a, b = buf.as_strided((T, wa), (lda, 1), 80), buf.as_strided((T, wb), (ldb, 1), 80 + off)
        a.fill_(1)
        shared = bool((b == 1).any())
        said = _rows_overlap(a, lda, b, ldb)
        both[said] += 1
        assert said == shared or (said and lda != ldb and T > 1)
    assert min(both) > 100


@pytest.mark.parametrize("which", ["y", "x", "out", "a"])
def test_inputs_that_ask_for_a_gradient_are_refused(monkeypatch, which):
    """The kernels have no backward: the module refuses what device_ops refuses, and neither drops a gradient."""
    from baidu_cti_grab_b200 import adapters, device_ops

    calls = []
    monkeypatch.setattr(device_ops, "_device_of", lambda name, first, *others: first.device)
    monkeypatch.setattr(device_ops, "_plan_bytes", lambda *args: 0)
    monkeypatch.setattr(device_ops, "_call_on", lambda dev, name, *args: calls.append(name))
    t = {k: torch.zeros(4, 8, dtype=torch.bfloat16) for k in ("y", "x", "out")}
    bank = adapters.AdapterBank(*(torch.zeros(2, 8, 8, dtype=torch.bfloat16) for _ in range(2)))
    who = torch.zeros(4, dtype=torch.int32)
    bank(t["y"], t["x"], who, out=t["out"])
    assert calls == ["rb_low_rank_add"]
    (bank.a if which == "a" else t[which]).requires_grad_()
    for call in (lambda: bank(t["y"], t["x"], who, out=t["out"]),
                 lambda: device_ops.low_rank_add(t["y"], t["x"], bank.a, bank.b, who, bank.scale, out=t["out"])):
        with pytest.raises(RuntimeError, match="no backward"):
            call()
    assert calls == ["rb_low_rank_add"]
    with torch.no_grad():
        assert bank(t["y"], t["x"], who, out=t["out"]) is t["out"]
