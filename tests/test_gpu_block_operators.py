"""The operators together, as an encoder block uses them: the seam of the previous block (sandwich_norm) gives the
router its rows, the router the experts theirs, the experts' output goes through the next seam, and a shared
projection with per-user adapters reads the normalised rows.

Tolerance of the whole run: it passes six roundings to bf16 that the float64 run does not (y and z of the first seam,
scores, expert output, z of the second, the projection), each at most 2^-8 of its value and independent of the
others' signs, and the expert layer's own three: under 9 * 2^-8 in relative L2.
"""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _layer(D, F, E):
    nn = torch.nn

    class Expert(nn.Module):
        def __init__(self):
            super().__init__()
            self.fc1, self.fc2 = nn.Linear(D, F), nn.Linear(F, D)

    class Moe(nn.Module):
        def __init__(self, gate):
            super().__init__()
            self.experts = nn.ModuleList([Expert() for _ in range(E)])
            self.gate = gate

    return Moe


@pytest.mark.parametrize("T", [1, 37, 2000])
def test_block_of_seams_router_experts_and_adapters(cuda_device, T):
    from baidu_cti_grab_b200 import adapters, block_norm, device_ops, routing, smoe

    D, F, E, N, R = 512, 1024, 8, 768, 3
    torch.manual_seed(T)
    gate = routing.TopKRouter(D, E, 2, renormalize=True, balanced=True)
    moe = _layer(D, F, E)(gate).to(cuda_device, BF)
    seams = [block_norm.SandwichNorm(D, scale=0.5, channel_gate=True, gate_init=0.8).to(cuda_device, BF) for _ in range(2)]
    linear = torch.nn.Linear(D, N).to(cuda_device, BF)
    bank = adapters.AdapterBank((torch.randn(R, 16, D) / D ** 0.5).to(BF), (torch.randn(R, N, 16) / 4).to(BF)).to(cuda_device)
    offsets = torch.tensor([0, T // 3, T // 2, T], device=cuda_device)
    who = bank.per_token(torch.tensor([2, -1, 0], device=cuda_device), offsets, T)
    x = torch.randn(T, D, device=cuda_device).to(BF)
    h = torch.randn(T, D, device=cuda_device).to(BF)
    with torch.no_grad():
        y0, z0 = seams[0](x, h)
        moe_out, loss = smoe.smoe_forward(moe, z0.view(1, T, D))
        y1, z1 = seams[1](y0, moe_out[0])
        base = linear(z1)
        out = bank(base, z1, who)
        r = gate.route(z0, want_counts=True)
        assert int(r.counts.sum()) == 2 * T and bool(loss.isfinite())
        gate.update_balance(r.counts, 1e-3)

        # the same in float64, with the experts that the router chose
        def seam(m, x, h):
            ln = lambda v, w, b: torch.nn.functional.layer_norm(v, (D,), w.double(), b.double(), m.eps)  # noqa: E731
            y = x + m.scale * m.gate.double() * ln(h, m.post_weight, m.post_bias)
            return y, ln(y, m.pre_weight, m.pre_bias)

        yr, zr = seam(seams[0], x.double(), h.double())
        score = torch.softmax(torch.nn.functional.linear(zr, gate.w_g.weight.double(), gate.w_g.bias.double()), -1)
        w = score.gather(1, r.idx)
        w = w / w.sum(-1, keepdim=True)
        mixed = torch.zeros_like(zr)
        for e, ex in enumerate(moe.experts):
            f = torch.relu(torch.nn.functional.linear(zr, ex.fc1.weight.double(), ex.fc1.bias.double()))
            f = torch.nn.functional.linear(f, ex.fc2.weight.double(), ex.fc2.bias.double())
            mixed += f * (w * (r.idx == e)).sum(-1, keepdim=True)
        _, zr = seam(seams[1], yr, mixed)
        want = torch.nn.functional.linear(zr, linear.weight.double(), linear.bias.double())
        for i in range(R):
            rows = who == i
            want[rows] += zr[rows] @ bank.a[i].double().t() @ bank.b[i].double().t()
    assert float((out.double() - want).norm() / want.norm()) <= 9 * 2.0 ** -8
    torch.cuda.synchronize()
    assert device_ops.device_error() == 0


def test_training_step_through_seam_and_router(cuda_device):
    """Gradients of a seam, a router and dense experts in one autograd graph, fp32: each kernel's gradient is
    within 2^-13 of its terms (their own tests), two of them and fp32 products in a row under 2^-10."""
    from baidu_cti_grab_b200 import block_norm, routing

    D, E, T = 96, 12, 150
    torch.manual_seed(3)
    seam = block_norm.SandwichNorm(D, post="rms", pre="layer", scale=0.7, channel_gate=True, gate_act="sigmoid").to(cuda_device)
    gate = routing.TopKRouter(D, E, 3, renormalize=True).to(cuda_device)
    mix = torch.randn(E, D, D, device=cuda_device) / D ** 0.5
    x, h = (torch.randn(T, D, device=cuda_device, requires_grad=True) for _ in range(2))
    y, z = seam(x, h)
    idx, score, probs = gate(z)
    out = y + (torch.einsum("td,edf->tef", z, mix).gather(1, idx[..., None].expand(-1, -1, D)) * score[..., None]).sum(1)
    (out.square().mean() + 0.1 * probs.sum(0).var()).backward()
    leaves = dict(x=x, h=h, **dict(seam.named_parameters()), **{"gate_" + n: p for n, p in gate.named_parameters()})
    ref = {n: p.detach().double().requires_grad_() for n, p in leaves.items()}
    n = ref["h"] / torch.sqrt(ref["h"].square().mean(-1, keepdim=True) + 1e-5) * ref["post_weight"]
    y64 = ref["x"] + 0.7 * torch.sigmoid(ref["gate"]) * n
    z64 = torch.nn.functional.layer_norm(y64, (D,), ref["pre_weight"], ref["pre_bias"], 1e-5)
    p64 = torch.softmax(torch.nn.functional.linear(z64, ref["gate_w_g.weight"], ref["gate_w_g.bias"]), -1)
    w64 = p64.gather(1, idx)
    w64 = w64 / w64.sum(-1, keepdim=True)
    o64 = y64 + (torch.einsum("td,edf->tef", z64, mix.double()).gather(1, idx[..., None].expand(-1, -1, D)) * w64[..., None]).sum(1)
    grads = torch.autograd.grad(o64.square().mean() + 0.1 * p64.sum(0).var(), list(ref.values()))
    for (name, p), want in zip(leaves.items(), grads):
        assert float((p.grad.double() - want).norm()) <= 2.0 ** -10 * float(want.norm()), name
