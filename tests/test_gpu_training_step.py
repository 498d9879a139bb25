"""A training step as the operators are used together: embedding rows go through the seam between blocks into attention
within packed users, the loss's gradient comes back through all of them to the table, and everything is clipped by one
norm; and the same table's gradient for the touched rows alone.

Tolerance: in bf16 the forward run passes seven roundings that the float64 run does not (rows, y and z of the seam, the two
projections, the attention's weights and its output), the gradients about as many again on their way back (through the
projections, the attention's e and p, dq, dk, dv, the seam's dx), each at most 2^-8 of its value: under 16 * 2^-8 in
relative L2.  In fp32, where attention takes no fp32 rows, only the parts around it are compared.
"""

import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _reference(w, ids, offsets, slopes, cap, scale, heads, kv, width, eps):
    """The step's output in float64 from parameters by name."""
    lin = torch.nn.functional.linear
    x = w["table.weight"][ids] * scale
    D = x.shape[-1]
    y = x + 0.5 * w["seam.gate"] * torch.nn.functional.layer_norm(x, (D,), w["seam.post_weight"], w["seam.post_bias"], eps)
    z = torch.nn.functional.layer_norm(y, (D,), w["seam.pre_weight"], w["seam.pre_bias"], eps)
    q, k, v = lin(z, w["attention.qkv.weight"], w["attention.qkv.bias"]).view(-1, heads + 2 * kv, width).split((heads, kv, kv), 1)
    rows = []
    for a, b in zip(offsets[:-1], offsets[1:]):
        i = torch.arange(int(b - a), device=ids.device)
        far = i[:, None] - i
        s = torch.einsum("ihd,jhd->hij", q[a:b], k[a:b].repeat_interleave(heads // kv, 1)) / math.sqrt(width)
        s = cap * torch.tanh(s / cap) - slopes.double()[:, None, None] * far.abs()
        p = torch.softmax(s.masked_fill(far < 0, -math.inf), -1)
        rows.append(torch.einsum("hij,jhd->ihd", p, v[a:b].repeat_interleave(heads // kv, 1)).flatten(1))
    return y + lin(torch.cat(rows), w["attention.out.weight"], w["attention.out.bias"])


class Step(torch.nn.Module):
    def __init__(self, rows, D, heads, kv):
        super().__init__()
        from baidu_cti_grab_b200 import attention, block_norm, embedding

        self.table = embedding.RowEmbedding(rows, D, scale=4.0, std=0.25)
        self.seam = block_norm.SandwichNorm(D, scale=0.5, channel_gate=True, gate_init=0.8)
        self.attention = attention.SegmentAttention(D, heads, kv, cap=20.0, distance=True)

    def forward(self, ids, offsets):
        x = self.table(ids)
        y, z = self.seam(x, x)
        return y + self.attention(z, offsets)


@pytest.mark.parametrize("lengths,D,heads,kv", [([1], 64, 2, 1), ([70, 1, 130, 5], 128, 4, 2), ([300, 260], 256, 2, 2)])
def test_training_step(cuda_device, lengths, D, heads, kv):
    from baidu_cti_grab_b200 import device_ops, embedding, grad_clip

    torch.manual_seed(len(lengths))
    V = 97
    step = Step(V, D, heads, kv).to(cuda_device, BF)
    ids = torch.randint(0, V, (sum(lengths),), device=cuda_device)
    offsets = torch.tensor([0, *lengths], device=cuda_device).cumsum(0)
    out = step(ids, offsets)
    g = torch.randn_like(out)
    out.backward(g)
    w = {n: p.detach().double().requires_grad_() for n, p in step.named_parameters()}
    want = _reference(w, ids, offsets, step.attention.slopes, 20.0, 4.0, heads, kv, D // heads, step.seam.eps)
    grads = dict(zip(w, torch.autograd.grad((want * g.double()).sum(), list(w.values()))))
    rel = lambda a, b: float((a.double() - b).norm() / b.norm())  # noqa: E731
    assert rel(out, want.detach()) <= 16 * 2.0 ** -8
    names = [n for n in w if float(grads[n].norm()) > 0 and not (len(ids) == 1 and "qkv" in n)]  # (one key: no score matters)
    for n in names:
        # a key's bias moves all of a query's scores alike but for what tanh and the rounding make of it: left to the weights
        if n != "attention.qkv.bias":
            assert rel(step.get_parameter(n).grad, grads[n]) <= 16 * 2.0 ** -8, n
    # the table's gradient of the touched rows alone is the dense one's, and both clip by one norm
    own = {n: p.grad.clone() for n, p in step.named_parameters()}
    norm = math.sqrt(sum(float(t.double().square().sum()) for t in own.values()))
    total = grad_clip.clip_grad_norm(step.parameters(), 0.5 * norm)
    assert abs(float(total) - norm) <= 7 * 2.0 ** -24 * norm
    for n, p in step.named_parameters():
        assert rel(p.grad, own[n].double() * 0.5) <= 2.0 ** -8 + 2.0 ** -20 or not own[n].any()
    x = torch.randn(len(ids), D, device=cuda_device).to(BF)
    s = embedding.SparseRows(*device_ops.embed_rows_backward_sparse(x, ids, V, scale=4.0))
    dense = device_ops.embed_rows_backward(x, ids, V, scale=4.0)
    m = int(s.count)
    assert torch.equal(s.ids[:m], ids.unique()) and torch.equal(s.rows[:m], dense[s.ids[:m]])
    a, b = grad_clip.grad_norm([], sparse=[s]), device_ops.grad_norm([dense])
    assert abs(float(a) - float(b)) <= 14 * 2.0 ** -24 * float(b)
    torch.cuda.synchronize()
    assert device_ops.device_error() == 0


def test_captured_step(cuda_device):
    """The step's plain calls in a graph, replayed on other ids and users."""
    from baidu_cti_grab_b200 import device_ops

    torch.manual_seed(0)
    V, D, heads, n = 60, 64, 2, 90
    table = torch.randn(V, D, device=cuda_device, dtype=BF)
    ids, other = (torch.randint(0, V, (n,), device=cuda_device) for _ in range(2))
    offsets, split = (torch.tensor(o, dtype=torch.int32, device=cuda_device) for o in ([0, 40, 90], [0, 1, 90]))
    g = torch.randn(n, heads, D // heads, device=cuda_device, dtype=BF)

    def step(ids, offsets):
        x = device_ops.embed_rows(table, ids).view(n, heads, D // heads)
        out, lse = device_ops.segment_attention(x, x, x, offsets, want_lse=True)
        dq, dk, dv = device_ops.segment_attention_backward(g, x, x, x, out, lse, offsets)
        dt = device_ops.embed_rows_backward((dq + dk + dv).view(n, D), ids, V)
        return out, dt, device_ops.clip_grads([dt], 1.0)

    want = [[t.clone() for t in step(i, o)] for i, o in ((ids, offsets), (other, split))]
    held = ids.clone(), offsets.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*held)
    for (i, o), w in zip(((other, split), (ids, offsets)), reversed(want)):
        held[0].copy_(i)
        held[1].copy_(o)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, w))
