"""The layer and optimizer operators as they are used together: one training step of a typed graph layer -- nodes sorted by type through
GroupedLinear, back in graph order through GroupNorm with an activation, a second product, a loss, AdamW -- against the same step in 64 bits.

Tolerances: the operators' own tests bound each result in units of its terms; here the chain's values are of order 1 and sums of at most 2000 terms pass
through three layers, so an fp32 chain is off by at most a few hundred times 2^-24 of the largest value: 2^-14 of it.  AdamW's first step moves every
parameter by lr * sign(gradient) up to eps, so the updated parameter is compared where the gradient is over 2^-10 of its largest."""
import pytest
import torch

from dgcnn_amd import layers, optim
from dgcnn_amd.batch import Graph, collate

gpu = pytest.mark.gpu


class TypedBlock(torch.nn.Module):
    def __init__(self, types, fin, hidden, out):
        super().__init__()
        self.lin1 = layers.GroupedLinear(types, fin, hidden)
        self.norm = layers.GroupNorm(4, hidden, act="silu")
        self.lin2 = layers.GroupedLinear(types, hidden, out)

    def forward(self, x, order, type_ptr, graph_ptr):
        h = torch.empty_like(x[:, :1]).expand(-1, self.lin1.out_features).clone()
        h = h.index_copy(0, order, self.lin1(x[order], type_ptr))      # rows by type -> rows by graph
        h = self.norm(h, graph_ptr)
        return self.lin2(h[order], type_ptr)


def batch_of(sizes, fin, types, seed=0):
    g = torch.Generator().manual_seed(seed)
    graphs = [Graph(torch.randn(n, fin, generator=g), torch.tensor([[0], [0]]), 0) for n in sizes]
    b = collate(graphs)
    kind = torch.randint(0, types, (b.num_nodes,), generator=g)
    order = torch.sort(kind, stable=True).indices
    type_ptr = torch.searchsorted(kind[order], torch.arange(types + 1))
    return b, kind, order, type_ptr


def reference(m, b, kind, order, target, groups=4, eps=1e-5):
    """loss and gradients in 64 bits, row by row from the definitions"""
    P = {k: v.detach().cpu().double().requires_grad_(True) for k, v in m.named_parameters()}
    x = b.x.double()
    h = torch.stack([P["lin1.weight"][kind[i]] @ x[i] + P["lin1.bias"][kind[i]] for i in range(x.shape[0])])
    out = []
    for s in range(b.num_graphs):
        t = h[b.batch == s].reshape(int((b.batch == s).sum()), groups, -1)
        out.append(((t - t.mean((0, 2), keepdim=True)) / (t.var((0, 2), correction=0, keepdim=True) + eps).sqrt()).reshape(t.shape[0], -1))
    z = torch.cat(out) * P["norm.weight"] + P["norm.bias"]
    z = z * torch.sigmoid(z)
    y = torch.stack([P["lin2.weight"][kind[i]] @ z[i] + P["lin2.bias"][kind[i]] for i in range(x.shape[0])])
    loss = ((y[order] - target) ** 2).mean()
    return loss, dict(zip(P, torch.autograd.grad(loss, list(P.values())))), P


@gpu
@pytest.mark.parametrize("sizes,fin,hidden,out,types", [([5, 1, 40], 7, 32, 6, 3), ([30, 60, 3, 17], 16, 24, 9, 5)])
def test_one_training_step(sizes, fin, hidden, out, types):
    torch.manual_seed(1)
    m = TypedBlock(types, fin, hidden, out)
    b, kind, order, type_ptr = batch_of(sizes, fin, types)
    target = torch.randn(b.num_nodes, out)
    want_loss, want, P = reference(m, b, kind, order, target.double())
    m = m.to("cuda")
    d = b.to("cuda")
    opt = optim.AdamW(m.parameters(), lr=1e-2, weight_decay=0.1)
    y = m(d.x, order.to("cuda"), type_ptr.to("cuda"), layers.graph_ptr(d))
    loss = ((y - target.to("cuda")) ** 2).mean()
    loss.backward()
    before = {k: v.detach().cpu().double().clone() for k, v in m.named_parameters()}
    assert abs(loss.item() - want_loss.item()) <= 2.0 ** -14 * want_loss.item()
    for k, p in m.named_parameters():
        g = p.grad.cpu().double()
        assert float((g - want[k]).abs().max()) <= 2.0 ** -14 * float(want[k].abs().max()), k
    opt.step()
    for k, p in m.named_parameters():
        sure = want[k].abs() > 2.0 ** -10 * want[k].abs().max()
        moved = before[k] * (1 - 1e-3) - 1e-2 * want[k].sign()
        assert float((p.detach().cpu().double() - moved)[sure].abs().max()) <= 2.0 ** -18 + 1e-2 * 2.0 ** -10, k


@gpu
def test_captured_training_step_replays():
    """forward, backward and a capturable AdamW step in one graph: four replays on changing data equal four eager steps bit for bit (rows sorted by type and
    by graph at once, and the loss's gradient written out: nothing but these operators and elementwise ones is captured)"""
    if not torch.cuda.is_available():
        pytest.skip("graphs need the GPU")
    type_ptr, graph_ptr = (torch.tensor(t, device="cuda") for t in ([0, 90, 90, 93, 263, 263], [0, 30, 90, 93, 263]))
    target = torch.randn(263, 8).cuda()
    data = [torch.randn(263, 16).cuda() for _ in range(5)]

    def new():
        torch.manual_seed(3)
        m = TypedBlock(5, 16, 64, 8).cuda()
        return m, optim.AdamW(m.parameters(), lr=1e-2, capturable=True, state_bits=8)

    def step(m, o, x):
        o.zero_grad(set_to_none=False)
        y = m.lin2(m.norm(m.lin1(x, type_ptr), graph_ptr), type_ptr)
        torch.autograd.backward(y, y.detach() - target)
        o.step()

    (m, o), (e, eo) = new(), new()
    x = data[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(m, o, x)
    torch.cuda.current_stream().wait_stream(side)
    step(e, eo, data[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(m, o, x)
    for t in data[1:]:
        x.copy_(t)
        graph.replay()
        step(e, eo, t)
        torch.cuda.synchronize()
        for p, q in zip(m.parameters(), e.parameters()):
            assert torch.equal(p, q)


@gpu
def test_example_in_bf16_runs_and_has_gradients():
    torch.manual_seed(2)
    b, kind, order, type_ptr = batch_of([20, 44], 16, 3)
    m = TypedBlock(3, 16, 32, 8).to(torch.bfloat16).to("cuda")
    d = b.to("cuda")
    o = optim.AdamW(m.parameters(), lr=1e-2, state_bits=8, master_weights=True)
    y = m(d.x.to(torch.bfloat16), order.to("cuda"), type_ptr.to("cuda"), layers.graph_ptr(d))
    y.float().square().mean().backward()
    for p in m.parameters():
        assert p.grad is not None and torch.isfinite(p.grad.float()).all() and p.grad.float().abs().sum() > 0
    start = [p.detach().clone() for p in m.parameters()]
    o.step()
    assert any(not torch.equal(a, p.detach()) for a, p in zip(start, m.parameters()))


@gpu
@pytest.mark.parametrize("op", ["norm", "linear"])
def test_backward_reads_what_saved_tensor_hooks_return(op):
    """saved tensors may be moved between the passes (offloaded and brought back): the backward takes them where they are then"""
    g = torch.Generator().manual_seed(2)
    ptr = torch.tensor([0, 4, 4, 9]).to("cuda")
    x0 = torch.randn(9, 8, generator=g)
    w0 = torch.randn(8, generator=g) if op == "norm" else torch.randn(3, 5, 8, generator=g)
    dy = torch.randn(9, 8 if op == "norm" else 5, generator=g).to("cuda")
    got = []
    for moved in (False, True):
        x, w = (t.clone().to("cuda").requires_grad_(True) for t in (x0, w0))
        with torch.autograd.graph.saved_tensors_hooks((lambda t: t.detach().clone()) if moved else (lambda t: t), lambda t: t):
            y = layers.group_norm(x, 2, w, ptr=ptr, act="silu") if op == "norm" else layers.grouped_linear(x, w, ptr)
        if moved:
            x.data.zero_()
            w.data.zero_()
        got.append(torch.autograd.grad(y, (x, w), dy))
    for a, b in zip(*got):
        assert torch.equal(a, b) and bool(a.abs().max() > 0)
