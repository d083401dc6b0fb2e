"""AdamW over parameters of any dense memory layout: one step of a tensor is that of its elements, wherever they lie.  Results are compared bit for bit with those of the
same elements in contiguous tensors."""
import pytest
import torch

from dgcnn_amd import _lib, optim

gpu = pytest.mark.gpu
LAYOUTS = {
    "transposed": lambda t: t.t().contiguous().t(),
    "permuted": lambda t: t.view(6, 5, 4).permute(2, 0, 1).contiguous().permute(1, 2, 0),
    "channels_last": lambda t: t.view(2, 3, 4, 5).contiguous(memory_format=torch.channels_last),
    "size_one": lambda t: t.view(30, 1, 4).permute(2, 1, 0).contiguous().permute(2, 1, 0),
}


def pair(layout, dtype=torch.float32):
    g = torch.Generator().manual_seed(1)
    a = torch.randn(30, 4, generator=g).to(dtype).to("cuda")
    b = LAYOUTS[layout](a)
    assert not b.is_contiguous() or layout == "size_one"
    return torch.nn.Parameter(a.clone()), torch.nn.Parameter(b.clone())      # (clone keeps the strides)


@gpu
@pytest.mark.parametrize("layout", sorted(LAYOUTS))
@pytest.mark.parametrize("dtype,kw", [(torch.float32, {}), (torch.bfloat16, dict(master_weights=True)), (torch.float32, dict(capturable=True))])
def test_a_step_of_a_permuted_parameter(layout, dtype, kw):
    p, q = pair(layout, dtype)
    a, b = optim.AdamW([p], lr=1e-2, **kw), optim.AdamW([q], lr=1e-2, **kw)
    for k in range(3):
        g = torch.randn(30, 4, generator=torch.Generator().manual_seed(10 + k)).to(dtype).to("cuda")
        p.grad = g
        q.grad = g.view(q.shape).contiguous() if k == 1 else torch.empty_like(q).copy_(g.view(q.shape))      # (gradients of another layout too)
        a.step(); b.step()
    assert torch.equal(p.detach().reshape(-1).cpu(), q.detach().reshape(-1).cpu())
    for name in ("exp_avg", "exp_avg_sq", *(("master",) if kw.get("master_weights") else ())):
        assert torch.equal(a.state[p][name].reshape(-1).cpu(), b.state[q][name].reshape(-1).cpu()), name


@gpu
@pytest.mark.parametrize("layout", sorted(LAYOUTS))
def test_8_bit_states_follow_the_memory_order(layout):
    """blocks, scales and random bits go by the elements as they lie: those of a contiguous tensor with the same memory"""
    _, q = pair(layout)
    flat = q.detach().as_strided((q.numel(),), (1,)).clone()
    p = torch.nn.Parameter(flat)
    a, b = (optim.AdamW([t], lr=1e-2, state_bits=8, seed=3) for t in (p, q))
    for k in range(3):
        q.grad = torch.empty_like(q).copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(k)).to("cuda"))
        p.grad = q.grad.as_strided((q.numel(),), (1,)).clone()
        a.step(); b.step()
    assert torch.equal(p.detach().cpu(), q.detach().as_strided((q.numel(),), (1,)).cpu())
    assert torch.equal(a.state[p]["exp_avg"].view(torch.uint8).cpu(), b.state[q]["exp_avg"].view(torch.uint8).as_strided((q.numel(),), (1,)).cpu())


@gpu
def test_lists_whose_strides_differ_in_dimensions_of_one_element_only():
    t = torch.zeros(4, 1, 6).to("cuda").transpose(0, 2).contiguous().transpose(0, 2)
    others = [torch.ones(24).to("cuda").as_strided((4, 1, 6), (1, 77, 4)) for _ in range(3)]
    optim.adamw_step([t], others[:1], [torch.zeros_like(t)], [torch.zeros_like(t)], step=1)
    assert (t.cpu() < 0).all()


@gpu
def test_states_load_between_layouts():
    p, q = pair("transposed")
    r = torch.nn.Parameter(LAYOUTS["permuted"](p.detach()))
    a, b = optim.AdamW([p]), optim.AdamW([q])
    p.grad = torch.randn(30, 4, generator=torch.Generator().manual_seed(2)).to("cuda")
    a.step()
    b.load_state_dict(a.state_dict())
    assert torch.equal(b.state[q]["exp_avg"].cpu(), a.state[p]["exp_avg"].cpu()) and b.state[q]["exp_avg"].stride() == q.stride()
    q.grad = torch.zeros_like(q)
    b.step()
    c, d = optim.AdamW([q], state_bits=8), optim.AdamW([q], state_bits=8)
    c.step()
    d.load_state_dict(c.state_dict())                # the same layout: the same blocks
    with pytest.raises(ValueError):                  # another one, neither of them contiguous
        c8 = optim.AdamW([torch.nn.Parameter(r.detach().clone())], state_bits=8)
        s = c.state_dict()
        for k in ("exp_avg", "exp_avg_sq"):
            s["state"][0][k] = s["state"][0][k].view(torch.uint8).view(6, 5, 4).contiguous().permute(1, 2, 0).contiguous().permute(2, 0, 1).view(torch.float8_e4m3fn)
        c8.load_state_dict(s)


@gpu
def test_what_is_not_dense_is_refused():
    for x in (torch.zeros(8, 8).to("cuda")[:, :4], torch.zeros(8, 1).to("cuda").expand(8, 4), torch.zeros(4).to("cuda").as_strided((2, 3), (1, 1))):
        with pytest.raises(_lib.DgcnnError, match="dense"):
            optim.adamw_step([x], [x], [x], [x], step=1)


@gpu
def test_lists_of_other_shapes_are_refused():
    """[3, 2] with the parameter's strides (1, 2) holds five places where [2, 3] has six: elements behind its end would be written"""
    p = torch.zeros(3, 2).to("cuda").t()
    short = torch.zeros(5).to("cuda").as_strided((3, 2), (1, 2))
    ok = torch.zeros_like(p)
    for lists in ((p, short, ok, ok), (p, ok, short, ok), (p, ok, ok, short)):
        with pytest.raises(_lib.DgcnnError):
            optim.adamw_step(*([t] for t in lists), step=1)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_state_of_torchs_adamw_over_16_bit_parameters_loads(dtype):
    """torch holds the moments in the parameter's type: they are widened, which is exact"""
    p = torch.nn.Parameter(torch.linspace(-1, 1, 50).to(dtype).to("cuda"))
    q = torch.nn.Parameter(p.detach().clone())
    a, b = torch.optim.AdamW([p], lr=1e-2, foreach=False), optim.AdamW([q], lr=1e-2)
    g = torch.linspace(1, 2, 50).to(dtype).to("cuda")
    p.grad = g
    a.step()
    b.load_state_dict(a.state_dict())
    for name in ("exp_avg", "exp_avg_sq"):
        assert b.state[q][name].dtype == torch.float32 and torch.equal(b.state[q][name].cpu(), a.state[p][name].float().cpu())
    m = b.state[q]["exp_avg"].cpu().double()
    q.grad = g
    b.step()
    want = 0.9 * m + 0.1 * g.cpu().double()
    assert b.state[q]["step"] == 2 and ((b.state[q]["exp_avg"].cpu().double() - want).abs() <= 4 * 2.0 ** -24 * want.abs()).all()
