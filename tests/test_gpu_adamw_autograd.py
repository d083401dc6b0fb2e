"""An optimizer step is a change in place that autograd can see: what a graph saved before it is not used behind it."""
import pytest
import torch

from dgcnn_amd import optim

gpu = pytest.mark.gpu


def lists(bits=32, dtype=torch.float32, master=False, n=300):
    p, g = torch.randn(n).to(dtype).to("cuda"), torch.randn(n).to(dtype).to("cuda")
    if bits == 32:
        m, v, more = torch.zeros(n).to("cuda"), torch.zeros(n).to("cuda"), {}
    else:
        m, v = (torch.zeros(n, dtype=torch.uint8).to("cuda").view(torch.float8_e4m3fn) for _ in range(2))
        more = {k: [torch.zeros(2).to("cuda")] for k in ("exp_avg_scales", "exp_avg_sq_scales")}
    if master:
        more["masters"] = [p.float()]
    return [p], [g], [m], [v], more


@gpu
@pytest.mark.parametrize("bits,dtype,master", [(32, torch.float32, False), (8, torch.float32, False), (32, torch.bfloat16, True), (8, torch.float16, True)])
def test_everything_a_step_writes_gets_a_new_version(bits, dtype, master):
    p, g, m, v, more = lists(bits, dtype, master)
    written = [*p, *m, *v, *(t for ts in more.values() for t in ts)]
    for step in (1, 2):
        before, kept = [t._version for t in written], [t._version for t in g]
        optim.adamw_step(p, g, m, v, step=step, **more)
        assert all(t._version > b for t, b in zip(written, before)) and [t._version for t in g] == kept
    count = torch.zeros(1, dtype=torch.int64).to("cuda")
    optim.adamw_step(p, g, m, v, step=count, **more)
    assert int(count) == 1 and count._version > 0


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_backward_pass_behind_the_step_is_an_error(bits):
    """y = w . x saved w: behind a step its gradient in x would be the new w"""
    w = torch.nn.Parameter(torch.ones(4).to("cuda"))
    x = torch.ones(4).to("cuda").requires_grad_(True)
    opt = optim.AdamW([w], lr=0.5, state_bits=bits)
    y = (w * x).sum()
    w.grad = torch.ones(4).to("cuda")
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    z = (w * x).sum()      # (a graph built behind the step is right)
    assert torch.equal(torch.autograd.grad(z, x)[0], w.detach())


@gpu
def test_a_parameter_that_an_optimizer_leaves_alone_keeps_its_version():
    w, u = (torch.nn.Parameter(torch.ones(4).to("cuda")) for _ in range(2))
    opt = optim.AdamW([w, u])
    w.grad = torch.ones(4).to("cuda")
    before = u._version
    opt.step()
    assert u._version == before


@gpu
def test_tensors_made_in_inference_mode_have_no_version_and_are_updated():
    with torch.inference_mode():
        p, g, m, v, more = lists()
        before = p[0].clone()
        optim.adamw_step(p, g, m, v, step=1, **more)
        assert not torch.equal(p[0].cpu(), before.cpu())
