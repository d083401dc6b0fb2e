"""The layer functions under torch's autograd: what they do not differentiate is refused, never dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from dgcnn_amd import layers

gpu = pytest.mark.gpu
with fwd.dual_level():      # (the first tangent loads torch's decompositions, which have to be compiled before the CPU emulation replaces torch's functions)
    fwd.make_dual(torch.zeros(1), torch.zeros(1))


def calls():
    x, ptr = torch.randn(10, 8).to("cuda"), torch.tensor([0, 4, 10]).to("cuda")
    weight, bias, w, b = (torch.randn(s).to("cuda") for s in ((2, 3, 8), (2, 3), (8,), (8,)))
    linear = lambda x=x, weight=weight, bias=bias: layers.grouped_linear(x, weight, ptr, bias)      # noqa: E731
    norm = lambda x=x, weight=w, bias=b: layers.group_norm(x, 2, weight, bias, ptr=ptr, act="silu")      # noqa: E731
    dense = lambda x=x.view(2, 5, 8), weight=w, bias=b: layers.group_norm(x, 2, weight, bias)      # noqa: E731
    return [(linear, dict(x=x, weight=weight, bias=bias)), (norm, dict(x=x, weight=w, bias=b)), (dense, dict(x=x.view(2, 5, 8), weight=w, bias=b))]


@gpu
@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("which", ["x", "weight", "bias"])
def test_a_forward_mode_tangent_is_refused(which, grad_mode):
    """these have no forward-mode rule: a result without a tangent would read as a derivative of zero"""
    for f, args in calls():
        with torch.set_grad_enabled(grad_mode), fwd.dual_level():
            dual = fwd.make_dual(args[which], torch.ones_like(args[which]))
            with pytest.raises(NotImplementedError):
                f(**{which: dual})
            y = f()                      # (other tensors inside a dual level are ordinary ones)
        assert torch.isfinite(y.cpu()).all()


@gpu
def test_a_tangent_of_strided_rows_is_refused():
    with fwd.dual_level():
        x = fwd.make_dual(torch.randn(8, 10).to("cuda"), torch.ones(8, 10).to("cuda")).t()      # (copied before the call)
        with pytest.raises(NotImplementedError):
            layers.grouped_linear(x, torch.randn(2, 3, 8).to("cuda"), torch.tensor([0, 4, 10]).to("cuda"))
        with pytest.raises(NotImplementedError):
            layers.group_norm(x, 2)


@gpu
def test_function_transforms_are_refused():
    f = lambda x: layers.group_norm(x, 2)      # noqa: E731
    x = torch.randn(4, 6, 8).to("cuda")
    for call in (lambda: torch.func.jvp(f, (x,), (x,)), lambda: torch.func.grad(lambda t: f(t).sum())(x), lambda: torch.func.vmap(f)(x)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()


@gpu
def test_second_derivatives_are_refused():
    for f, args in calls():
        x = args["x"].clone().requires_grad_(True)
        (g,) = torch.autograd.grad(f(x=x).square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()
