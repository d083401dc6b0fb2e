"""The random bits that round 8-bit moments: a hash of (seed, index of the tensor, step, element).  A tensor's index is its own -- its place among the optimizer's
parameters, or what the caller says --, so neither the other tensors of a call nor the calls that a step is made of change its codes, and no two tensors share theirs."""
import pytest
import torch

from dgcnn_amd import _lib, optim
from test_gpu_adamw import KW, call, check_codes, formula, hash_bits, make

gpu = pytest.mark.gpu
N = 2000


def codes(opt, p):
    return torch.cat([opt.state[p][k].view(torch.uint8).cpu().reshape(-1) for k in ("exp_avg", "exp_avg_sq")])


def params(n, dtype=torch.float32):
    return [torch.nn.Parameter(torch.zeros(N, dtype=dtype).to("cuda")) for _ in range(n)]


def grads(k):
    return torch.randn(N, generator=torch.Generator().manual_seed(k))


def steps(opt, ps, skip=(), count=3):
    for k in range(count):
        for i, p in enumerate(ps):
            p.grad = None if i in skip else grads(k).to(p.dtype).to("cuda")      # (every tensor the same gradient)
        opt.step()


@gpu
def test_equal_gradients_are_rounded_apart_in_every_list():
    """two groups, and two types in one group: a call each, no two tensors with the same bits"""
    ps = params(2) + params(2, torch.bfloat16)
    grouped = optim.AdamW([dict(params=[ps[0], ps[2]]), dict(params=[ps[1], ps[3]], weight_decay=0.0)], state_bits=8, seed=1)
    steps(grouped, ps)
    for i in range(4):
        for j in range(i):
            if ps[i].dtype == ps[j].dtype:
                same = float((codes(grouped, ps[i]) == codes(grouped, ps[j])).float().mean())
                # (of a continuous distribution of places between two codes about two thirds fall on the same side of two random thresholds)
                assert same < 0.9, (i, j, same)


@gpu
def test_an_absent_gradient_elsewhere_changes_nothing():
    a, b = params(4), params(4)
    steps(optim.AdamW(a, state_bits=8, seed=2), a)
    oa, ob = optim.AdamW(a, state_bits=8, seed=2), optim.AdamW(b, state_bits=8, seed=2)
    steps(oa, a); steps(ob, b, skip=(0, 2))
    for i in (1, 3):
        assert torch.equal(codes(oa, a[i]), codes(ob, b[i])), i


@gpu
def test_groups_do_not_change_the_bits():
    a, b = params(3), params(3)
    oa = optim.AdamW(a, state_bits=8, seed=3)
    ob = optim.AdamW([dict(params=b[:1]), dict(params=b[1:], weight_decay=0.5)], state_bits=8, seed=3)
    steps(oa, a); steps(ob, b)
    for p, q in zip(a, b):
        assert torch.equal(codes(oa, p), codes(ob, q))


@gpu
def test_indices_of_a_call():
    """indices[i] stands in the hash for tensor i; without them its place in the list"""
    sizes, idx, seed = [700, 5, 256, 3000], [70, 0, (1 << 40) + 3, 2], 9
    t = make(sizes, torch.float32, torch.float32, 8, False)
    want = [formula(t, i, 8, False, 4, KW["lr"], KW["betas"], KW["eps"], KW["weight_decay"]) for i in range(4)]
    call(t, 8, False, step=4, seed=seed, indices=idx, **KW)
    for i, (_, m, v, _, _) in enumerate(want):
        nm, nv = hash_bits(sizes[i], idx[i], seed, 4)
        check_codes(t["m"][i], t["ms"][i], m, nm, False)
        check_codes(t["v"][i], t["vs"][i], v.sqrt(), nv, True)
    # ... whatever list the tensor is in: the 130th of three launches, or alone
    sizes = [1 + (37 * i) % 900 for i in range(130)]
    a, b, c = (make(sizes, torch.float32, torch.float32, 8, False) for _ in range(3))
    call(a, 8, False, step=7, seed=3, **KW)
    call(b, 8, False, step=7, seed=3, indices=range(130), **KW)
    for i in (0, 47, 48, 129):
        assert torch.equal(a["m"][i].view(torch.uint8).cpu(), b["m"][i].view(torch.uint8).cpu())
        one = {k: v[i:i + 1] for k, v in c.items()}
        call(one, 8, False, step=7, seed=3, indices=[i], **KW)
        for k in ("m", "v"):
            assert torch.equal(one[k][0].view(torch.uint8).cpu(), a[k][i].view(torch.uint8).cpu()), (i, k)


@gpu
def test_indices_that_do_not_fit_are_refused():
    t = make([10, 20], torch.float32, torch.float32, 8, False)
    for bad in ([0], [0, 1, 2], [0, -1], [0, 1 << 63], [0, 1.5], ["a", "b"]):
        with pytest.raises(_lib.DgcnnError):
            call(t, 8, False, step=1, indices=bad, **KW)
