"""Products grouped by type (dgcnn_amd.layers.grouped_linear) against the formula in 64 bits.

Tolerances: products of 16-bit values are exact in fp32, of fp32 values off by 2^-24; a sum of n terms accumulated in fp32 in any order is off by at most
n 2^-24 sum|t|, and random signs make that sqrt(n): 4 sqrt(n) + 8 is five standard deviations and more.  A result is rounded to its type once more."""
import math

import pytest
import torch

from dgcnn_amd import _lib, layers

gpu = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def inputs(rows, groups, k, n, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)      # noqa: E731
    return r(rows, k).to(dtype), (r(groups, n, k) * k ** -0.5).to(dtype), (r(groups, n) * 0.1).to(dtype), r(rows, n).to(dtype)


def reference(x, w, b, ptr, dy):
    """(value, sum of magnitudes, terms) of each result"""
    X, W, B, G = (t.double() for t in (x, w, b, dy))
    out = {}
    for name, a, z in (("y", 0, None), ("abs", 1, None)):
        f = (lambda t: t.abs()) if a else (lambda t: t)
        y, dx = torch.zeros(X.shape[0], W.shape[1], dtype=torch.float64), torch.zeros_like(X)
        dw, db = torch.zeros_like(W), torch.zeros_like(B)
        for e, (lo, hi) in enumerate(zip(ptr[:-1].tolist(), ptr[1:].tolist())):
            y[lo:hi] = f(X[lo:hi]) @ f(W[e]).t() + f(B[e])
            dx[lo:hi] = f(G[lo:hi]) @ f(W[e])
            dw[e] = f(G[lo:hi]).t() @ f(X[lo:hi])
            db[e] = f(G[lo:hi]).sum(0)
        out[name] = (y, dx, dw, db)
    most = int((ptr[1:] - ptr[:-1]).max()) if ptr.numel() > 1 else 0
    return [(v, m, n) for v, m, n in zip(out["y"], out["abs"], (X.shape[1] + 1, W.shape[1], most, most))]


def near(got, want, dtype, what):
    v, m, n = want
    got = got.detach().cpu().double()
    tol = (4 * math.sqrt(n) + 8) * U * m
    tol = tol + HALF[dtype] * (v.abs() + tol) + TINY[dtype]
    assert got.shape == v.shape
    bad = ~((got - v).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - v).abs() / tol).max()):.2f} tolerances, first {bad.nonzero()[0].tolist()}"


def run(x, w, b, ptr, dy):
    X, W, B = (t.clone().to("cuda").requires_grad_(True) for t in (x, w, b))
    y = layers.grouped_linear(X, W, ptr.to("cuda"), B)
    return (y, *torch.autograd.grad(y, (X, W, B), dy.to("cuda")))


def check(x, w, b, ptr, dy):
    for got, want, what in zip(run(x, w, b, ptr, dy), reference(x, w, b, ptr, dy), ("y", "dx", "dweight", "dbias")):
        assert got.dtype == x.dtype
        near(got, want, x.dtype, what)


@gpu
@pytest.mark.parametrize("sizes", [[5, 60, 0, 33], [0, 0, 1], [129]])
@pytest.mark.parametrize("k,n", [(32, 32), (97, 40), (64, 136), (7, 3), (24, 72), (130, 66), (1, 1)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_small(dtype, k, n, sizes):
    ptr = torch.tensor([0] + sizes).cumsum(0)
    check(*inputs(int(ptr[-1]), len(sizes), k, n, dtype)[:3], ptr, inputs(int(ptr[-1]), len(sizes), k, n, dtype)[3])


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,n", [(40, 16), (13, 50)])
def test_rows_outside_every_group(dtype, k, n):
    """in front, behind, and none at all"""
    for ptr, rows in (([7, 20, 20, 60], 90), ([0, 0, 0], 20), ([50, 50], 50)):
        p = torch.tensor(ptr)
        x, w, b, dy = inputs(rows, len(ptr) - 1, k, n, dtype)
        check(x, w, b, p, dy)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_many_groups(dtype):
    """more groups than a wave has lanes, most of them of a few rows or none"""
    g = torch.Generator().manual_seed(1)
    sizes = torch.randint(0, 6, (150,), generator=g)
    sizes[70] = 200
    ptr = torch.cat([torch.zeros(1, dtype=torch.int64), sizes.cumsum(0)])
    x, w, b, dy = inputs(int(ptr[-1]), 150, 16, 24, dtype)
    check(x, w, b, ptr, dy)


@gpu
@pytest.mark.parametrize("dtype,k,n", [(torch.float32, 33, 20), (torch.bfloat16, 32, 48), (torch.float16, 48, 40)])
def test_long_groups_are_summed_in_slices(dtype, k, n):
    ptr = torch.tensor([0, 3000, 3001, 3001, 4700])
    x, w, b, dy = inputs(4700, 4, k, n, dtype)
    check(x, w, b, ptr, dy)


@gpu
@pytest.mark.parametrize("dtype,rows,groups,k,n", [(torch.bfloat16, 20000, 5, 512, 384), (torch.float32, 6000, 3, 200, 260), (torch.float16, 48, 8, 1024, 1024),
                                                   (torch.bfloat16, 1, 4, 1000, 520), (torch.bfloat16, 9000, 64, 264, 1024)])
def test_large(dtype, rows, groups, k, n):
    if not torch.cuda.is_available():
        pytest.skip("too large for the emulation")
    g = torch.Generator().manual_seed(2)
    cut = torch.sort(torch.randint(0, rows + 1, (groups - 1,), generator=g)).values
    ptr = torch.cat([torch.zeros(1, dtype=torch.int64), cut, torch.tensor([rows])])
    x, w, b, dy = inputs(rows, groups, k, n, dtype)
    check(x, w, b, ptr, dy)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,n", [(40, 1024), (1024, 40), (33, 1030)])
def test_many_rows_and_wide_results(dtype, k, n):
    """enough tiles for the largest form, forward (wide out) and backward (wide in), with groups that end inside tiles and rows of none"""
    if not torch.cuda.is_available():
        pytest.skip("too large for the emulation")
    ptr = torch.tensor([100, 9000, 9000, 9001, 31777, 33000])
    x, w, b, dy = inputs(33300, 5, k, n, dtype)
    check(x, w, b, ptr, dy)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,n", [(64, 96), (50, 33)])
def test_between_few_rows_and_many(dtype, k, n):
    """rows enough for the 128-row tiles at a width that keeps the emulation quick"""
    ptr = torch.tensor([0, 700, 703, 2900])
    if dtype == torch.float32:
        n += 200
    x, w, b, dy = inputs(2900 if torch.cuda.is_available() else 1500, 3, k, n, dtype)
    ptr = ptr.clamp_max(x.shape[0])
    check(x, w, b, ptr, dy)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_views_and_alignment(dtype):
    """rows with a stride, a start in the middle of a vector, a transposed x, an int32 ptr, an expanded dy, no bias"""
    x, w, b, dy = inputs(70, 3, 16, 24, dtype)
    ptr = torch.tensor([0, 30, 31, 70])
    want = reference(x, w, torch.zeros_like(b), ptr, torch.ones_like(dy))
    wide = torch.full((70, 48), 9.0, dtype=dtype).to("cuda")
    wide[:, 16:32] = x.to("cuda")
    buf = torch.empty(70 * 16 + 3, dtype=dtype).to("cuda")
    off = buf[3:].view(70, 16)
    off.copy_(x.to("cuda"))
    for X in (wide[:, 16:32], off, x.to("cuda").t().contiguous().t()):
        X = X.detach().requires_grad_(True)
        W = w.clone().to("cuda").requires_grad_(True)
        y = layers.grouped_linear(X, W, ptr.to(torch.int32).to("cuda"))
        dx, dw = torch.autograd.grad(y.sum(), (X, W))
        for got, k in ((y, 0), (dx, 1), (dw, 2)):
            near(got, want[k], dtype, f"result {k}")


@gpu
def test_each_gradient_alone():
    x, w, b, dy = inputs(50, 2, 12, 20, torch.float32)
    ptr = torch.tensor([0, 20, 50])
    want = reference(x, w, b, ptr, dy)
    for k in range(3):
        args = [t.clone().to("cuda") for t in (x, w, b)]
        args[k].requires_grad_(True)
        y = layers.grouped_linear(args[0], args[1], ptr.to("cuda"), args[2])
        near(torch.autograd.grad(y, args[k], dy.to("cuda"))[0], want[k + 1], torch.float32, f"gradient {k}")


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_non_finite_rows_stay_in_their_group(dtype):
    """NaN in one group's rows and weights, and in rows of no group, reaches no other group -- padding is zeros, not garbage times zero"""
    x, w, b, dy = inputs(100, 3, 20, 12, dtype)
    ptr = torch.tensor([10, 40, 45, 90])
    x[41], dy[42], w[1, 3], x[95], dy[3] = (float("nan"),) * 5
    y, dx, dw, db = (t.detach().cpu() for t in run(x, w, b, ptr, dy))
    for t in (y, dx):
        assert torch.isfinite(t[:40]).all() and torch.isfinite(t[45:]).all()
    assert torch.isnan(y[41]).all() and torch.isnan(dw[1]).any()
    assert torch.isfinite(dw[0]).all() and torch.isfinite(dw[2]).all() and torch.isfinite(db[0]).all() and torch.isfinite(db[2]).all()
    assert not y[:10].any() and not y[90:].any() and not dx[:10].any() and not dx[90:].any()


@gpu
@pytest.mark.parametrize("ptr", [[0, 40, 10, 64], [0, 100, 200, 300], [-5, -1, 20, 64], [0, 64, 0, 64]])
def test_a_ptr_that_does_not_ascend_reads_nothing_outside(ptr):
    x, w, b, dy = inputs(64, 3, 8, 8, torch.float32)
    guard = torch.full((64 * 8 + 512,), 7.0).to("cuda")
    X = guard[256:256 + 512].view(64, 8)
    X.copy_(x.to("cuda"))
    X = X.detach().requires_grad_(True)
    W = w.clone().to("cuda").requires_grad_(True)
    y = layers.grouped_linear(X, W, torch.tensor(ptr).to("cuda"))
    torch.autograd.grad(y, (X, W), dy.to("cuda"))
    assert (guard[:256] == 7).all() and (guard[256 + 512:] == 7).all()


@gpu
def test_no_rows_and_no_groups():
    for rows, groups in ((0, 3), (4, 0), (0, 0)):
        x, w, b = (torch.ones(*s).to("cuda").requires_grad_(True) for s in ((rows, 5), (groups, 6, 5), (groups, 6)))
        y = layers.grouped_linear(x, w, torch.zeros(groups + 1, dtype=torch.int64).to("cuda"), b)
        assert y.shape == (rows, 6) and not y.any()
        for t, g in zip((x, w, b), torch.autograd.grad(y, (x, w, b), torch.ones_like(y))):
            assert g.shape == t.shape and not g.any()


@gpu
def test_gradient_against_differences():
    """the product is linear in each argument: a difference of step 1/8 is the slope up to rounding (2^-24 * 8 of the values)"""
    x, w, b, dy = inputs(40, 2, 11, 9, torch.float32)
    ptr = torch.tensor([0, 15, 40])
    _, *grads = run(x, w, b, ptr, dy)
    f = lambda X, W, B: float((layers.grouped_linear(X.to("cuda"), W.to("cuda"), ptr.to("cuda"), B.to("cuda")).detach().cpu().double() * dy.double()).sum())      # noqa: E731
    g = torch.Generator().manual_seed(1)
    for k, grad in enumerate(grads):
        args = [x, w, b]
        v = torch.randn(args[k].shape, generator=g)
        hi, lo = list(args), list(args)
        hi[k], lo[k] = args[k] + v / 8, args[k] - v / 8
        want = float((grad.cpu().double() * v.double()).sum())
        assert abs((f(*hi) - f(*lo)) * 4 - want) <= 1e-4 * (abs(want) + float(grad.cpu().norm()))


@gpu
def test_module():
    torch.manual_seed(0)
    m = layers.GroupedLinear(3, 10, 6).to("cuda")
    x = torch.randn(20, 10)
    ptr = torch.tensor([0, 5, 5, 20])
    y = m(x.to("cuda"), ptr.to("cuda"))
    near(y, reference(x, m.weight.detach().cpu(), m.bias.detach().cpu(), ptr, torch.zeros(20, 6))[0], torch.float32, "y")
    y.sum().backward()
    assert m.weight.grad.shape == (3, 6, 10) and not m.weight.grad[1].any() and m.bias.grad[0].cpu().tolist() == [5.0] * 6
    assert set(m.state_dict()) == {"weight", "bias"} and layers.GroupedLinear(2, 3, 4, bias=False).bias is None


@gpu
def test_equal_calls_give_equal_bits_and_streams_do_not_meet():
    if not torch.cuda.is_available():
        pytest.skip("second streams are not emulated")
    x, w, b, dy = (t.cuda() for t in inputs(9000, 4, 96, 160, torch.bfloat16))
    ptr = torch.tensor([0, 10, 4000, 4001, 8800], device="cuda")
    first = run(x, w, b, ptr, dy)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    out = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                out.append(run(x, w, b, ptr, dy))
    torch.cuda.synchronize()
    for o in out:
        assert all(torch.equal(p, q) for p, q in zip(first, o))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_forward_and_backward_in_a_graph_with_other_groups_at_each_replay(dtype):
    if not torch.cuda.is_available():
        pytest.skip("graphs need the GPU")
    x, w, b, dy = (t.cuda() for t in inputs(3000, 3, 64, 80, dtype))
    ptr = torch.tensor([0, 1000, 2500, 3000], device="cuda")
    X, W, B = (t.clone().requires_grad_(True) for t in (x, w, b))

    def step():
        y = layers.grouped_linear(X, W, ptr, B)
        return (y, *torch.autograd.grad(y, (X, W, B), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k, p in enumerate(([0, 1000, 2500, 3000], [0, 3000, 3000, 3000], [5, 6, 7, 2000], [0, 0, 1500, 3000])):
        ptr.copy_(torch.tensor(p))
        graph.replay()
        torch.cuda.synchronize()
        want = run(x, w, b, ptr, dy)
        assert all(torch.equal(p, q) for p, q in zip(out, want)), k


@gpu
def test_the_largest_form_in_a_graph():
    """128 KB of LDS, which is asked for at the call, also where the call is captured"""
    if not torch.cuda.is_available():
        pytest.skip("graphs need the GPU")
    x, w, b, _ = (t.cuda() for t in inputs(33000, 2, 64, 1024, torch.bfloat16))
    ptr = torch.tensor([0, 20000, 33000], device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layers.grouped_linear(x, w, ptr, b)
    for p in ([0, 20000, 33000], [0, 1, 32999], [300, 300, 33000]):
        ptr.copy_(torch.tensor(p))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, layers.grouped_linear(x, w, ptr, b)), p


@gpu
def test_rows_of_unusual_strides():
    """one row with any stride, rows too far apart for 32-bit offsets, expanded rows: as if contiguous"""
    x, w, b, _ = (t.to("cuda") for t in inputs(3, 1, 16, 8, torch.float32))
    ptr = torch.tensor([0, 3]).to("cuda")
    far = torch.zeros(2, 1 << 22).to("cuda")
    far[:, :16] = x[:2]
    want = layers.grouped_linear(x, w, ptr, b)
    assert torch.equal(layers.grouped_linear(far[:, :16], w, ptr.clamp_max(2), b), want[:2])
    assert torch.equal(layers.grouped_linear(far[:1, :16], w, ptr.clamp_max(1), b), want[:1])
    assert torch.equal(layers.grouped_linear(x[:1].expand(3, 16), w, ptr, b), want[:1].expand(3, 8))


@gpu
def test_refusals_on_device_tensors():
    x, w, b, _ = (t.to("cuda") for t in inputs(10, 2, 6, 4, torch.float32))
    ptr = torch.tensor([0, 4, 10]).to("cuda")
    bad = [lambda: layers.grouped_linear(x, w[:, :, :5], ptr), lambda: layers.grouped_linear(x, w[0], ptr), lambda: layers.grouped_linear(x[0], w, ptr),
           lambda: layers.grouped_linear(x, w.half(), ptr), lambda: layers.grouped_linear(x.double(), w.double(), ptr), lambda: layers.grouped_linear(x, w, ptr[:2]),
           lambda: layers.grouped_linear(x, w, ptr.float()), lambda: layers.grouped_linear(x, w, ptr, b[:, :3]), lambda: layers.grouped_linear(x, w, ptr, b.half()),
           lambda: layers.grouped_linear(x[:, :0], w[:, :, :0], ptr)]
    for f in bad:
        with pytest.raises(_lib.DgcnnError):
            f()


# ---- CPU ------------------------------------------------------------------------------------------------------------------------------
def test_cpu_tensors_are_refused():
    with pytest.raises(_lib.DgcnnError):
        layers.grouped_linear(torch.zeros(4, 8), torch.zeros(1, 2, 8), torch.tensor([0, 4]))


def test_module_constructor_refusals():
    for args in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        with pytest.raises(ValueError):
            layers.GroupedLinear(*args)


def test_c_entries_refuse_bad_arguments():
    import ctypes
    L = _lib.lib()
    ptr = ctypes.addressof((ctypes.c_float * 64)())

    def args(**kw):
        return ctypes.byref(_lib.GroupedLinearArgs(**{**dict(rows=4, ldx=8, in_features=8, out_features=4, groups=2, x=ptr, weight=ptr, ptr=ptr), **kw}))

    fwd = lambda y=ptr, **kw: L.dgcnn_grouped_linear_fwd(args(**kw), y, None)      # noqa: E731
    bwd = lambda dy=ptr, dx=ptr, dw=None, db=None, ws=None, **kw: L.dgcnn_grouped_linear_bwd(args(**kw), dy, dx, dw, db, ws, None)      # noqa: E731
    assert L.dgcnn_grouped_linear_fwd(None, ptr, None) == -1
    for f in (fwd, bwd):
        for kw in (dict(rows=-1), dict(in_features=0), dict(out_features=0), dict(groups=-1), dict(dtype=3), dict(x=None), dict(weight=None), dict(ptr=None), dict(ldx=7)):
            assert f(**kw) == -1, kw
        for kw in (dict(rows=1 << 40), dict(groups=(1 << 20) + 1)):
            assert f(**kw) == -3, kw
    assert fwd(y=None) == -1 and bwd(dy=None) == -1 and bwd(dw=ptr) == -1 and bwd(db=ptr, ws=ptr) == -1
    assert fwd(rows=0, x=None, y=None) == 0
    ask = L.dgcnn_grouped_linear_workspace_bytes
    assert ask(100, 8, 4, 2, 0) > 0 and ask(-1, 8, 4, 2, 0) == -1 and ask(1, 0, 4, 2, 0) == -1 and ask(1, 8, 4, 2, 9) == -1
