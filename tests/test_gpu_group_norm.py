"""Group norm with an activation (dgcnn_amd.layers.group_norm) against the formula in 64 bits.

Tolerances, U = 2^-24 (half a step of fp32, relative).  A sum is made of at most 128 terms a thread, 32 LDS items and 6 exchanges, then up to 64 partial sums
one after the other: fewer than K = 256 rounded additions on any path, so a sum of t is off by at most K U sum|t|.  That gives, with s the group's deviation,
h off by   dh = K U (1 + |h| + mean|x| / s),   z by dz = |w| dh + 4 U (|z| + |b|),   q = dy act'(z) by dq = |dy| (2 dz + 8 U)   (|act''| < 2), and the
sums of the gradients by the sums of those; a result is rounded to its type once."""
import pytest
import torch

from dgcnn_amd import _lib, layers
from dgcnn_amd.batch import Graph, collate

gpu = pytest.mark.gpu
U, K = 2.0 ** -24, 256
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}
ACT = {"none": lambda z: z, "relu": torch.relu, "silu": lambda z: z * torch.sigmoid(z), "tanh": torch.tanh,
       "gelu": lambda z: 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))}


def segments_of(ptr, rows, shape):
    if ptr is None:
        per = rows // shape[0] if shape[0] else 0
        return [(i * per, (i + 1) * per) for i in range(shape[0])]
    p = ptr.tolist()
    return list(zip(p[:-1], p[1:]))


def reference(x, w, b, ptr, groups, eps, act, dy=None):
    """y (and dx, dw, db) in 64 bits with the tolerance of each"""
    C = x.shape[-1]
    X, W, B = x.double().reshape(-1, C), w.double(), b.double()
    D = C // groups
    y, ty = torch.zeros_like(X), torch.zeros_like(X)
    dx, tdx = torch.zeros_like(X), torch.zeros_like(X)
    dw, db, tdw, tdb = (torch.zeros(C, dtype=torch.float64) for _ in range(4))
    for lo, hi in segments_of(ptr, X.shape[0], x.shape):
        if lo == hi:
            continue
        t = X[lo:hi].reshape(hi - lo, groups, D)
        mean = t.mean((0, 2), keepdim=True)
        var = ((t - mean) ** 2).mean((0, 2), keepdim=True)
        s = (var + eps).sqrt()
        h = ((t - mean) / s).reshape(hi - lo, C)
        spread = lambda v: v.expand(1, groups, D).reshape(1, C)      # noqa: E731
        gm = lambda v: spread(v.reshape(hi - lo, groups, D).mean((0, 2), keepdim=True))      # noqa: E731
        dh = K * U * (1 + h.abs() + spread(t.abs().mean((0, 2), keepdim=True) / s))
        z = (h * W + B).detach().requires_grad_(True)
        dz = W.abs() * dh + 4 * U * (z.detach().abs() + B.abs())
        out = ACT[act](z)
        y[lo:hi] = out.detach()
        ty[lo:hi] = 1.2 * dz + 8 * U * out.detach().abs()
        if dy is None:
            continue
        (slope,) = torch.autograd.grad(out.sum(), z)
        DY = dy.double().reshape(-1, C)[lo:hi]
        q = DY * slope
        dq = DY.abs() * (2 * dz + 8 * U)
        if act == "relu":
            dq = torch.where(z.detach().abs() <= dz, DY.abs(), torch.zeros_like(dq) + U * DY.abs())
        a, c = gm(q * W), gm(q * W * h)
        rs = spread(1 / s)
        dx[lo:hi] = rs * (q * W - a - h * c)
        e = dq * W.abs()
        tdx[lo:hi] = rs * (e + gm(e) + h.abs() * gm(e * h.abs() + (q * W).abs() * dh) + dh * c.abs()
                           + K * U * ((q * W).abs() + gm((q * W).abs()) + h.abs() * gm((q * W * h).abs())))
        dw += (q * h).sum(0); tdw += (dq * h.abs() + q.abs() * dh).sum(0) + K * U * (q * h).abs().sum(0)
        db += q.sum(0); tdb += dq.sum(0) + K * U * q.abs().sum(0)
    return dict(y=(y, ty), dx=(dx, tdx), dw=(dw, tdw), db=(db, tdb))


def near(got, want, dtype, what):
    v, tol = want
    got = got.detach().cpu().double().reshape(v.shape)
    tol = tol + HALF[dtype] * (v.abs() + tol) + TINY[dtype]
    bad = (got - v).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - v).abs() / tol).max()):.2f} tolerances"


def inputs(rows, C, dtype, wdtype=None, seed=0, shape=None):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, C, generator=g) * (0.5 + torch.rand(C, generator=g)) + torch.randn(C, generator=g)).to(dtype)
    w = (1 + 0.2 * torch.randn(C, generator=g)).to(wdtype or dtype)
    b = (0.2 * torch.randn(C, generator=g)).to(wdtype or dtype)
    dy = torch.randn(rows, C, generator=g).to(dtype)
    return (x.view(shape), w, b, dy.view(shape)) if shape else (x, w, b, dy)


def run(x, w, b, dy, ptr, groups, act, eps=1e-5):
    X, W, B = (t.clone().to("cuda").requires_grad_(True) for t in (x, w, b))
    y = layers.group_norm(X, groups, W, B, ptr=None if ptr is None else ptr.to("cuda"), act=act, eps=eps)
    return (y, *torch.autograd.grad(y, (X, W, B), dy.to("cuda")))


def check(x, w, b, dy, ptr, groups, act, eps=1e-5):
    want = reference(x, w, b, ptr, groups, eps, act, dy)
    y, dx, dw, db = run(x, w, b, dy, ptr, groups, act, eps)
    assert y.dtype == dx.dtype == x.dtype and dw.dtype == w.dtype and y.shape == x.shape
    near(y, want["y"], x.dtype, "y"); near(dx, want["dx"], x.dtype, "dx")
    near(dw, want["dw"], w.dtype, "dweight"); near(db, want["db"], w.dtype, "dbias")


PTRS = {
    "graphs": [0, 17, 40, 41, 90],
    "empty": [0, 0, 0, 5, 5, 30, 30],           # empty ones in front, in the middle, at the end
    "one_row": [0, 1, 2, 3],
    "covered_in_part": [3, 10, 50],             # rows 0..2 and those behind 50 lie in no segment
    "one": [0, 77],
}


@gpu
@pytest.mark.parametrize("ptr", sorted(PTRS))
@pytest.mark.parametrize("C,groups", [(32, 4), (97, 1), (12, 3), (6, 6)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_ragged(dtype, C, groups, ptr):
    p = torch.tensor(PTRS[ptr])
    rows = int(p[-1]) + (13 if ptr == "covered_in_part" else 0)
    check(*inputs(rows, C, dtype), p, groups, "silu")


@gpu
@pytest.mark.parametrize("act", sorted(ACT))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_activations(dtype, act):
    check(*inputs(60, 40, dtype, seed=3), torch.tensor([0, 25, 60]), 5, act)


@gpu
@pytest.mark.parametrize("shape,groups", [((2, 5, 7, 16), 4), ((3, 1, 10), 5), ((4, 8), 2), ((1, 300, 24), 3), ((2, 3, 66), 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_dense_samples(dtype, shape, groups):
    n = 1
    for s in shape[:-1]:
        n *= s
    check(*inputs(n, shape[-1], dtype, shape=shape), None, groups, "gelu")


@gpu
@pytest.mark.parametrize("dtype,C,groups,lens", [(torch.float32, 64, 8, [700, 3, 0, 1, 900, 64]), (torch.bfloat16, 96, 1, [1500, 2, 40]),
                                                 (torch.float32, 33, 3, [2500, 10, 5])])
def test_long_segments_are_split(dtype, C, groups, lens):
    """more than 256 KB of rows with segments longer than a workgroup holds: the two-launch form, with rows in front and behind"""
    p = torch.tensor([5] + lens).cumsum(0)
    check(*inputs(int(p[-1]) + 50, C, dtype, seed=7), p, groups, "tanh")


@gpu
@pytest.mark.parametrize("dtype,shape,groups", [(torch.bfloat16, (2, 40, 32, 128), 32), (torch.float32, (3, 700, 50), 1)])
def test_long_dense_samples_are_split(dtype, shape, groups):
    n = 1
    for s in shape[:-1]:
        n *= s
    check(*inputs(n, shape[-1], dtype, seed=8, shape=shape), None, groups, "silu")


@gpu
def test_weights_of_another_type_and_absent_ones():
    x, w, b, dy = inputs(50, 24, torch.bfloat16, wdtype=torch.float32)
    ptr = torch.tensor([0, 20, 50])
    check(x, w, b, dy, ptr, 3, "silu")
    one, zero = torch.ones(24), torch.zeros(24)
    want = reference(x, one, zero, ptr, 3, 1e-5, "none", dy)
    X = x.clone().to("cuda").requires_grad_(True)
    y = layers.group_norm(X, 3, ptr=ptr.to("cuda"))
    near(y, want["y"], x.dtype, "y")
    near(torch.autograd.grad(y, X, dy.to("cuda"))[0], want["dx"], x.dtype, "dx")
    W = one.to("cuda").requires_grad_(True)
    y = layers.group_norm(x.to("cuda"), 3, weight=W, ptr=ptr.to("cuda"))
    near(torch.autograd.grad(y, W, dy.to("cuda"))[0], want["dw"], torch.float32, "dweight alone")


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_views_and_alignment(dtype):
    """an x that starts in the middle of a vector, one with strides, an int32 ptr, a dy that is expanded"""
    x, w, b, dy = inputs(64, 16, dtype)
    ptr = torch.tensor([0, 30, 64])
    want = reference(x, w, b, ptr, 2, 1e-5, "relu", dy)
    buf = torch.empty(64 * 16 + 1, dtype=dtype).to("cuda")
    off = buf[1:].view(64, 16)
    off.copy_(x.to("cuda"))
    wide = torch.zeros(64, 40, dtype=dtype).to("cuda")
    wide[:, 8:24] = x.to("cuda")
    for X in (off, wide[:, 8:24]):
        X = X.detach().requires_grad_(True)
        y = layers.group_norm(X, 2, w.to("cuda"), b.to("cuda"), ptr=ptr.to(torch.int32).to("cuda"), act="relu")
        near(y, want["y"], dtype, "y")
        near(torch.autograd.grad(y, X, dy.to("cuda"))[0], want["dx"], dtype, "dx")
    X = x.clone().to("cuda").requires_grad_(True)
    y = layers.group_norm(X, 2, w.to("cuda"), b.to("cuda"), ptr=ptr.to("cuda"))
    (dx,) = torch.autograd.grad(y.sum(), X)
    near(dx, reference(x, w, b, ptr, 2, 1e-5, "none", torch.ones_like(dy))["dx"], dtype, "dx of a sum")


@gpu
def test_large_mean_does_not_cancel():
    """x = 1000 + noise: the squares' difference would lose the variance altogether (1000^2 U = 0.06)"""
    x, w, b, dy = inputs(200, 32, torch.float32)
    check(x + 1000, w, b, dy, torch.tensor([0, 90, 200]), 4, "none")


@gpu
def test_constant_and_non_finite_segments_stay_to_themselves():
    x, w, b, dy = inputs(90, 16, torch.float32)
    x[:30] = 2.5                       # variance 0: y = act(b)
    x[40, 3] = float("nan")
    x[70, 9] = float("inf")
    ptr = torch.tensor([0, 30, 60, 80, 90])
    y, dx, _, _ = run(x, w, b, dy, ptr, 2, "none")
    y, dx = y.detach().cpu(), dx.cpu()
    assert torch.equal(y[:30], b.expand(30, 16))
    assert torch.isnan(y[30:60, :8]).all() and torch.isfinite(y[30:60, 8:]).all()
    assert torch.isfinite(y[60:80, :8]).all() and torch.isnan(y[70, 9])
    assert torch.isfinite(y[80:]).all() and torch.isfinite(dx[80:]).all() and torch.isfinite(dx[:30]).all()


@gpu
@pytest.mark.parametrize("ptr", [[0, 40, 10, 64], [0, 100, 200, 300], [-5, -1, 20, 64]])
def test_a_ptr_that_does_not_ascend_reads_nothing_outside(ptr):
    """unspecified values, but inside the tensors: guards around them keep theirs"""
    x, w, b, dy = inputs(64, 8, torch.float32)
    guard = torch.full((64 * 8 + 512,), 7.0).to("cuda")
    X = guard[256:256 + 512].view(64, 8)
    X.copy_(x.to("cuda"))
    X = X.detach().requires_grad_(True)
    y = layers.group_norm(X, 2, w.to("cuda"), b.to("cuda"), ptr=torch.tensor(ptr).to("cuda"))
    torch.autograd.grad(y, X, dy.to("cuda"))
    assert (guard[:256] == 7).all() and (guard[256 + 512:] == 7).all()


@gpu
def test_no_rows_and_no_segments():
    w, b = torch.ones(8).to("cuda").requires_grad_(True), torch.zeros(8).to("cuda").requires_grad_(True)
    for x, ptr in ((torch.zeros(0, 8), [0, 0, 0]), (torch.randn(5, 8), [0]), (torch.zeros(0, 8), [0])):
        X = x.to("cuda").requires_grad_(True)
        y = layers.group_norm(X, 2, w, b, ptr=torch.tensor(ptr).to("cuda"), act="silu")
        dx, dw, db = torch.autograd.grad(y.sum() if y.numel() else y, (X, w, b), None if y.numel() else torch.zeros_like(y))
        assert y.shape == x.shape and not y.any() and not dx.any() and not dw.any() and not db.any()
    y = layers.group_norm(torch.zeros(0, 3, 8).to("cuda"), 2, w, b)
    assert y.shape == (0, 3, 8)


@gpu
def test_gradient_against_differences():
    """along random directions, step 1/64: the third derivative's share is below 1e-3 of the values here, rounding 2^-24 * 64 below 1e-5"""
    x, w, b, dy = inputs(40, 12, torch.float32, seed=5)
    ptr = torch.tensor([0, 11, 40])
    _, dx, dw, db = run(x, w, b, dy, ptr, 3, "silu")
    f = lambda X, W, B: float((layers.group_norm(X.to("cuda"), 3, W.to("cuda"), B.to("cuda"), ptr=ptr.to("cuda"), act="silu").detach().cpu().double() * dy.double()).sum())      # noqa: E731
    g = torch.Generator().manual_seed(1)
    for k, grad in enumerate((dx, dw, db)):
        args = [x, w, b]
        v = torch.randn(args[k].shape, generator=g)
        hi, lo = list(args), list(args)
        hi[k], lo[k] = args[k] + v / 64, args[k] - v / 64
        slope = (f(*hi) - f(*lo)) * 32
        want = float((grad.cpu().double() * v.double()).sum())
        assert abs(slope - want) <= 1e-3 * (abs(want) + float(grad.cpu().norm()))


@gpu
def test_module_on_a_batch_of_graphs():
    torch.manual_seed(0)
    graphs = [Graph(torch.randn(n, 24), torch.tensor([[0], [0]]), 0) for n in (5, 1, 30)]
    batch = collate(graphs).to("cuda")
    ptr = layers.graph_ptr(batch)
    assert ptr.cpu().tolist() == [0, 5, 6, 36]
    m = layers.GroupNorm(4, 24, act="relu").to("cuda")
    y = m(batch.x, ptr)
    want = reference(batch.x.cpu(), m.weight.detach().cpu(), m.bias.detach().cpu(), ptr.cpu(), 4, 1e-5, "relu")
    near(y, want["y"], torch.float32, "y")
    y.square().sum().backward()
    assert m.weight.grad.shape == (24,) and torch.isfinite(m.bias.grad).all()
    assert set(m.state_dict()) == {"weight", "bias"} and not layers.GroupNorm(4, 24, affine=False).state_dict()


@gpu
def test_equal_calls_give_equal_bits_and_streams_do_not_meet():
    if not torch.cuda.is_available():
        pytest.skip("second streams are not emulated")
    x, w, b, dy = (t.cuda() for t in inputs(6000, 128, torch.bfloat16))
    ptr = torch.tensor([0, 10, 3000, 3001, 5800], device="cuda")
    first = run(x, w, b, dy, ptr, 8, "silu")
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    out = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                out.append(run(x, w, b, dy, ptr, 8, "silu"))
    torch.cuda.synchronize()
    for o in out:
        assert all(torch.equal(a, b) for a, b in zip(first, o))


@gpu
def test_forward_and_backward_in_a_graph():
    if not torch.cuda.is_available():
        pytest.skip("graphs need the GPU")
    for lens in ([30, 70, 28], [2000, 1, 1500]):
        ptr = torch.tensor([0] + lens, device="cuda").cumsum(0)
        x, w, b, dy = (t.cuda() for t in inputs(int(ptr[-1]), 64, torch.float32))
        X, W, B = (t.clone().requires_grad_(True) for t in (x, w, b))

        def step():
            y = layers.group_norm(X, 4, W, B, ptr=ptr, act="silu")
            return (y, *torch.autograd.grad(y, (X, W, B), dy))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for k in range(4):
            with torch.no_grad():
                X.copy_(x * (1 + k))
            graph.replay()
            torch.cuda.synchronize()
            want = run(x * (1 + k), w, b, dy, ptr, 4, "silu")
            assert all(torch.equal(p, q) for p, q in zip(out, want)), (lens, k)


@gpu
@pytest.mark.parametrize("long_rows", [0, 5000, 300000])
def test_workgroups_that_walk_several_segments_and_chunks(long_rows):
    """1100 graphs are more than the workgroups of a role, and so are the chunks of a long one among them"""
    if long_rows > 5000 and not torch.cuda.is_available():
        pytest.skip("too long for the emulation")
    g = torch.Generator().manual_seed(11)
    lens = torch.randint(0, 4, (1100,), generator=g)
    if long_rows:
        lens[700] = long_rows
    ptr = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)])
    check(*inputs(int(ptr[-1]) + 2, 32, torch.float32, seed=4), ptr, 4, "silu")


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_widest_groups_at_odd_addresses(dtype):
    """2048 channels fit a workgroup as vectors only: tensors that are not aligned for them are copied"""
    x, w, b, dy = inputs(5, 2048, dtype, seed=6)
    ptr = torch.tensor([0, 2, 5])

    def odd(t):
        v = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda" if torch.cuda.is_available() else "cpu")[1:].view(t.shape)
        return v.copy_(t)

    X, W, B = odd(x).requires_grad_(True), w.to("cuda").requires_grad_(True), b.to("cuda").requires_grad_(True)
    y = layers.group_norm(X, 1, W, B, ptr=ptr.to("cuda"), act="silu")
    got = (y, *torch.autograd.grad(y, (X, W, B), odd(dy)))
    for p, q in zip(got, run(x, w, b, dy, ptr, 1, "silu")):
        assert torch.equal(p, q)
    check(x, w, b, dy, ptr, 1, "silu")


@gpu
def test_more_segments_than_workgroups():
    if not torch.cuda.is_available():
        pytest.skip("2^17 segments take the emulation minutes")
    n = (1 << 17) + 77
    x = torch.randn(n, 2, 4, generator=torch.Generator().manual_seed(5)).cuda()
    y = layers.group_norm(x, 2, act="tanh")
    ptr = torch.arange(0, 2 * n + 1, 2, device="cuda")
    assert torch.equal(y.view(-1, 4), layers.group_norm(x.view(-1, 4), 2, ptr=ptr, act="tanh"))
    d = x.double().view(n, 2, 2, 2)      # [sample, row, group, channel]
    want = torch.tanh((d - d.mean((1, 3), keepdim=True)) / (d.var((1, 3), correction=0, keepdim=True) + 1e-5).sqrt()).view(n, 2, 4)
    # (|h| <= sqrt(3) for four values; a difference of two values near each other and its root: 16 roundings of the largest value, over a deviation of at
    # least sqrt(eps))
    bound = 16 * 2.0 ** -24 * (1 + d.abs().amax((1, 3), keepdim=True) / (d.var((1, 3), correction=0, keepdim=True) + 1e-5).sqrt())
    assert bool(((y.double() - want).view(n, 2, 2, 2).abs() <= bound).all())


@gpu
def test_refusals_on_device_tensors():
    x, w, b, _ = (t.to("cuda") for t in inputs(10, 12, torch.float32))
    ptr = torch.tensor([0, 4, 10]).to("cuda")
    bad = [lambda: layers.group_norm(x, 5, w, b, ptr=ptr), lambda: layers.group_norm(x, 0), lambda: layers.group_norm(x, 3, act="elu"),
           lambda: layers.group_norm(x, 3, w[:4], b), lambda: layers.group_norm(x, 3, w, b.to(torch.bfloat16)), lambda: layers.group_norm(x, 3, eps=-1.0),
           lambda: layers.group_norm(x.double(), 3), lambda: layers.group_norm(x[0], 3), lambda: layers.group_norm(x, 3, ptr=ptr.float()),
           lambda: layers.group_norm(x, 3, ptr=ptr.view(1, -1)), lambda: layers.group_norm(x.view(2, 5, 12), 3, ptr=ptr),
           lambda: layers.group_norm(torch.zeros(2, 1025).to("cuda"), 1)]                       # more columns a group than a workgroup has threads
    for f in bad:
        with pytest.raises(_lib.DgcnnError):
            f()


# ---- CPU ------------------------------------------------------------------------------------------------------------------------------
def test_cpu_tensors_are_refused():
    with pytest.raises(_lib.DgcnnError):
        layers.group_norm(torch.zeros(4, 8), 2)


def test_module_constructor_refusals():
    for kw in (dict(num_groups=3), dict(num_groups=0), dict(act="swish")):
        with pytest.raises(ValueError):
            layers.GroupNorm(**{**dict(num_groups=2, num_channels=8), **kw})


def test_c_entries_refuse_bad_arguments():
    import ctypes
    L = _lib.lib()
    buf = (ctypes.c_float * 64)()
    ptr = ctypes.addressof(buf)

    def args(**kw):
        return _lib.GroupNormArgs(**{**dict(rows=4, channels=8, groups=2, segments=2, eps=1e-5, x=ptr, mean=ptr, rstd=ptr), **kw})

    def fwd(y=ptr, ws=ptr, **kw):
        return L.dgcnn_group_norm_fwd(ctypes.byref(args(**kw)), y, ws, None)

    def bwd(dy=ptr, dx=ptr, ws=ptr, **kw):
        return L.dgcnn_group_norm_bwd(ctypes.byref(args(**kw)), dy, dx, None, None, ws, None)

    assert L.dgcnn_group_norm_fwd(None, ptr, ptr, None) == -1
    for f in (fwd, bwd):
        for kw in (dict(rows=-1), dict(channels=0), dict(groups=3), dict(groups=0), dict(segments=-1), dict(dtype=5), dict(act=9), dict(eps=-1.0), dict(eps=float("nan")),
                   dict(x=None), dict(mean=None), dict(rstd=None), dict(segments=3), dict(segments=0), dict(weight=ptr, weight_dtype=9), dict(ws=None)):
            assert f(**kw) == -1, kw
        assert f(rows=1 << 41, segments=1) == -3
        assert f(channels=1025, groups=1) == -3
        assert f(rows=0, segments=0) == 0
    assert fwd(y=None) == -1 and bwd(dy=None) == -1 and bwd(dx=None) == -1
    ask = L.dgcnn_group_norm_workspace_bytes
    assert ask(100, 8, 2, 3, 0, 0, 1) > 0 and ask(0, 8, 2, 0, 1, 0, 0) > 0
    assert ask(-1, 8, 2, 3, 0, 0, 1) == -1 and ask(4, 8, 3, 3, 0, 0, 1) == -1 and ask(4, 8, 2, 2, 0, 7, 1) == -1


def test_counts_beyond_the_grids_are_refused():
    import ctypes
    L = _lib.lib()
    buf = (ctypes.c_float * 64)()
    at = ctypes.addressof(buf)
    for kw in (dict(channels=1 << 25, groups=1 << 25), dict(segments=1 << 28, rows=1 << 28)):
        a = _lib.GroupNormArgs(**{**dict(rows=4, channels=8, groups=2, segments=2, eps=1e-5, x=at, mean=at, rstd=at), **kw})
        assert L.dgcnn_group_norm_fwd(ctypes.byref(a), at, at, None) == -3
        assert L.dgcnn_group_norm_bwd(ctypes.byref(a), at, at, None, None, at, None) == -3
        assert L.dgcnn_group_norm_workspace_bytes(a.rows, a.channels, a.groups, a.segments, 1, 0, 0) == -3
