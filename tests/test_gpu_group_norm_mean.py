"""Group norm where the mean is large against the deviation (constant segments, small noise on an offset), in all three forms of the kernel: a segment in one
workgroup's registers, streamed through them, and cut into chunks.

Tolerances, U = 2^-24.  The mean is a sum of t = x - m over a first, rounded mean m, added to m: the sum is off by K U sum|t| (K = 256 rounded additions on any
path), m only passes into t, exactly.  So the mean is off by its own rounding, U |mean| -- and in the form of chunks by those of the chunks' means and of their
first one too, 3 U |mean| in all -- and by K U mean|t|, where |t| is at most s, the root of the variance + eps, plus K U |x|.  The variance is off by K U of itself and by what
the mean's error shifts it.  Together    dh = (1 + |h|) (4 K U + (3 U + (K U)^2) max|x| / s)
for h = (x - mean) / s.   y = h w + b:  |w| dh + 4 U (|h w| + |b|).   dx = (q w - a - h c) / s, dw = sum q h, db = sum q, with q = dy: sums are off by K U of the sum
of their terms' magnitudes, and what holds h by dh."""
import pytest
import torch

from dgcnn_amd import layers

gpu = pytest.mark.gpu
U, K = 2.0 ** -24, 256
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def check(x, w, b, dy, lens, groups, eps=1e-5, dense=False):
    C = x.shape[1]
    D = C // groups
    ptr = torch.tensor([0] + lens).cumsum(0)
    X, W, B = (t.clone().to("cuda").requires_grad_(True) for t in (x, w, b))
    if dense:
        y = layers.group_norm(X.view(len(lens), -1, C), groups, W, B, eps=eps).view(-1, C)
    else:
        y = layers.group_norm(X, groups, W, B, ptr=ptr.to("cuda"), eps=eps)
    dx, dw, db = (g.cpu().double() for g in torch.autograd.grad(y, (X, W, B), dy.to("cuda")))
    y = y.detach().cpu().double()
    x, w, b, dy, half = x.double(), w.double(), b.double(), dy.double(), HALF[x.dtype]
    sums = torch.zeros(4, C, dtype=torch.float64)      # dw, db and their tolerances
    for lo, hi in zip(ptr[:-1].tolist(), ptr[1:].tolist()):
        if lo == hi:
            continue
        t = x[lo:hi].view(hi - lo, groups, D)
        spread = lambda v: v.expand(1, groups, D).reshape(1, C)      # noqa: E731
        gm = lambda v: spread(v.reshape(hi - lo, groups, D).mean((0, 2), keepdim=True))      # noqa: E731
        mean = t.mean((0, 2), keepdim=True)
        s = (((t - mean) ** 2).mean((0, 2), keepdim=True) + eps).sqrt()
        top = spread(t.abs().amax((0, 2), keepdim=True) / s)
        h, s = ((t - mean) / s).reshape(hi - lo, C), spread(s)
        dh = (1 + h.abs()) * (4 * K * U + (3 * U + (K * U) ** 2) * top)

        def near(got, want, tol, what):
            tol = tol + half * (want.abs() + tol) + 1e-37
            assert ((got - want).abs() <= tol).all(), (what, float(((got - want).abs() / tol).max()), float((got - want).abs().max()))

        near(y[lo:hi], h * w + b, w.abs() * dh + 4 * U * ((h * w).abs() + b.abs()), "y")
        q = dy[lo:hi]
        a, c = gm(q * w), gm(q * w * h)
        e = gm((q * w).abs() * dh)
        near(dx[lo:hi], (q * w - a - h * c) / s,
             (4 * dh * ((q * w).abs() + a.abs() + (h * c).abs()) + dh * c.abs() + h.abs() * e
              + K * U * ((q * w).abs() + gm((q * w).abs()) + h.abs() * gm((q * w * h).abs()))) / s, "dx")
        sums += torch.stack([(q * h).sum(0), q.sum(0), (q.abs() * dh).sum(0) + K * U * (q * h).abs().sum(0), K * U * q.abs().sum(0)])
    wh = HALF[W.dtype]
    for got, want, tol in ((dw, sums[0], sums[2]), (db, sums[1], sums[3])):
        assert ((got - want).abs() <= tol + wh * (want.abs() + tol) + 1e-37).all(), float((got - want).abs().max())


def affine(rows, C, seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (1 + 0.2 * torch.randn(C, generator=g)).to(dtype), (0.25 + 0.1 * torch.randn(C, generator=g)).to(dtype), torch.randn(rows, C, generator=g).to(dtype), g


# rows of 32 channels: within a workgroup's registers; streamed (at most 512 KB in all); in chunks
FORMS = {"whole": [120, 200, 1, 0, 77], "streamed": [4000], "streamed_some": [5, 3000, 400, 1], "chunks": [6000, 3, 2500]}


@gpu
@pytest.mark.parametrize("form", sorted(FORMS))
@pytest.mark.parametrize("value", [0.1, 3.3, -1000.1, 16777.215])
def test_a_constant_segment_gives_exactly_the_bias(form, value):
    """y = b to the last bit, dw = 0 and a finite dx, also where n times the value is no fp32 number"""
    rows = sum(FORMS[form])
    w, b, dy, _ = affine(rows, 32)
    x = torch.full((rows, 32), value)
    ptr = torch.tensor([0] + FORMS[form]).cumsum(0)
    for groups in (1, 4):
        X, W, B = (t.clone().to("cuda").requires_grad_(True) for t in (x, w, b))
        y = layers.group_norm(X, groups, W, B, ptr=ptr.to("cuda"))
        dx, dw, db = torch.autograd.grad(y, (X, W, B), dy.to("cuda"))
        assert torch.equal(y.detach().cpu(), b.expand(rows, 32))
        assert not dw.cpu().any() and torch.isfinite(dx.cpu()).all()
    check(x, w, b, dy, FORMS[form], 4)


@gpu
@pytest.mark.parametrize("form", sorted(FORMS))
@pytest.mark.parametrize("offset,noise", [(100.1, 1e-3), (1000.1, 1e-2), (-7.7, 1e-4), (3.3, 1.0)])
def test_small_noise_on_an_offset(form, offset, noise):
    rows = sum(FORMS[form])
    w, b, dy, g = affine(rows, 32, seed=2)
    x = offset + noise * torch.randn(rows, 32, generator=g)
    check(x, w, b, dy, FORMS[form], 1)
    check(x, w, b, dy, FORMS[form], 8)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("form", sorted(FORMS))
def test_16_bit_offsets(dtype, form):
    rows = sum(FORMS[form])
    w, b, dy, g = affine(rows, 32, seed=4, dtype=dtype)
    x = (200.3 + torch.randn(rows, 32, generator=g)).to(dtype)
    check(x, w, b, dy, FORMS[form], 2)


@gpu
@pytest.mark.parametrize("C,groups,rows", [(33, 3, 3900), (97, 1, 1300), (5, 5, 20000)])
def test_narrow_vectors_streamed(C, groups, rows):
    """one channel a thread: the longest run of rows a thread walks"""
    w, b, dy, g = affine(rows, C, seed=6)
    x = 50.5 + 0.01 * torch.randn(rows, C, generator=g)
    check(x, w, b, dy, [rows], groups)
    check(x.bfloat16(), w.bfloat16(), b.bfloat16(), dy.bfloat16(), [rows], groups)


@gpu
def test_dense_samples():
    w, b, dy, g = affine(6000, 32, seed=8)
    x = 1000.1 + 0.01 * torch.randn(6000, 32, generator=g)
    check(x, w, b, dy, [2000] * 3, 4, dense=True)
    check(x[:3000], w, b, dy[:3000], [1500] * 2, 4, dense=True)


@gpu
def test_a_very_long_segment():
    """more than a thousand chunks: the join adds partial means in long runs too"""
    if not torch.cuda.is_available():
        pytest.skip("too long for the emulation")
    rows = 400000
    w, b, dy, g = affine(rows, 32, seed=9)
    x = 1000.1 + 0.01 * torch.randn(rows, 32, generator=g)
    # (dw, db: a workgroup adds two chunks and the last launch 12 partial rows a lane: still fewer than K)
    check(x, w, b, dy, [rows - 11, 11], 2)
    check(torch.full_like(x, 0.1), w, b, dy, [rows], 1)
