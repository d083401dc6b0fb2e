"""What the layer and optimizer entries read and write: every tensor and workspace has exactly its size and lies between guards of bytes 0xff, which are NaN in every
type.  A write outside changes a guard; a read outside, or of a place that nothing wrote, brings a NaN into the results.  With a ptr that does not ascend the values
are unspecified, the bounds are not; the sizes reach the sliced weight gradient and the norm in chunks."""
import ctypes

import pytest
import torch

from dgcnn_amd import _lib

gpu = pytest.mark.gpu
DT = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
GUARD = 4096


class Box:
    """tensors between guards; `shift` bytes off the alignment that torch's own allocations have (workspaces not)"""

    def __init__(self, shift=0):
        self.shift, self.all = shift, []

    def _place(self, nbytes, fill, shift=None):
        buf = torch.full((2 * GUARD + nbytes,), 0xFF, dtype=torch.uint8).to("cuda")
        at = GUARD + (self.shift if shift is None else shift)
        if fill is not None:
            buf[at:at + nbytes] = fill
        self.all.append((buf, at, nbytes))
        return buf[at:at + nbytes]

    def put(self, t):
        out = self._place(t.numel() * t.element_size(), None).view(t.dtype).view(t.shape)
        out.copy_(t.to("cuda"))
        return out

    def out(self, shape, dtype, clean):
        n = 1
        for s in shape:
            n *= s
        return self._place(n * dtype.itemsize, 0 if clean else None, self.shift // dtype.itemsize * dtype.itemsize).view(dtype).view(shape)

    def space(self, nbytes, clean):
        return self._place(nbytes, 0 if clean else None, 0)

    def check(self):
        for buf, at, n in self.all:
            b = buf.cpu()
            assert (b[:at] == 0xFF).all() and (b[at + n:] == 0xFF).all()


def stream():
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device() if torch.cuda.is_available() else 0)


def ok(rc):
    assert rc == 0, rc


def finite(*ts):
    for t in ts:
        assert torch.isfinite(t.cpu().float()).all()


def ptrs(rows):
    return {"good": [0, rows // 5, rows // 5, rows - 700, rows], "good_in_part": [7, 9, 500, 501, rows - 3], "crossed": [0, rows - 100, 100, rows - 50, rows],
            "too_far": [0, 2 * rows, 3 * rows, 1 << 40, 1 << 62], "negative": [-(1 << 62), -5, rows // 2, rows // 2 - 1, rows], "descending": [rows, rows // 2, 0, rows, 0],
            "all_behind": [rows + 1] * 5}


NAMES = sorted(ptrs(1000))


@gpu
@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("dtype,rows,fin,fout,shift", [(torch.float32, 1700, 24, 40, 0), (torch.bfloat16, 1700, 24, 40, 0), (torch.float32, 1300, 13, 7, 4),
                                                       (torch.float16, 1300, 13, 7, 2), (torch.bfloat16, 3000, 72, 136, 0)])
def test_grouped_linear(dtype, rows, fin, fout, shift, name):
    g = torch.Generator().manual_seed(1)
    good, groups, box = name.startswith("good"), 4, Box(shift)
    x, w, b, dy = (box.put(torch.randn(s, generator=g).to(dtype)) for s in ((rows, fin), (groups, fout, fin), (groups, fout), (rows, fout)))
    ptr = torch.tensor(ptrs(rows)[name]).to("cuda")
    a = _lib.GroupedLinearArgs(rows, fin, fin, fout, groups, DT[dtype], x.data_ptr(), w.data_ptr(), b.data_ptr(), ptr.data_ptr())
    L = _lib.lib()
    y, dx = box.out((rows, fout), dtype, not good), box.out((rows, fin), dtype, not good)
    dw, db = box.out(tuple(w.shape), dtype, not good), box.out(tuple(b.shape), dtype, not good)
    nbytes = L.dgcnn_grouped_linear_workspace_bytes(rows, fin, fout, groups, DT[dtype])
    assert nbytes > 256                       # (the weight gradient is sliced)
    ws = box.space(nbytes, not good)
    ok(L.dgcnn_grouped_linear_fwd(ctypes.byref(a), y.data_ptr(), stream()))
    ok(L.dgcnn_grouped_linear_bwd(ctypes.byref(a), dy.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(), ws.data_ptr(), stream()))
    box.check()
    finite(y, dx, dw, db)


@gpu
@pytest.mark.parametrize("name", NAMES + ["dense"])
@pytest.mark.parametrize("dtype,rows,C,groups,shift", [(torch.float32, 6000, 32, 4, 0), (torch.bfloat16, 9000, 33, 3, 0), (torch.float32, 3000, 48, 2, 4),
                                                       (torch.float16, 9000, 32, 1, 2), (torch.float32, 1500, 16, 4, 0)])
def test_group_norm(dtype, rows, C, groups, shift, name):
    g = torch.Generator().manual_seed(2)
    good, segments, box = name.startswith("good") or name == "dense", 4, Box(shift)
    if name == "dense":
        segments = 3
    x, dy = (box.put(torch.randn(rows, C, generator=g).to(dtype)) for _ in range(2))
    w, b = (box.put(torch.randn(C, generator=g).to(dtype)) for _ in range(2))
    ptr = None if name == "dense" else torch.tensor(ptrs(rows)[name]).to("cuda")
    L = _lib.lib()
    y, dx = (box.out((rows, C), dtype, not good) for _ in range(2))
    dw, db = (box.out((C,), dtype, not good) for _ in range(2))
    mean, rstd = (box.out((segments, groups), torch.float32, not good) for _ in range(2))
    a = _lib.GroupNormArgs(rows, C, groups, segments, DT[dtype], DT[dtype], 2, 1e-5, 0, x.data_ptr(), w.data_ptr(), b.data_ptr(), None if ptr is None else ptr.data_ptr(),
                           mean.data_ptr(), rstd.data_ptr())
    wss = [box.space(L.dgcnn_group_norm_workspace_bytes(rows, C, groups, segments, ptr is None, DT[dtype], back), not good) for back in (0, 1)]
    ok(L.dgcnn_group_norm_fwd(ctypes.byref(a), y.data_ptr(), wss[0].data_ptr(), stream()))
    ok(L.dgcnn_group_norm_bwd(ctypes.byref(a), dy.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(), wss[1].data_ptr(), stream()))
    box.check()
    finite(y, dx, dw, db, mean, rstd)


@gpu
@pytest.mark.parametrize("shift", [0, 4])
@pytest.mark.parametrize("dtype,bits,master", [(torch.float32, 32, False), (torch.bfloat16, 32, True), (torch.float32, 8, False), (torch.float16, 8, True)])
def test_adamw(dtype, bits, master, shift):
    g, box, n_of = torch.Generator().manual_seed(3), Box(shift), [1, 7, 255, 257, 2049, 4096, 0, 5000]
    table = (_lib.AdamwTensor * len(n_of))()
    keep, at = [], lambda t: t.data_ptr() if t.numel() else None      # noqa: E731
    for i, n in enumerate(n_of):
        p, gr = (box.put(torch.randn(n, generator=g).to(dtype)) for _ in range(2))
        if bits == 32:
            m, v = (box.put(torch.rand(n, generator=g)) for _ in range(2))
            s = [None, None]
        else:
            m, v = (box.put(torch.randint(0, 0x70, (n,), generator=g, dtype=torch.uint8)) for _ in range(2))
            s = [box.put(torch.rand(-(-n // 256), generator=g)) for _ in range(2)]
        copy = box.put(p.cpu().float()) if master else None
        keep.append([t for t in (p, copy, *s) if t is not None] + ([m, v] if bits == 32 else [m.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn)]))
        table[i] = _lib.AdamwTensor(at(p), at(gr), at(m), at(v), s[0] is not None and at(s[0]) or None, s[1] is not None and at(s[1]) or None,
                                    copy is not None and at(copy) or None, n)
    a = _lib.AdamwArgs(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01, step=3, seed=1, param_dtype=DT[dtype], grad_dtype=DT[dtype], state_bits=bits, count=len(n_of))
    a.tensors = ctypes.addressof(table)
    ok(_lib.lib().dgcnn_adamw_step(ctypes.byref(a), stream()))
    box.check()
    for ts in keep:
        finite(*ts)
