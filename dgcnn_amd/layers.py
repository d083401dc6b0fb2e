"""Layer operators for networks around the graph convolutions: differentiable functions and modules over the node rows of a batch.

* :func:`grouped_linear` / :class:`GroupedLinear` -- a linear map for each type (relation, expert) of the rows, sorted by type.
* :func:`group_norm` / :class:`GroupNorm` -- group norm with an activation, channels last, over every graph of a batch (``ptr``) or over dense
  samples ``[B, ..., C]``.

Rows are the nodes of a :class:`dgcnn_amd.Batch` (or edges, messages, pixels); ``ptr`` says where each graph's rows begin, as
:func:`graph_ptr` returns it.  fp32, bf16 and fp16; sums and statistics in fp32.  Everything runs on the current stream of the tensors' device through
``libdgcnn_hip.so`` without synchronising, and equal inputs at equally aligned addresses give equal bits.  Forward and backward may be captured into a graph; as
with torch's own operators, no eager autograd graph of the same leaves may be alive then (drop its outputs first: its leaves' nodes belong to the eager
stream).  As in the rest of the package there is no CPU fallback: CPU tensors raise :class:`dgcnn_amd._lib.DgcnnError`.  Derivatives are first ones in reverse mode;
forward-mode tangents and function transforms raise.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch import nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "tanh": 4}


def _no(msg: str):
    raise _lib.DgcnnError(msg)


def _no_type(t: torch.Tensor, what: str):
    _no(f"{what} must be float32, bfloat16 or float16, got {t.dtype}")


def _no_gpu():
    _no("dgcnn_amd.layers runs only on an AMD GPU through libdgcnn_hip.so; got a CPU tensor (there is deliberately no CPU fallback)")


def _launch(fn, name: str, device: torch.device, *args) -> None:
    """One call of the library on the current stream of `device`, which has to be the current device for it."""
    index = device.index
    if index is None or index == torch.cuda.current_device():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc, name)


_BYTES = {}      # workspace sizes: pure functions of their arguments (one library call a step otherwise)


def _bytes(name: str, *args) -> int:
    key = (name, *args)
    n = _BYTES.get(key)
    if n is None:
        if len(_BYTES) > 4096:
            _BYTES.clear()
        n = _BYTES[key] = _lib.checked_bytes(getattr(_lib.lib(), name)(*args), name)
    return n


def _check_ptr(ptr: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    if ptr.dim() != 1 or ptr.numel() < 1:
        _no(f"ptr must be [segments + 1], got {tuple(ptr.shape)}")
    if ptr.dtype is not torch.int64 and ptr.dtype is not torch.int32:
        _no(f"ptr must be int64 or int32, got {ptr.dtype}")
    if ptr.get_device() != x.get_device():
        _no(f"ptr on {ptr.device}, x on {x.device}")
    if ptr.dtype is torch.int64 and ptr.is_contiguous():
        return ptr
    return ptr.to(torch.int64).contiguous()


def _wants_grad(*ts) -> bool:
    """Whether autograd has to see the call.  For a forward-mode tangent, which no_grad does not switch off, it raises there: the functions have no rule for it."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in ts):
        return True
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def graph_ptr(data) -> torch.Tensor:
    """``ptr`` [B + 1] (int64, on the batch's device) of a batch: graph ``g`` is rows ``ptr[g] .. ptr[g + 1] - 1``.  No synchronisation where the batch
    knows its ``num_graphs``."""
    batch = data.batch
    n = getattr(data, "num_graphs", None)
    if n is None:
        n = int(batch[-1].item()) + 1 if batch.numel() else 0
    return torch.searchsorted(batch.contiguous(), torch.arange(n + 1, device=batch.device, dtype=batch.dtype))


# ---- products grouped by type ----------------------------------------------------------------------------------------------------------
def _grouped_args(x, weight, bias, ptr):
    rows, fin = x.shape
    groups, fout = weight.shape[:2]
    return _lib.GroupedLinearArgs(rows, x.stride(0) if rows > 1 else fin, fin, fout, groups, _DTYPES[x.dtype], x.data_ptr(), weight.data_ptr(),
                                  None if bias is None else bias.data_ptr(), ptr.data_ptr())


def _grouped_forward(x, weight, bias, ptr):
    a = _grouped_args(x, weight, bias, ptr)
    y = x.new_empty(a.rows, a.out_features)
    _launch(_lib.lib().dgcnn_grouped_linear_fwd, "dgcnn_grouped_linear_fwd", x.device, ctypes.byref(a), y.data_ptr())
    return y


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, ptr):
        ctx.save_for_backward(x, weight, bias, ptr)
        return _grouped_forward(x, weight, bias, ptr)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, ptr = ctx.saved_tensors
        a = _grouped_args(x, weight, bias, ptr)
        if not dy.is_contiguous():
            dy = dy.contiguous()
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dx = x.new_empty(a.rows, a.in_features) if need_x else None
        dw = torch.empty_like(weight) if need_w or need_b else None
        db = torch.empty_like(bias) if need_b else None
        ws = None
        if dw is not None:
            ws = torch.empty(_bytes("dgcnn_grouped_linear_workspace_bytes", a.rows, a.in_features, a.out_features, a.groups, a.dtype), dtype=torch.uint8,
                             device=x.device)
        _launch(_lib.lib().dgcnn_grouped_linear_bwd, "dgcnn_grouped_linear_bwd", x.device, ctypes.byref(a), dy.data_ptr(), None if dx is None else dx.data_ptr(),
                None if dw is None else dw.data_ptr(), None if db is None else db.data_ptr(), None if ws is None else ws.data_ptr())
        return dx, dw if need_w else None, db, None


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, ptr: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y[i] = weight[e] @ x[i] + bias[e]`` for the rows ``ptr[e] <= i < ptr[e + 1]`` of every group ``e``: ``x`` [N, in] sorted by group, ``weight``
    [groups, out, in] (as ``nn.Linear``'s), ``bias`` [groups, out], ``ptr`` [groups + 1] (ascending, on the device; never read by the host).

    Groups may be empty; rows outside every group give 0 and get gradient 0.  Everything of one type; sums in fp32, results rounded once.  The rows
    of ``x`` may be strided.  Differentiable once in ``x``, ``weight`` and ``bias``."""
    if not x.is_cuda:
        _no_gpu()
    if x.dim() != 2 or weight.dim() != 3 or x.shape[1] != weight.shape[2] or min(weight.shape[1:]) < 1:
        _no(f"x must be [N, in] and weight [groups, out, in], got {tuple(x.shape)} and {tuple(weight.shape)}")
    if x.dtype not in _DTYPES:
        _no_type(x, "x")
    if weight.dtype != x.dtype or weight.get_device() != x.get_device():
        _no(f"weight must be {x.dtype} on {x.device}, got {weight.dtype} on {weight.device}")
    if bias is not None and (bias.shape != weight.shape[:2] or bias.dtype != x.dtype or bias.get_device() != x.get_device()):
        _no(f"bias must be {tuple(weight.shape[:2])} {x.dtype} on {x.device}, got {tuple(bias.shape)} {bias.dtype} on {bias.device}")
    ptr = _check_ptr(ptr, x)
    if ptr.numel() != weight.shape[0] + 1:
        _no(f"ptr must be [{weight.shape[0] + 1}] for {weight.shape[0]} groups, got [{ptr.numel()}]")
    if x.stride(1) != 1 or (x.shape[0] > 1 and not x.shape[1] <= x.stride(0) <= 1 << 21):      # (rows may be strided; anything else is copied)
        x = x.contiguous()
    weight = weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if not _wants_grad(x, weight, bias):
        return _grouped_forward(x, weight, bias, ptr)
    return _GroupedLinear.apply(x, weight, bias, ptr)


class GroupedLinear(nn.Module):
    """:func:`grouped_linear` with its parameters, each group's initialised as ``nn.Linear``'s."""

    def __init__(self, num_groups: int, in_features: int, out_features: int, bias: bool = True, device=None, dtype=None):
        super().__init__()
        if min(num_groups, in_features, out_features) < 1:
            raise ValueError(f"num_groups, in_features and out_features must be positive, got {num_groups}, {in_features}, {out_features}")
        self.num_groups, self.in_features, self.out_features = num_groups, in_features, out_features
        bound = in_features ** -0.5
        self.weight = nn.Parameter(torch.empty(num_groups, out_features, in_features, device=device, dtype=dtype).uniform_(-bound, bound))
        self.bias = nn.Parameter(torch.empty(num_groups, out_features, device=device, dtype=dtype).uniform_(-bound, bound)) if bias else None

    def forward(self, x: torch.Tensor, ptr: torch.Tensor) -> torch.Tensor:
        return grouped_linear(x, self.weight, ptr, self.bias)

    def extra_repr(self) -> str:
        return f"{self.num_groups}, {self.in_features}, {self.out_features}, bias={self.bias is not None}"


# ---- group norm ----------------------------------------------------------------------------------------------------------------------
def _wide(t, channels: int):
    """contiguous, and aligned where a group's channels only fit a workgroup as vectors"""
    t = t.contiguous()
    return t.clone() if channels > 1024 and t.data_ptr() & 15 else t


def _norm_args(head, x, weight, bias, ptr, stats):
    at = stats.data_ptr()
    return _lib.GroupNormArgs(*head, x.data_ptr(), None if weight is None else weight.data_ptr(), None if bias is None else bias.data_ptr(),
                              None if ptr is None else ptr.data_ptr(), at, at + 2 * stats.numel())


def _norm_forward(x, weight, bias, ptr, groups, eps, act):
    C = x.shape[-1]
    segments = x.shape[0] if ptr is None else ptr.numel() - 1
    rows = x.numel() // C
    some = weight if weight is not None else bias
    dtype = _DTYPES[x.dtype]
    y = torch.empty_like(x) if segments else torch.zeros_like(x)
    stats = torch.empty(2, segments, groups, dtype=torch.float32, device=x.device)
    ws = torch.empty(_bytes("dgcnn_group_norm_workspace_bytes", rows, C, groups, segments, ptr is None, dtype, 0), dtype=torch.uint8, device=x.device)
    head = (rows, C, groups, segments, dtype, 0 if some is None else _DTYPES[some.dtype], act, eps, 0)
    _launch(_lib.lib().dgcnn_group_norm_fwd, "dgcnn_group_norm_fwd", x.device, ctypes.byref(_norm_args(head, x, weight, bias, ptr, stats)), y.data_ptr(),
            ws.data_ptr())
    return y, stats, head


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, ptr, groups, eps, act):
        y, stats, ctx.head = _norm_forward(x, weight, bias, ptr, groups, eps, act)
        ctx.save_for_backward(x, weight, bias, ptr, stats)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, ptr, stats = ctx.saved_tensors
        rows, C, groups, segments, dtype = ctx.head[:5]
        dy = _wide(dy, C // groups)
        dx = torch.empty_like(x) if segments else torch.zeros_like(x)
        dw = torch.empty_like(weight) if ctx.needs_input_grad[1] else None
        db = torch.empty_like(bias) if ctx.needs_input_grad[2] else None
        ws = torch.empty(_bytes("dgcnn_group_norm_workspace_bytes", rows, C, groups, segments, ptr is None, dtype, 1), dtype=torch.uint8, device=x.device)
        _launch(_lib.lib().dgcnn_group_norm_bwd, "dgcnn_group_norm_bwd", x.device, ctypes.byref(_norm_args(ctx.head, x, weight, bias, ptr, stats)),
                dy.data_ptr(), dx.data_ptr(), None if dw is None else dw.data_ptr(), None if db is None else db.data_ptr(), ws.data_ptr())
        return dx, dw, db, None, None, None, None


def group_norm(x: torch.Tensor, num_groups: int, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               ptr: Optional[torch.Tensor] = None, eps: float = 1e-5, act: str = "none") -> torch.Tensor:
    """``act(group_norm(x) * weight + bias)`` with the channels last: the mean and the (biased) variance are taken over a sample's rows and a
    group's ``C / num_groups`` consecutive channels.

    ``ptr`` None: ``x`` is ``[B, ..., C]`` and a sample is everything behind the first dimension.  Otherwise ``x`` is ``[N, C]`` and sample ``s`` is rows
    ``ptr[s] .. ptr[s + 1] - 1`` (ascending, on the device; never read by the host); samples may be empty, rows outside every sample give 0 and
    get gradient 0.  A group has at most 1024 channels (2048 if even).  ``act``: "none", "relu", "silu", "gelu" (with erf) or "tanh".  ``weight`` and ``bias`` may be of another type than ``x``;
    ``y`` is of ``x``'s.  Differentiable once in ``x``, ``weight`` and ``bias``."""
    if act not in ACTS:
        _no(f"act must be one of {sorted(ACTS)}, got {act!r}")
    if not x.is_cuda:
        _no_gpu()
    if x.dim() < 2:
        _no(f"x must be [B, ..., C] or [N, C], got {tuple(x.shape)}")
    if x.dtype not in _DTYPES:
        _no_type(x, "x")
    C = x.shape[-1]
    if C < 1 or num_groups < 1 or C % num_groups != 0:
        _no(f"num_groups {num_groups} does not divide {C} channels")
    if not eps >= 0.0:
        _no(f"eps must not be negative, got {eps}")
    for t in (weight, bias):
        if t is not None:
            if t.dtype not in _DTYPES:
                _no_type(t, "weight and bias")
            if t.dim() != 1 or t.shape[0] != C or t.get_device() != x.get_device():
                _no(f"weight and bias must be [{C}] on {x.device}, got {tuple(t.shape)} on {t.device}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        _no("weight and bias must be of one type")
    if ptr is not None:
        if x.dim() != 2:
            _no(f"with ptr, x must be [N, C], got {tuple(x.shape)}")
        ptr = _check_ptr(ptr, x)
    x = _wide(x, C // num_groups)
    weight, bias = (None if t is None else t.contiguous() for t in (weight, bias))
    if not _wants_grad(x, weight, bias):
        return _norm_forward(x, weight, bias, ptr, num_groups, eps, ACTS[act])[0]
    return _GroupNorm.apply(x, weight, bias, ptr, num_groups, eps, ACTS[act])


class GroupNorm(nn.Module):
    """:func:`group_norm` with its affine parameters (``weight`` 1, ``bias`` 0)."""

    def __init__(self, num_groups: int, num_channels: int, eps: float = 1e-5, affine: bool = True, act: str = "none", device=None, dtype=None):
        super().__init__()
        if num_groups < 1 or num_channels % num_groups:
            raise ValueError(f"num_groups {num_groups} does not divide num_channels {num_channels}")
        if act not in ACTS:
            raise ValueError(f"act must be one of {sorted(ACTS)}, got {act!r}")
        self.num_groups, self.num_channels, self.eps, self.act = num_groups, num_channels, eps, act
        self.weight = nn.Parameter(torch.ones(num_channels, device=device, dtype=dtype)) if affine else None
        self.bias = nn.Parameter(torch.zeros(num_channels, device=device, dtype=dtype)) if affine else None

    def forward(self, x: torch.Tensor, ptr: Optional[torch.Tensor] = None) -> torch.Tensor:
        return group_norm(x, self.num_groups, self.weight, self.bias, ptr=ptr, eps=self.eps, act=self.act)

    def extra_repr(self) -> str:
        return f"{self.num_groups}, {self.num_channels}, eps={self.eps}, affine={self.weight is not None}, act={self.act!r}"
