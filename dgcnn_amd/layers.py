"""Layer operators for networks around the graph convolutions: differentiable functions and modules over the node rows of a batch.

* :func:`grouped_linear` / :class:`GroupedLinear` -- a linear map for each type (relation, expert) of the rows, sorted by type.
* :func:`group_norm` / :class:`GroupNorm` -- group norm with an activation, channels last, over every graph of a batch (``ptr``) or over dense
  samples ``[B, ..., C]``.

Rows are the nodes of a :class:`dgcnn_amd.Batch` (or edges, messages, pixels); ``ptr`` says where each graph's rows begin, as
:func:`graph_ptr` returns it.  fp32, bf16 and fp16; sums and statistics in fp32.  Everything runs on the current stream of the tensors' device through
``libdgcnn_hip.so`` without synchronising, forward and backward may be captured into a graph, and equal inputs give equal bits.  As in the rest of the
package there is no CPU fallback: CPU tensors raise :class:`dgcnn_amd._lib.DgcnnError`.
"""
from __future__ import annotations

import contextlib
import ctypes
from typing import Optional

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "tanh": 4}


def _refuse(cond: bool, msg: str) -> None:
    if cond:
        raise _lib.DgcnnError(msg)


def _dtype(t: torch.Tensor, what: str) -> int:
    d = _DTYPES.get(t.dtype)
    _refuse(d is None, f"{what} must be float32, bfloat16 or float16, got {t.dtype}")
    return d


def _on(device: torch.device):
    """The device a launch goes to has to be the current one."""
    if device.index is None or device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _check_ptr(ptr: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    _refuse(ptr.dim() != 1 or ptr.numel() < 1, f"ptr must be [segments + 1], got {tuple(ptr.shape)}")
    _refuse(ptr.dtype not in (torch.int64, torch.int32), f"ptr must be int64 or int32, got {ptr.dtype}")
    _refuse(ptr.device != x.device, f"ptr on {ptr.device}, x on {x.device}")
    return ptr.to(torch.int64).contiguous()


def graph_ptr(data) -> torch.Tensor:
    """``ptr`` [B + 1] (int64, on the batch's device) of a batch: graph ``g`` is rows ``ptr[g] .. ptr[g + 1] - 1``.  No synchronisation where the batch
    knows its ``num_graphs``."""
    batch = data.batch
    n = getattr(data, "num_graphs", None)
    if n is None:
        n = int(batch[-1].item()) + 1 if batch.numel() else 0
    return torch.searchsorted(batch.contiguous(), torch.arange(n + 1, device=batch.device, dtype=batch.dtype))


# ---- products grouped by type ----------------------------------------------------------------------------------------------------------
class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def _args(x, weight, bias, ptr):
        a = _lib.GroupedLinearArgs()
        a.rows, a.in_features = x.shape
        a.groups, a.out_features = weight.shape[:2]
        a.ldx, a.dtype = max(x.stride(0), a.in_features), _DTYPES[x.dtype]
        a.x, a.weight, a.ptr = x.data_ptr(), weight.data_ptr(), ptr.data_ptr()
        a.bias = None if bias is None else bias.data_ptr()
        return a

    @staticmethod
    def forward(ctx, x, weight, bias, ptr):
        if x.stride(1) != 1 or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
            x = x.contiguous()
        weight = weight.contiguous()
        bias = None if bias is None else bias.contiguous()
        a = _GroupedLinear._args(x, weight, bias, ptr)
        y = torch.empty(a.rows, a.out_features, dtype=x.dtype, device=x.device)
        with _on(x.device):
            _lib.check(_lib.lib().dgcnn_grouped_linear_fwd(ctypes.byref(a), y.data_ptr(), _stream(x.device)), "dgcnn_grouped_linear_fwd")
        ctx.save_for_backward(x, weight, bias, ptr)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, ptr = ctx.saved_tensors
        a = _GroupedLinear._args(x, weight, bias, ptr)
        dy = dy.contiguous()
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dx = torch.empty(a.rows, a.in_features, dtype=x.dtype, device=x.device) if need_x else None
        dw = torch.empty_like(weight) if need_w or need_b else None
        db = torch.empty_like(bias) if need_b else None
        L, ws = _lib.lib(), None
        if dw is not None:
            ws = torch.empty(_lib.checked_bytes(L.dgcnn_grouped_linear_workspace_bytes(a.rows, a.in_features, a.out_features, a.groups, a.dtype),
                                                "dgcnn_grouped_linear_workspace_bytes"), dtype=torch.uint8, device=x.device)
        at = lambda t: None if t is None else t.data_ptr()      # noqa: E731
        with _on(x.device):
            _lib.check(L.dgcnn_grouped_linear_bwd(ctypes.byref(a), dy.data_ptr(), at(dx), at(dw), at(db), at(ws), _stream(x.device)), "dgcnn_grouped_linear_bwd")
        return dx, dw if need_w else None, db, None


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, ptr: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y[i] = weight[e] @ x[i] + bias[e]`` for the rows ``ptr[e] <= i < ptr[e + 1]`` of every group ``e``: ``x`` [N, in] sorted by group, ``weight``
    [groups, out, in] (as ``nn.Linear``'s), ``bias`` [groups, out], ``ptr`` [groups + 1] (ascending, on the device; never read by the host).

    Groups may be empty; rows outside every group give 0 and get gradient 0.  Everything of one type; sums in fp32, results rounded once.  The rows
    of ``x`` may be strided.  Differentiable once in ``x``, ``weight`` and ``bias``."""
    _refuse(not x.is_cuda, "dgcnn_amd.layers runs only on an AMD GPU through libdgcnn_hip.so; got a CPU tensor (there is deliberately no CPU fallback)")
    _refuse(x.dim() != 2 or weight.dim() != 3 or x.shape[1] != weight.shape[2] or min(weight.shape[1:]) < 1,
            f"x must be [N, in] and weight [groups, out, in], got {tuple(x.shape)} and {tuple(weight.shape)}")
    _dtype(x, "x")
    _refuse(weight.dtype != x.dtype or weight.device != x.device, f"weight must be {x.dtype} on {x.device}, got {weight.dtype} on {weight.device}")
    if bias is not None:
        _refuse(bias.shape != weight.shape[:2] or bias.dtype != x.dtype or bias.device != x.device,
                f"bias must be {tuple(weight.shape[:2])} {x.dtype} on {x.device}, got {tuple(bias.shape)} {bias.dtype} on {bias.device}")
    ptr = _check_ptr(ptr, x)
    _refuse(ptr.numel() != weight.shape[0] + 1, f"ptr must be [{weight.shape[0] + 1}] for {weight.shape[0]} groups, got [{ptr.numel()}]")
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
class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, ptr, groups, eps, act):
        C = x.shape[-1]
        xc = x.contiguous()
        segments = x.shape[0] if ptr is None else ptr.numel() - 1
        rows = xc.numel() // C
        a = _lib.GroupNormArgs()
        a.rows, a.channels, a.groups, a.segments, a.dtype, a.act, a.eps = rows, C, groups, segments, _DTYPES[x.dtype], act, eps
        wb = [None if t is None else t.contiguous() for t in (weight, bias)]
        some = wb[0] if wb[0] is not None else wb[1]
        a.weight_dtype = 0 if some is None else _DTYPES[some.dtype]
        y = torch.empty_like(xc) if segments else torch.zeros_like(xc)
        stats = torch.empty(2, segments, groups, dtype=torch.float32, device=x.device)
        L = _lib.lib()
        ws = torch.empty(_lib.checked_bytes(L.dgcnn_group_norm_workspace_bytes(rows, C, groups, segments, ptr is None, a.dtype, 0),
                                            "dgcnn_group_norm_workspace_bytes"), dtype=torch.uint8, device=x.device)
        a.x, a.mean, a.rstd = xc.data_ptr(), stats[0].data_ptr(), stats[1].data_ptr()
        a.weight, a.bias = (None if t is None else t.data_ptr() for t in wb)
        a.ptr = None if ptr is None else ptr.data_ptr()
        with _on(x.device):
            _lib.check(L.dgcnn_group_norm_fwd(ctypes.byref(a), y.data_ptr(), ws.data_ptr(), _stream(x.device)), "dgcnn_group_norm_fwd")
        ctx.save_for_backward(xc, *wb, ptr, stats)
        ctx.args = (rows, C, groups, segments, a.dtype, a.weight_dtype, act, eps)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, ptr, stats = ctx.saved_tensors
        a = _lib.GroupNormArgs()
        a.rows, a.channels, a.groups, a.segments, a.dtype, a.weight_dtype, a.act, a.eps = ctx.args
        dyc = dy.contiguous()
        dx = torch.empty_like(x) if a.segments else torch.zeros_like(x)
        dw = torch.empty_like(weight) if ctx.needs_input_grad[1] else None
        db = torch.empty_like(bias) if ctx.needs_input_grad[2] else None
        L = _lib.lib()
        ws = torch.empty(_lib.checked_bytes(L.dgcnn_group_norm_workspace_bytes(a.rows, a.channels, a.groups, a.segments, ptr is None, a.dtype, 1),
                                            "dgcnn_group_norm_workspace_bytes"), dtype=torch.uint8, device=x.device)
        a.x, a.mean, a.rstd = x.data_ptr(), stats[0].data_ptr(), stats[1].data_ptr()
        a.weight, a.bias = (None if t is None else t.data_ptr() for t in (weight, bias))
        a.ptr = None if ptr is None else ptr.data_ptr()
        with _on(x.device):
            _lib.check(L.dgcnn_group_norm_bwd(ctypes.byref(a), dyc.data_ptr(), dx.data_ptr(), None if dw is None else dw.data_ptr(),
                                              None if db is None else db.data_ptr(), ws.data_ptr(), _stream(x.device)), "dgcnn_group_norm_bwd")
        return dx, dw, db, None, None, None, None


def group_norm(x: torch.Tensor, num_groups: int, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               ptr: Optional[torch.Tensor] = None, eps: float = 1e-5, act: str = "none") -> torch.Tensor:
    """``act(group_norm(x) * weight + bias)`` with the channels last: the mean and the (biased) variance are taken over a sample's rows and a
    group's ``C / num_groups`` consecutive channels.

    ``ptr`` None: ``x`` is ``[B, ..., C]`` and a sample is everything behind the first dimension.  Otherwise ``x`` is ``[N, C]`` and sample ``s`` is rows
    ``ptr[s] .. ptr[s + 1] - 1`` (ascending, on the device; never read by the host); samples may be empty, rows outside every sample give 0 and
    get gradient 0.  ``act``: "none", "relu", "silu", "gelu" (with erf) or "tanh".  ``weight`` and ``bias`` may be of another type than ``x``;
    ``y`` is of ``x``'s.  Differentiable once in ``x``, ``weight`` and ``bias``."""
    _refuse(act not in ACTS, f"act must be one of {sorted(ACTS)}, got {act!r}")
    _refuse(not x.is_cuda, "dgcnn_amd.layers runs only on an AMD GPU through libdgcnn_hip.so; got a CPU tensor (there is deliberately no CPU fallback)")
    _refuse(x.dim() < 2, f"x must be [B, ..., C] or [N, C], got {tuple(x.shape)}")
    _dtype(x, "x")
    C = x.shape[-1]
    _refuse(C < 1 or num_groups < 1 or C % num_groups != 0, f"num_groups {num_groups} does not divide {C} channels")
    _refuse(not eps >= 0.0, f"eps must not be negative, got {eps}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            _dtype(t, name)
            _refuse(tuple(t.shape) != (C,) or t.device != x.device, f"{name} must be [{C}] on {x.device}, got {tuple(t.shape)} on {t.device}")
    _refuse(weight is not None and bias is not None and weight.dtype != bias.dtype, "weight and bias must be of one type")
    if ptr is not None:
        _refuse(x.dim() != 2, f"with ptr, x must be [N, C], got {tuple(x.shape)}")
        ptr = _check_ptr(ptr, x)
    return _GroupNorm.apply(x, weight, bias, ptr, int(num_groups), float(eps), ACTS[act])


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
