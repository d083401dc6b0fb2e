"""``Adam`` with the call signature of ``torch.optim.Adam`` that updates a :class:`dgcnn_amd.Model` with ONE kernel.

The reference builds its optimizer as ``Adam(model.parameters())`` (/root/reference/train.py:11,99).  With this
build's ``Model`` all 16 parameters are views of one flat buffer and ``loss.backward()`` leaves their ``.grad`` as views
of one flat gradient buffer in the same layout, so ``optimizer.step()`` can be a single ``dgcnn_adam_step`` launch over
the flat buffers instead of torch's multi-tensor path (~10 launches and ~190 us of host time per step for 16 small
tensors).  Changing the import is the only edit to the reference loop::

    from dgcnn_amd.optim import Adam          # instead of: from torch.optim import Adam

Semantics are those of ``torch.optim.Adam`` defaults (no weight decay, no amsgrad; `step`, `exp_avg`, `exp_avg_sq`
per parameter in ``state_dict()``).  Whenever the flat layout is NOT recognised (other modules' parameters, gradients
that are not views of one buffer, a parameter without gradient, ...) the step falls back to torch's own implementation
for that call -- same numbers, just slower.  GPU tensors only take the fused route.

:class:`AdamW` (decoupled weight decay) updates ANY list of GPU tensors with one launch for each 48 of them, through
:func:`adamw_step`: fp32, bf16 and fp16 parameters, fp32 copies of 16-bit ones, moments in 32 or in 8 bits, captured steps.
"""
from __future__ import annotations

import contextlib
import ctypes
import operator
from array import array
from itertools import chain
from typing import Optional, Sequence, Union

import torch
from torch.optim import Optimizer

from . import _lib


def _global_step_hooks() -> bool:
    from torch.optim import optimizer as _o
    return bool(getattr(_o, "_global_optimizer_pre_hooks", None)) or bool(getattr(_o, "_global_optimizer_post_hooks", None))


class Adam(Optimizer):
    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.0,
                 amsgrad: bool = False):
        if weight_decay != 0.0 or amsgrad:
            raise ValueError("dgcnn_amd.optim.Adam implements torch.optim.Adam's defaults (weight_decay=0, amsgrad=False); "
                             "use torch.optim.Adam for the other variants")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps))
        self._flat = {}          # id(group) -> [params_flat, exp_avg, exp_avg_sq, offsets, step tensor, step] once recognised

    # ---- layout recognition ---------------------------------------------------------------------------
    @staticmethod
    def _flat_of(tensors):
        """the 1-D tensor spanning the storage range [min offset, max end) that all `tensors` are views of, plus
        each tensor's offset inside it -- or None when they do not share one storage / overlap / are not dense"""
        t0 = tensors[0]
        st = t0.untyped_storage()
        base, spans = st.data_ptr(), []
        for t in tensors:
            if t.untyped_storage().data_ptr() != base or not t.is_contiguous() or t.dtype != torch.float32 \
                    or t.device != t0.device:
                return None
            spans.append((t.storage_offset(), t.numel()))
        lo = min(o for o, _ in spans)
        hi = max(o + n for o, n in spans)
        order = sorted(spans)
        for (o1, n1), (o2, _) in zip(order, order[1:]):
            if o1 + n1 > o2:
                return None
        if (hi - lo) > 2 * sum(n for _, n in spans) + 64:        # not one packed buffer
            return None
        flat = torch.empty(0, dtype=torch.float32, device=t0.device).set_(st, lo, (hi - lo,))
        return flat, [o - lo for o, _ in spans]

    def _state_views(self, group, pflat, offs):
        m = torch.zeros_like(pflat)
        v = torch.zeros_like(pflat)
        for p, off in zip(group["params"], offs):
            stt = self.state[p]
            prev_m, prev_v = stt.get("exp_avg"), stt.get("exp_avg_sq")
            mv = m[off:off + p.numel()].view(p.shape)
            vv = v[off:off + p.numel()].view(p.shape)
            if prev_m is not None:                     # continue from a loaded / torch-produced state
                mv.copy_(prev_m); vv.copy_(prev_v)
            stt["exp_avg"], stt["exp_avg_sq"] = mv, vv
        # ONE step counter object shared by the group's parameters (torch keeps one per parameter; a state_dict saved
        # from here holds 16 equal values and loads back either way)
        prev = self.state[group["params"][0]].get("step")
        shared = torch.tensor(float(prev) if prev is not None else 0.0, dtype=torch.float32)
        for p in group["params"]:
            self.state[p]["step"] = shared
        return m, v, shared

    def load_state_dict(self, state_dict) -> None:
        """As ``Optimizer.load_state_dict``; the cached flat moment buffers are dropped so that the next ``step()``
        rebuilds them FROM the loaded ``exp_avg`` / ``exp_avg_sq`` / ``step`` (a resumed run must not continue from
        the moments it had before the load)."""
        super().load_state_dict(state_dict)
        self._flat.clear()

    def zero_grad(self, set_to_none: bool = True) -> None:
        """``Optimizer.zero_grad``; the default (``set_to_none=True``) without torch's profiler range and per-device grouping"""
        if not set_to_none:
            return super().zero_grad(set_to_none=False)
        for group in self.param_groups:
            for p in group["params"]:
                p.grad = None

    # ---- step -----------------------------------------------------------------------------------------
    def step(self, closure=None):
        # (torch wraps every optimizer's ``step`` in a profiler range + hook dispatch, ~25 us of host time per call: this
        #  method is marked ``hooked`` so that the wrapper is not installed, and takes the wrapped route itself whenever a
        #  step hook is registered, on the optimizer or globally)
        if self._optimizer_step_pre_hooks or self._optimizer_step_post_hooks or _global_step_hooks():
            return self._hooked_step(closure)
        return self._step_impl(closure)

    step.hooked = True

    def _hooked_step(self, closure=None):
        fn = self.__dict__.get("_wrapped_impl")
        if fn is None:
            fn = self.__dict__["_wrapped_impl"] = Optimizer.profile_hook_step(Adam._step_impl)
        return fn(self, closure)

    def _step_impl(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            params = group["params"]
            if not self._fused_step(group, params):
                with torch.no_grad():
                    self._torch_step(group, params)
        return loss

    def _fused_step(self, group, params) -> bool:
        if not params:
            return False
        key = id(group)
        ent = self._flat.get(key)
        p0 = params[0]
        if ent is None or ent[0].data_ptr() != p0.data_ptr() - 4 * ent[3][0] or ent[6] != len(params):
            if not p0.is_cuda or any(p.grad is None for p in params):
                return False
            rec = self._flat_of(params)
            if rec is None:
                return False
            pflat, offs = rec
            with torch.no_grad():
                m, v, shared = self._state_views(group, pflat, offs)
            ent = self._flat[key] = [pflat, m, v, offs, shared, int(shared.item()), len(params)]
        pflat, m, v, offs, shared, nstep, _ = ent
        if self.state[p0]["step"] is not shared:       # a state_dict was loaded: adopt its counter
            shared.fill_(float(self.state[p0]["step"]))
            nstep = ent[5] = int(shared.item())
            for p in params:
                self.state[p]["step"] = shared
        # parameters AND gradients must mirror the flat layout: parameter i at pflat + offs[i] (a parameter re-pointed by hand
        # since the layout was recognised fails here), its gradient at the same offset of ONE gradient buffer, dense fp32
        g0 = p0.grad
        if g0 is None:
            return False
        pbase = pflat.data_ptr()
        gbase = g0.data_ptr() - 4 * offs[0]
        f32 = torch.float32
        for p, off in zip(params, offs):
            g = p.grad
            if g is None or g.data_ptr() != gbase + 4 * off or p.data_ptr() != pbase + 4 * off or g.dtype is not f32 \
                    or not g.is_contiguous():
                return False
        # ... and that buffer is one allocation spanning the whole layout (the alignment gaps included)
        n = pflat.numel()
        gst = g0.untyped_storage()
        lo = gbase - gst.data_ptr()
        if lo < 0 or lo + 4 * n > gst.nbytes() or g0.device != pflat.device:
            return False
        step = nstep + 1
        b1, b2 = group["betas"]
        stream = torch.cuda.current_stream(pflat.device).cuda_stream
        # the gaps between segments hold zeros in both buffers (zero gradient -> zero update), so one launch over the
        # whole span is exact
        _lib.check(_lib.lib().dgcnn_adam_step(pbase, gbase, m.data_ptr(), v.data_ptr(), n, step,
                                              float(group["lr"]), float(b1), float(b2), float(group["eps"]), 0, stream),
                   "dgcnn_adam_step")
        shared += 1
        ent[5] = step
        return True

    def _torch_step(self, group, params) -> None:
        """torch's own multi-tensor Adam on this group (layout not recognised)"""
        from torch.optim.adam import adam as _adam
        # a group that HAS taken the flat route shares one step counter between its parameters: torch's multi-tensor Adam would
        # increment that one tensor once per parameter.  Back to one counter per parameter (the moments stay views of the flat
        # buffers, which is fine), and the flat entry is dropped: the next step whose layout checks out rebuilds it from the state.
        ent = self._flat.pop(id(group), None)
        if ent is not None:
            for p in params:
                self.state[p]["step"] = ent[4].clone()
        with_grad = [p for p in params if p.grad is not None]
        if not with_grad:
            return
        grads, ms, vs, steps = [], [], [], []
        for p in with_grad:
            stt = self.state[p]
            if "exp_avg" not in stt:
                stt["step"] = torch.tensor(0.0, dtype=torch.float32)
                stt["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                stt["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
            grads.append(p.grad); ms.append(stt["exp_avg"]); vs.append(stt["exp_avg_sq"]); steps.append(stt["step"])
        b1, b2 = group["betas"]
        _adam(with_grad, grads, ms, vs, [], steps, amsgrad=False, beta1=b1, beta2=b2, lr=group["lr"], weight_decay=0.0,
              eps=group["eps"], maximize=False, foreach=None, capturable=False, differentiable=False, fused=None,
              grad_scale=None, found_inf=None, has_complex=False)


# ---- AdamW over many tensors -------------------------------------------------------------------------------------------------------------
STATE_BLOCK = 256           # elements of a tensor that share one scale of an 8-bit moment
_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _refuse(cond: bool, msg: str) -> None:
    if cond:
        raise _lib.DgcnnError(msg)


def _capturing() -> bool:
    return torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()


_numel, _is_contiguous, _get_device, _data_ptr = (getattr(torch.Tensor, k) for k in ("numel", "is_contiguous", "get_device", "data_ptr"))
_get_dtype = operator.attrgetter("dtype")


def _layout(t):
    """how a tensor's elements lie in memory: sizes and strides of the dimensions that have more than one"""
    return [(n, s) for n, s in zip(t.shape, t.stride()) if n != 1]


def _dense(t) -> bool:
    """every place from the first element to the last one holds exactly one, in whatever order"""
    if t.is_contiguous():
        return True
    want = 1
    for n, s in sorted(_layout(t), key=operator.itemgetter(1)):
        if s != want:
            return False
        want *= n
    return True


def _check_list(name, ts, like, numels, device, dtypes) -> torch.dtype:
    """Every tensor of one of `dtypes`, with `numels` elements, laid out as those of `like` (True: contiguous; None: no matter); the type."""
    # (a few C loops over the whole list; the tensors are looked at one by one only to say which it is)
    kinds = set(map(_get_dtype, ts))
    if len(ts) == len(numels) and len(kinds) == 1 and kinds <= dtypes and set(map(_get_device, ts)) == device and list(map(_numel, ts)) == numels and \
            (like is None or (all(map(_is_contiguous, ts)) if like is True else all(_layout(t) == _layout(p) for t, p in zip(ts, like)))):
        return kinds.pop()
    raise _lib.DgcnnError(f"{name} must be {len(numels)} tensors of one type ({', '.join(sorted(map(str, dtypes)))}) on one device, "
                          + (f"contiguous with one element for each {STATE_BLOCK} of the parameter" if name.endswith("scales") else "with their parameters' sizes and strides")
                          + f"; got {len(ts)}: " + ", ".join(f"{t.dtype} {tuple(t.shape)} {t.stride()} on {t.device}" for t in list(ts)[:4]))


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avgs: Sequence[torch.Tensor], exp_avg_sqs: Sequence[torch.Tensor], *,
               step: Union[int, torch.Tensor], lr: Union[float, torch.Tensor] = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
               masters: Optional[Sequence[torch.Tensor]] = None, exp_avg_scales: Optional[Sequence[torch.Tensor]] = None,
               exp_avg_sq_scales: Optional[Sequence[torch.Tensor]] = None, seed: int = 0,
               indices: Optional[Sequence[int]] = None) -> None:
    """One AdamW step over lists of tensors on one device, in place, without synchronising::

        m = b1 m + (1 - b1) g      v = b2 v + (1 - b2) g^2      p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)

    ``params`` are of one type (float32, bfloat16, float16), dense (contiguous in some order of their dimensions, which the other lists follow), and no two of
    them share memory; ``grads`` of the same type, or float32.
    Moments are float32, or -- with both scale lists -- 8 bits: ``exp_avgs`` and ``exp_avg_sqs`` then are ``torch.float8_e4m3fn`` codes of ``m`` and of
    ``sqrt(v)``, each times one float32 scale for 256 consecutive elements (``[ceil(numel / 256)]``).  Codes are rounded stochastically by a hash of
    (``seed``, index, step, element), so that the means do not stall between two codes; equal arguments give equal bits.  A tensor's index is its place in
    the list, or what ``indices`` says: one that keeps it gets the same bits in any list, and tensors of calls with one seed need different ones.
    ``masters``: float32 copies of 16-bit parameters, which are what is updated; the parameters get the rounded values.

    ``step`` is this step's number, from 1 on.  For a step captured into a graph, ``step`` is an int64 device tensor of one element that holds the steps done
    so far (each replay counts it up), and ``lr`` may be a float32 device tensor of one element."""
    if len(params) == 0:
        return
    p0 = params[0]
    dev = p0.device
    if not p0.is_cuda:
        _refuse(True, "dgcnn_amd.optim.adamw_step runs only on an AMD GPU through libdgcnn_hip.so; got a CPU tensor")
    numels, device = list(map(_numel, params)), {p0.get_device()}
    kind = _check_list("params", params, None, numels, device, _DTYPES.keys())
    like = all(map(_is_contiguous, params)) or params
    if like is params and not all(map(_dense, params)):
        _refuse(True, "parameters must be dense tensors: contiguous in some order of their dimensions")
    bits = 32 if exp_avg_scales is None else 8
    if (exp_avg_scales is None) != (exp_avg_sq_scales is None):
        _refuse(True, "8-bit moments need both exp_avg_scales and exp_avg_sq_scales")
    gkind = _check_list("grads", grads, like, numels, device, {kind, torch.float32})
    state = {torch.float32} if bits == 32 else {torch.float8_e4m3fn}
    _check_list("exp_avgs", exp_avgs, like, numels, device, state)
    _check_list("exp_avg_sqs", exp_avg_sqs, like, numels, device, state)
    if bits == 8:
        blocks = [-(-n // STATE_BLOCK) for n in numels]
        _check_list("exp_avg_scales", exp_avg_scales, True, blocks, device, {torch.float32})
        _check_list("exp_avg_sq_scales", exp_avg_sq_scales, True, blocks, device, {torch.float32})
    if masters is not None:
        if kind == torch.float32:
            _refuse(True, "masters are for bfloat16 and float16 parameters")
        _check_list("masters", masters, like, numels, device, {torch.float32})
    if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0 and eps >= 0.0):
        _refuse(True, f"betas must lie in [0, 1) and eps must not be negative, got {betas}, {eps}")

    a = _lib.AdamwArgs()
    keep, counter = None, ()
    if isinstance(step, torch.Tensor):
        counter = (step,)
        _refuse(step.dtype != torch.int64 or step.numel() != 1 or step.device != dev, f"step must be an int or an int64 tensor of one element on {dev}")
        keep = torch.empty(16, dtype=torch.float32, device=dev)
        a.step_dev, a.scalars_dev = step.data_ptr(), keep.data_ptr()
        if isinstance(lr, torch.Tensor):
            _refuse(lr.dtype != torch.float32 or lr.numel() != 1 or lr.device != dev, f"lr must be a float or a float32 tensor of one element on {dev}")
            a.lr_dev, lr = lr.data_ptr(), 0.0
    else:
        if step < 1:
            _refuse(True, f"step counts from 1, got {step}")
        if isinstance(lr, torch.Tensor):
            _refuse(True, "lr may be a tensor only where step is one")
        if _capturing():
            _refuse(True, "a captured step needs its counter on the device: step as an int64 tensor (AdamW: capturable=True)")
        a.step = step
    a.lr, a.beta1, a.beta2, a.eps, a.weight_decay = lr, betas[0], betas[1], eps, weight_decay
    a.seed = seed & 0xFFFFFFFFFFFFFFFF
    a.param_dtype, a.grad_dtype, a.state_bits, a.count = _DTYPES[kind], _DTYPES[gkind], bits, len(params)
    none = [0] * len(params)
    at = lambda ts: none if ts is None else map(_data_ptr, ts)      # noqa: E731
    where = list(map(_data_ptr, params))
    if len(set(where)) < len(where) and len({w for w, n in zip(where, numels) if n}) < sum(1 for n in numels if n):
        _refuse(True, "a parameter is in the list twice")
    if indices is not None:
        try:
            places = array("q", indices)
        except (TypeError, OverflowError):
            places = ()
        if len(places) != len(params) or min(places) < 0:
            _refuse(True, f"indices must be {len(params)} integers from 0 on, got {indices!r}")
        a.indices = places.buffer_info()[0]
    table = array("q", chain.from_iterable(zip(where, at(grads), at(exp_avgs), at(exp_avg_sqs), at(exp_avg_scales), at(exp_avg_sq_scales), at(masters), numels)))
    a.tensors = table.buffer_info()[0]
    # (the launch goes to the tensors' device, which has to be the current one)
    with contextlib.nullcontext() if dev.index is None or dev.index == torch.cuda.current_device() else torch.cuda.device(dev):
        rc = _lib.lib().dgcnn_adamw_step(ctypes.byref(a), torch._C._cuda_getCurrentRawStream(dev.index))
    _lib.check(rc, "dgcnn_adamw_step")
    # (the library writes through addresses: what a graph saved of these has to count as changed)
    torch.autograd.graph.increment_version(chain(params, exp_avgs, exp_avg_sqs, masters or (), exp_avg_scales or (), exp_avg_sq_scales or (), counter))


class AdamW(Optimizer):
    """``torch.optim.AdamW`` (no amsgrad) over GPU parameters of any dense layout: one launch for each 48 tensors of a type.

    ``state_bits`` 32: float32 moments, ``state_dict()`` as torch's (and torch's loads).  8: moments as :func:`adamw_step` describes them, a quarter of
    the bytes; the state then holds ``exp_avg``, ``exp_avg_sq`` (codes of the mean and of the root of the mean square) and their ``_scale`` tensors.
    ``master_weights``: bfloat16 / float16 parameters get a float32 copy (``master`` in the state) that carries the updates too small for their type.
    ``capturable``: the step counter lives on the device and ``step()`` may be captured into a graph; ``lr`` may then be a float32 device tensor of one
    element; parameters that were captured together share their counter, so eager steps beside the graph have to be for all of them.  A parameter without
    a gradient is left alone; ``seed`` picks the random rounding of 8-bit moments, in which a parameter's index is its place among all the optimizer's."""

    def __init__(self, params, lr: Union[float, torch.Tensor] = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, amsgrad: bool = False, *,
                 state_bits: int = 32, master_weights: bool = False, capturable: bool = False, seed: int = 0):
        if amsgrad:
            raise ValueError("dgcnn_amd.optim.AdamW has no amsgrad variant; use torch.optim.AdamW")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        if not isinstance(lr, torch.Tensor) and not lr >= 0.0:
            raise ValueError(f"lr must not be negative, got {lr}")
        if isinstance(lr, torch.Tensor) and not capturable:
            raise ValueError("lr may be a tensor only with capturable=True")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0) or not eps >= 0.0 or not weight_decay >= 0.0:
            raise ValueError(f"betas must lie in [0, 1), eps and weight_decay must not be negative: got {betas}, {eps}, {weight_decay}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits, master_weights=master_weights,
                                      capturable=capturable, seed=seed))

    def _state_of(self, p, group, fresh):
        st = self.state[p]
        if not st:
            _refuse(_capturing(), "run a step() before capturing one: the state would be set up anew by every replay")
            # (tensors that start together share their counter: they can go into one call)
            st["step"] = fresh.setdefault(p.device, torch.zeros(1, dtype=torch.int64, device=p.device)) if group["capturable"] else 0
            if group["state_bits"] == 32:
                st["exp_avg"], st["exp_avg_sq"] = (torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format) for _ in range(2))
            else:
                for k in ("exp_avg", "exp_avg_sq"):
                    st[k] = torch.zeros_like(p, dtype=torch.uint8, memory_format=torch.preserve_format).view(torch.float8_e4m3fn)
                    st[k + "_scale"] = torch.zeros(-(-p.numel() // STATE_BLOCK), dtype=torch.float32, device=p.device)
        if group["master_weights"] and p.dtype != torch.float32 and "master" not in st:
            st["master"] = p.detach().to(torch.float32, copy=True)
        t = st["step"]
        if group["capturable"] != isinstance(t, torch.Tensor) or (group["capturable"] and (t.dtype != torch.int64 or t.device != p.device)):
            _refuse(_capturing(), "run a step() after loading a state and before capturing one: its counters are not on the device yet")
            n = int(t)              # (a state of another kind was loaded: torch's counters are float32 tensors)
            st["step"] = fresh.setdefault((p.device, n), torch.full((1,), n, dtype=torch.int64, device=p.device)) if group["capturable"] else n
        return st

    def load_state_dict(self, state_dict) -> None:
        """As ``Optimizer.load_state_dict``, but every tensor of the state keeps its own type (torch's casts them to the parameter's, which codes, scales
        and the float32 moments of 16-bit parameters do not survive)."""
        for g in state_dict["param_groups"]:
            if g.get("amsgrad") or g.get("maximize"):
                raise ValueError("dgcnn_amd.optim.AdamW has no amsgrad or maximize variant: this state is another optimizer's")
        super().load_state_dict(state_dict)
        for g in self.param_groups:              # (torch's groups hold no state_bits, master_weights, seed)
            for k, v in self.defaults.items():
                g.setdefault(k, v)
        saved = list(chain.from_iterable(g["params"] for g in state_dict["param_groups"]))
        mine = list(chain.from_iterable(g["params"] for g in self.param_groups))
        for k, p in zip(saved, mine):
            for name, v in state_dict["state"].get(k, {}).items():
                if isinstance(v, torch.Tensor):
                    if name in ("exp_avg", "exp_avg_sq") and v.is_floating_point() and v.dtype.itemsize > 1:
                        v = v.float()            # (torch holds the moments of 16-bit parameters in 16 bits)
                    if name != "step" and v.shape == p.shape and _layout(v) != _layout(p):
                        if v.dtype.itemsize == 1:
                            raise ValueError("the 8-bit state of a parameter of another memory layout: its blocks are other elements")
                        v = torch.empty_like(p, dtype=v.dtype).copy_(v)
                    # (counters come back as host numbers: step() makes one device counter for all equal ones)
                    self.state[p][name] = int(v) if name == "step" else v.detach().to(p.device, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        behind = 0                                # parameters in front of the group's
        for group in self.param_groups:
            calls, fresh, first = {}, {}, behind
            behind += len(group["params"])
            for index, p in enumerate(group["params"], first):
                g = p.grad
                if g is None:
                    continue
                if g.is_sparse:
                    _refuse(True, "dgcnn_amd.optim.AdamW takes dense gradients")
                if g.stride() != p.stride() and _layout(g) != _layout(p) and _dense(p):
                    g = torch.empty_like(p, dtype=g.dtype).copy_(g)
                st = self._state_of(p, group, fresh)
                t = st["step"]
                calls.setdefault((p.device, p.dtype, g.dtype, "master" in st, t.data_ptr() if group["capturable"] else t, "exp_avg_scale" in st),
                                 []).append((p, g, st, index))
            if group["capturable"]:
                idle = {}                         # parameters that sit this step out keep their count
                for p in group["params"]:
                    t = self.state[p].get("step") if p.grad is None and p in self.state else None
                    if isinstance(t, torch.Tensor):
                        idle.setdefault(t.data_ptr(), []).append(self.state[p])
                for items in calls.values():
                    t = items[0][2]["step"]
                    if t.data_ptr() in idle:
                        _refuse(_capturing(), "run a step() with gradients for the same parameters before capturing one")
                        t = t.clone()
                        for st in idle.pop(items[0][2]["step"].data_ptr()):
                            st["step"] = t
                counted = set()
                for items in calls.values():      # a call counts its counter up: no two calls may share one
                    t = items[0][2]["step"]
                    if t.data_ptr() in counted:
                        _refuse(_capturing(), "run a step() with these gradients' types before capturing one")
                        t = t.clone()
                        for _, _, st, _ in items:
                            st["step"] = t
                    counted.add(t.data_ptr())
            for key, items in calls.items():
                ps, gs, sts, indices = zip(*items)
                t = sts[0]["step"] if group["capturable"] else sts[0]["step"] + 1
                more = {k + "s": [st[k] for st in sts] for k in ("exp_avg_scale", "exp_avg_sq_scale") if k in sts[0]}
                if key[3]:
                    more["masters"] = [st["master"] for st in sts]
                if key[5]:
                    more["indices"] = indices
                adamw_step(ps, gs, [st["exp_avg"] for st in sts], [st["exp_avg_sq"] for st in sts], step=t, lr=group["lr"], betas=group["betas"],
                           eps=group["eps"], weight_decay=group["weight_decay"], seed=group["seed"], **more)
                if not group["capturable"]:
                    for st in sts:
                        st["step"] = t
        return loss
