"""Operators on gradients, between the backward pass and the step.

Each function takes a list of tensors (``[p.grad for p in params if p.grad is
not None]``, the views of a flat gradient buffer, a ZeRO shard's segments) and
works on all of them in a few launches, without a host synchronisation:

* ``grad_norm`` — the norm of all elements of all tensors, and of each tensor;
* ``clip_coef`` — the norm and the coefficient that clipping multiplies by,
  for ``LUMA.step(grad_scale=coef)``; with a loss scale's reciprocal and its
  inf/NaN flag for mixed precision;
* ``scale_grads_``, ``clip_grads_`` — in place;
* ``accumulate_grads_`` — micro-batches into (wider) accumulators, with the
  norm and the coefficient of the result from the same pass.

``clip_grad_coef`` (clip.py) gives the same numbers as PyTorch's own clipping,
rounded to the grads' type where that is; the functions here sum in 64 bits
and return float32 whatever the grads' type.

Tensors are float32, bfloat16 or float16, mixed as they come, dense in memory
(contiguous in some order of their dimensions), all on one CUDA device, of any
size (0 included) and alignment.  Work is queued on the device's current
stream; results are tensors on the device and the same bits on every call with
the same tensors.  A call may be captured in a CUDA graph; replays then work
on the captured tensors' memory.  Where a list is empty, the result is what
nothing adds up to (norm 0, coefficient 1), on the CPU.
"""

from __future__ import annotations

import ctypes
import math
from array import array

import torch

from . import _lib

__all__ = ["grad_norm", "clip_coef", "scale_grads_", "clip_grads_", "accumulate_grads_"]

_PLAIN = {torch.Tensor, torch.nn.Parameter}
_CODE = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_KIND = {1.0: _lib.NORM_1, 2.0: _lib.NORM_2, math.inf: _lib.NORM_MAX}
_SCALARS = (torch.float32, torch.bfloat16, torch.float16)


class _List:
    """A checked list of tensors as the arrays the library takes."""

    __slots__ = ("tensors", "ptrs", "numels", "codes", "device", "sharded")

    def __init__(self, tensors, name: str):
        if isinstance(tensors, torch.Tensor):
            tensors = [tensors]
        ts = list(tensors)
        self.sharded = False
        if not set(map(type, ts)) <= _PLAIN:
            for i, t in enumerate(ts):
                if not isinstance(t, torch.Tensor):
                    raise TypeError(f"{name}[{i}] is {type(t).__name__}, not a tensor")
                if hasattr(t, "_local_tensor"):  # DTensor (FSDP2): this rank's shard
                    ts[i] = t._local_tensor
                    self.sharded = True
        self.tensors = ts
        self.device = None
        if not ts:
            self.ptrs = self.numels = array("q")
            self.codes = b""
            return
        for t in ts:
            if t.layout is not torch.strided:
                raise RuntimeError(f"LUMA does not support sparse gradients ({name})")
            if t.dtype not in _CODE:
                raise ValueError(f"{name} must be float32/bfloat16/float16 tensors "
                                 f"(got {t.dtype})")
            if not t.is_cuda:
                raise RuntimeError(f"LUMA backend 'cuda' requires CUDA tensors "
                                   f"({name} on {t.device})")
            if not t.is_contiguous() and not _dense(t):
                raise ValueError(f"{name} must be dense in memory (got strides {t.stride()} "
                                 f"for shape {tuple(t.shape)})")
        devices = {t.device for t in ts}
        if len(devices) > 1:
            raise ValueError(f"{name} must be on one device (got "
                             f"{', '.join(sorted(map(str, devices)))})")
        self.device = ts[0].device
        self.ptrs = array("Q", [t.data_ptr() for t in ts])
        self.numels = array("q", [t.numel() for t in ts])
        self.codes = bytes([_CODE[t.dtype] for t in ts])


def _dense(t: torch.Tensor) -> bool:
    """Whether t's elements are `numel` consecutive ones, in some order of its
    dimensions (a transposed or channels-last gradient)."""
    if t.numel() <= 1:
        return True
    room = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != room:
            return False
        room *= size
    return True


def _args(lst: _List, device: torch.device) -> _lib.LumaGradArgs:
    a = _lib.LumaGradArgs()
    a.grads = lst.ptrs.buffer_info()[0]
    a.numel = lst.numels.buffer_info()[0]
    a.dtypes = ctypes.cast(ctypes.c_char_p(lst.codes), ctypes.c_void_p)
    a.n = len(lst.tensors)
    a.host_scale = 1.0
    a.device = device.index
    return a


def _call(name: str, a: _lib.LumaGradArgs, device: torch.device) -> None:
    stream = torch.cuda.current_stream(device).cuda_stream
    _lib.check(getattr(_lib.lib(), name)(ctypes.byref(a), ctypes.c_void_p(stream)), name)


def _workspace(a: _lib.LumaGradArgs, device: torch.device) -> torch.Tensor:
    """Partial results of one call: memory of the current stream (of the graph,
    during a capture), so calls that overlap never share it."""
    n = _lib.grad_partials(a.n)
    ws = torch.empty(n, dtype=torch.float64, device=device)
    a.partials = ws.data_ptr()
    a.n_partials = n
    return ws


def _kind(norm_type) -> int:
    kind = _KIND.get(float(norm_type))
    if kind is None:
        raise ValueError(f"norm_type must be 1, 2 or inf (got {norm_type})")
    return kind


def _bound(max_norm) -> float:
    m = float(max_norm)
    if not m >= 0.0:
        raise ValueError(f"max_norm must be 0 or more (got {max_norm})")
    return m


def _factor(x, device: torch.device, name: str) -> tuple[float, torch.Tensor | None]:
    """(host factor, device factor or None) of a number or one-element tensor."""
    if not isinstance(x, torch.Tensor):
        return float(x), None
    if x.numel() != 1 or x.dtype not in _SCALARS:
        raise ValueError(f"{name} must be a number or a one-element float32, bfloat16 or "
                         f"float16 tensor")
    return 1.0, x.detach().reshape(1).to(device=device, dtype=torch.float32, non_blocking=True)


def _flag(x: torch.Tensor | None, device: torch.device, name: str) -> int | None:
    if x is None:
        return None
    if not isinstance(x, torch.Tensor) or x.numel() != 1 or x.dtype != torch.float32 \
            or not x.is_cuda or not x.is_contiguous():
        raise ValueError(f"{name} must be a one-element contiguous float32 CUDA tensor")
    if x.device != device:
        raise ValueError(f"{name} must be on the gradients' device")
    return x.data_ptr()


def _written(tensors) -> None:
    """Tell autograd that the tensors changed, as its own in-place operations do."""
    try:
        torch.autograd.graph.increment_version(tensors)
    except RuntimeError:  # inference tensors keep no version
        torch.autograd.graph.increment_version([t for t in tensors if not t.is_inference()])


def _check_finite(norm: torch.Tensor) -> None:
    if not bool(torch.isfinite(norm)):
        raise RuntimeError("the gradients' norm is not finite, so they cannot be clipped "
                           "(error_if_nonfinite=False clips them all the same)")


def _scalar(device: torch.device) -> torch.Tensor:
    return torch.empty((), dtype=torch.float32, device=device)


def _norm(lst: _List, kind: int, device: torch.device, *, max_norm: float | None = None,
          per_tensor: bool = False, inv_scale=None, found_inf=None, group=None):
    """(norm, coef or None, norms or None) of a list; with `group`, of the lists
    of all its ranks together."""
    a = _args(lst, device)
    a.norm_kind = kind
    ws = _workspace(a, device)  # noqa: F841 - alive until the launches are queued
    norm = _scalar(device)
    coef = norms = None
    if per_tensor:
        norms = torch.empty(len(lst.tensors), dtype=torch.float32, device=device)
        a.norms = norms.data_ptr()
    if group is not None:
        import torch.distributed as dist
        power = torch.empty(1, dtype=torch.float64, device=device)
        a.power = power.data_ptr()
        _call("luma_grad_norm", a, device)
        if kind == _lib.NORM_MAX:
            # a maximum over ranks may drop a NaN, but no infinity
            power.nan_to_num_(nan=math.inf, posinf=math.inf)
            dist.all_reduce(power, op=dist.ReduceOp.MAX, group=group)
        else:
            dist.all_reduce(power, op=dist.ReduceOp.SUM, group=group)
        a.power = a.norms = None
        a.partials, a.n_partials = power.data_ptr(), 1
    a.norm = norm.data_ptr()
    if max_norm is not None:
        coef = _scalar(device)
        a.coef = coef.data_ptr()
        a.max_norm = max_norm
    a.inv_scale, a.found_inf = inv_scale, found_inf
    _call("luma_grad_norm" if group is None else "luma_grad_finish", a, device)
    return norm, coef, norms


def _check_sharded(lst: _List, group) -> None:
    if lst.sharded and group is None:
        raise ValueError("the gradients are sharded (DTensor): pass process_group, over whose "
                         "ranks the norm is taken")


@torch.compiler.disable
@torch.no_grad()
def grad_norm(grads, norm_type: float = 2.0, *, per_tensor: bool = False,
              error_if_nonfinite: bool = False, process_group=None):
    """Norm of all elements of all tensors in `grads`, a float32 scalar on their
    device; `norm_type` is 1, 2 or inf.

    ``per_tensor=True`` returns ``(norm, norms)`` with ``norms[i]`` the norm of
    ``grads[i]`` (0 for an empty one), from the same pass.  With
    ``error_if_nonfinite`` the norm is read back and an inf or NaN raises.
    With `process_group` every rank passes shards of its own (DTensors, ZeRO
    segments) and gets the norm over all ranks' shards; every rank of the group
    has to call, one with an empty list included.  (There a NaN on some rank
    gives an inf norm where `norm_type` is inf.)"""
    kind = _kind(norm_type)
    lst = _List(grads, "grads")
    if per_tensor and (process_group is not None or lst.sharded):
        raise ValueError("per_tensor norms are of whole tensors, not of shards")
    _check_sharded(lst, process_group)
    if lst.device is None and process_group is None:
        zero = torch.tensor(0.0)
        return (zero, torch.zeros(0)) if per_tensor else zero
    device = lst.device or torch.device("cuda", torch.cuda.current_device())
    norm, _, norms = _norm(lst, kind, device, per_tensor=per_tensor, group=process_group)
    if error_if_nonfinite:
        _check_finite(norm)
    return (norm, norms) if per_tensor else norm


@torch.compiler.disable
@torch.no_grad()
def clip_coef(grads, max_norm: float, norm_type: float = 2.0, *,
              inv_scale: torch.Tensor | None = None, found_inf: torch.Tensor | None = None,
              error_if_nonfinite: bool = False,
              process_group=None) -> tuple[torch.Tensor, torch.Tensor]:
    """(norm, coef): the norm of `grads` and ``min(1, max_norm / (norm + 1e-6))``,
    float32 scalars on their device; the grads are not modified.  Pass `coef`
    to ``LUMA.step(grad_scale=coef)`` or ``scale_grads_``.

    `inv_scale`, a one-element float32 CUDA tensor, is the reciprocal of the
    loss scale the grads carry: the norm is then that of the unscaled grads and
    `coef` holds both factors (unscaling and clipping).  `found_inf`, likewise
    one element, is set to 1 if any element of the grads is inf or NaN, and
    left alone otherwise.  `error_if_nonfinite` and `process_group` are as in
    ``grad_norm``."""
    kind, bound = _kind(norm_type), _bound(max_norm)
    lst = _List(grads, "grads")
    _check_sharded(lst, process_group)
    if lst.device is None and process_group is None:
        return torch.tensor(0.0), torch.tensor(1.0)
    device = lst.device or torch.device("cuda", torch.cuda.current_device())
    norm, coef, _ = _norm(lst, kind, device, max_norm=bound, group=process_group,
                          inv_scale=_flag(inv_scale, device, "inv_scale"),
                          found_inf=_flag(found_inf, device, "found_inf"))
    if error_if_nonfinite:
        _check_finite(norm)
    return norm, coef


def _scale(lst: _List, host: float, factor: torch.Tensor | None) -> None:
    a = _args(lst, lst.device)
    a.host_scale = host
    a.scale = None if factor is None else factor.data_ptr()
    _call("luma_grad_scale", a, lst.device)
    _written(lst.tensors)


@torch.compiler.disable
@torch.no_grad()
def scale_grads_(grads, coef) -> None:
    """Multiply every tensor in `grads` by `coef` in place: each element becomes
    ``round_to_its_type(fl32(g) * fl32(coef))``.  `coef` is a number or a
    one-element float32, bfloat16 or float16 tensor; where it is 1 the grads
    are neither read nor written.  The tensors must not share memory."""
    lst = _List(grads, "grads")
    if lst.device is None:
        return
    _scale(lst, *_factor(coef, lst.device, "coef"))


@torch.compiler.disable
@torch.no_grad()
def clip_grads_(grads, max_norm: float, norm_type: float = 2.0, *,
                error_if_nonfinite: bool = False, process_group=None) -> torch.Tensor:
    """Scale `grads` in place so that their norm is at most `max_norm`, and
    return the norm they had: ``norm, coef = clip_coef(...)``, then
    ``scale_grads_(grads, coef)``.  With `error_if_nonfinite` an inf or NaN norm
    raises before anything is written."""
    kind, bound = _kind(norm_type), _bound(max_norm)
    lst = _List(grads, "grads")
    _check_sharded(lst, process_group)
    if lst.device is None and process_group is None:
        return torch.tensor(0.0)
    device = lst.device or torch.device("cuda", torch.cuda.current_device())
    if process_group is None and not error_if_nonfinite:
        a = _args(lst, device)
        a.norm_kind, a.max_norm = kind, bound
        ws = _workspace(a, device)  # noqa: F841
        norm, coef = _scalar(device), _scalar(device)
        a.norm, a.coef = norm.data_ptr(), coef.data_ptr()
        _call("luma_grad_clip", a, device)
        _written(lst.tensors)
        return norm
    norm, coef, _ = _norm(lst, kind, device, max_norm=bound, group=process_group)
    if error_if_nonfinite:
        _check_finite(norm)
    if lst.tensors:
        _scale(lst, 1.0, coef)
    return norm


@torch.compiler.disable
@torch.no_grad()
def accumulate_grads_(acc, grads, scale=1.0, *, overwrite: bool = False,
                      norm_type: float | None = None, max_norm: float | None = None):
    """``acc[i] += scale * grads[i]`` for every i, in one launch: one fused
    multiply-add in float32 per element, rounded to the accumulator's type.
    With `overwrite` it is ``acc[i] = scale * grads[i]`` (the first
    micro-batch), whatever `acc` held.

    `acc` are float32 or bfloat16 tensors, `grads` float32, bfloat16 or float16
    ones of the same shapes and dimension order; `scale` is a number or a
    one-element tensor as in ``scale_grads_``.  ``grads[i]`` may be ``acc[i]``
    itself; other overlaps are refused.

    With `norm_type` (1, 2 or inf) the norm of the accumulators as they are
    afterwards is returned, from the same pass; with `max_norm` it is
    ``(norm, coef)`` as ``clip_coef(acc, max_norm, norm_type or 2)`` gives
    them.  Otherwise nothing is returned."""
    kind = _lib.NORM_NONE
    if norm_type is not None or max_norm is not None:
        kind = _kind(2.0 if norm_type is None else norm_type)
    bound = None if max_norm is None else _bound(max_norm)
    dst, src = _List(acc, "acc"), _List(grads, "grads")
    if len(dst.tensors) != len(src.tensors):
        raise ValueError(f"acc and grads must be as long as one another (got "
                         f"{len(dst.tensors)} and {len(src.tensors)} tensors)")
    if kind != _lib.NORM_NONE and (dst.sharded or src.sharded):
        raise ValueError("the norm of sharded accumulators (DTensor): accumulate without one, "
                         "then clip_coef(acc, ..., process_group=...)")
    if dst.device is None:
        if kind == _lib.NORM_NONE:
            return None
        return torch.tensor(0.0) if bound is None else (torch.tensor(0.0), torch.tensor(1.0))
    device = dst.device
    if src.device != device:
        raise ValueError("acc and grads must be on one device")
    for i, (d, s) in enumerate(zip(dst.tensors, src.tensors)):
        if d.dtype == torch.float16:
            raise ValueError(f"acc must be float32 or bfloat16 tensors (got {d.dtype})")
        if d.shape != s.shape:
            raise ValueError(f"acc[{i}] and grads[{i}] differ in shape (got {tuple(d.shape)} "
                             f"and {tuple(s.shape)})")
        if d.stride() != s.stride() and not (d.is_contiguous() and s.is_contiguous()):
            raise ValueError(f"acc[{i}] and grads[{i}] differ in the order of their dimensions "
                             f"in memory (strides {d.stride()} and {s.stride()})")
        if d.is_neg() != s.is_neg():
            raise ValueError(f"acc[{i}] or grads[{i}] is a negated view")
    host, factor = _factor(scale, device, "scale")
    a = _args(src, device)
    a.accs = dst.ptrs.buffer_info()[0]
    a.acc_dtypes = ctypes.cast(ctypes.c_char_p(dst.codes), ctypes.c_void_p)
    a.host_scale, a.overwrite, a.norm_kind = host, int(overwrite), kind
    a.scale = None if factor is None else factor.data_ptr()
    norm = coef = None
    if kind != _lib.NORM_NONE:
        ws = _workspace(a, device)  # noqa: F841
        norm = _scalar(device)
        a.norm = norm.data_ptr()
        if bound is not None:
            coef = _scalar(device)
            a.coef, a.max_norm = coef.data_ptr(), bound
    _call("luma_grad_accumulate", a, device)
    _written(dst.tensors)
    if kind == _lib.NORM_NONE:
        return None
    return norm if coef is None else (norm, coef)
