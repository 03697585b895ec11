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
the same tensors (the same values at another alignment may differ by the
rounding of their sums).  All of it is outside autograd: nothing is recorded,
results carry no gradient, and tensors written in place change their version.
A function that ``torch.compile`` traces breaks its graph at these calls.  A
call may be captured in a CUDA graph; replays then work on the captured tensors'
memory.  Where a list is empty, the norm is 0 and the coefficient that of a norm
of 0, on the CPU (with an `inv_scale` on its device).

Of a DTensor in a list its local part is read and written.
"""

from __future__ import annotations

import math

import torch

from . import _lib

__all__ = ["grad_norm", "clip_coef", "scale_grads_", "clip_grads_", "accumulate_grads_"]

_KIND = {1.0: _lib.NORM_1, 2.0: _lib.NORM_2, math.inf: _lib.NORM_MAX}

_ext = None


def _ops():
    """The module that checks lists of tensors and calls the library (built
    beside it, see ``luma_b200/build.py``)."""
    global _ext
    if _ext is None:
        _lib.lib()  # with its own message where the library is missing
        try:
            from . import _grads_ext
        except ImportError as e:
            raise ImportError(f"{e}; build it with `python -m luma_b200.build`") from e
        _ext = _grads_ext
    return _ext


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


def local_scalar(t, name: str):
    """What this rank reads of a one-element factor: of a replicated DTensor its
    local copy, anything else as it is.  A part of one (sharded, or a term of a
    sum) is refused; getting the value would take a collective."""
    if type(t) is torch.Tensor or not hasattr(t, "_local_tensor"):
        return t
    if not all(p.is_replicate() for p in t.placements):
        raise ValueError(f"{name} must be replicated where it is a DTensor (got placements "
                         f"{t.placements}; full_tensor() gives its value)")
    with torch.no_grad():
        return t.to_local()


def local_flag(t, name: str):
    """A flag that this rank writes: no DTensor, whose other copies would not
    hear of it."""
    if type(t) is not torch.Tensor and hasattr(t, "_local_tensor"):
        raise ValueError(f"{name} must not be a DTensor")
    return t


def _coef_of_nothing(bound: float, inv_scale: torch.Tensor | None = None) -> torch.Tensor:
    """The coefficient where the norm is that of no elements, 0."""
    c = min(1.0, bound / 1e-6)
    if inv_scale is None:
        return torch.tensor(c)
    return inv_scale.detach().float().reshape(()).mul(c)


def _check_finite(norm: torch.Tensor) -> None:
    if not math.isfinite(float(norm)):
        raise RuntimeError("the gradients' norm is not finite, so they cannot be clipped "
                           "(error_if_nonfinite=False clips them all the same)")


def _counted(grads, group) -> list[torch.Tensor]:
    """What this rank adds to the norm over the ranks of `group`: its part of
    every tensor, but of a DTensor that several of them hold a copy of only
    where it is the first of them."""
    import torch.distributed as dist
    rank, ranks = dist.get_rank(), set(dist.get_process_group_ranks(group))
    known = {}  # (mesh, placements) -> whether this rank counts

    def counts(mesh, placements):
        if any(p.is_partial() for p in placements):
            raise ValueError("a DTensor with Partial placement holds terms of a sum, which have no "
                             f"norm of the sum (got placements {placements}; redistribute it first)")
        at = mesh.get_coordinate()
        if at is None:  # not of this mesh: no part of the tensor
            return False
        copies = mesh.mesh[tuple(slice(None) if p.is_replicate() else k
                                 for p, k in zip(placements, at))]
        return rank == min(ranks.intersection(copies.reshape(-1).tolist()), default=rank)

    out = []
    for g in [grads] if isinstance(grads, torch.Tensor) else grads:
        if hasattr(g, "_local_tensor"):
            key = g.device_mesh, g.placements
            if key not in known:
                known[key] = counts(*key)
            g = g._local_tensor if known[key] else g._local_tensor.new_empty(0)
        out.append(g)
    return out


def _over_ranks(grads, kind: int, group, max_norm=None, inv_scale=None, found_inf=None):
    """(norm, coef or None) of the lists of all ranks in `group` together."""
    import torch.distributed as dist
    if not isinstance(grads, (torch.Tensor, list, tuple)):
        grads = list(grads)
    power = _ops().power(grads, kind)  # 0 of a rank without shards
    if power is None:  # there are DTensors: which of them count takes the group
        power = _ops().power(_counted(grads, group), kind)
    if kind == _lib.NORM_MAX:
        # a maximum over ranks may drop a NaN, but no infinity
        power.nan_to_num_(nan=math.inf, posinf=math.inf)
        dist.all_reduce(power, op=dist.ReduceOp.MAX, group=group)
    else:
        dist.all_reduce(power, op=dist.ReduceOp.SUM, group=group)
    return _ops().finish(power, kind, max_norm, inv_scale, found_inf)


@torch.compiler.disable
def grad_norm(grads, norm_type: float = 2.0, *, per_tensor: bool = False,
              error_if_nonfinite: bool = False, process_group=None):
    """Norm of all elements of all tensors in `grads`, a float32 scalar on their
    device; `norm_type` is 1, 2 or inf.

    ``per_tensor=True`` returns ``(norm, norms)`` with ``norms[i]`` the norm of
    ``grads[i]`` (0 for an empty one), from the same pass.  With
    ``error_if_nonfinite`` the norm is read back and an inf or NaN raises.
    With `process_group` every rank passes its own part of the gradients and
    gets the norm over the parts of all ranks in the group; every rank of the
    group has to call, one with an empty list included.  A DTensor that several
    of them hold a copy of counts once, and one with a Partial placement is
    refused.  Other tensors (ZeRO segments) count on every rank that passes
    them: a gradient whose copies lie in plain tensors belongs into the list of
    one rank only.  (Over ranks a NaN gives an inf norm where `norm_type` is
    inf.)"""
    kind = _kind(norm_type)
    if process_group is not None:
        if per_tensor:
            raise ValueError("per_tensor norms are of whole tensors, not of shards")
        norm, norms = _over_ranks(grads, kind, process_group)[0], None
    else:
        out = _ops().norm(grads, kind, None, per_tensor, None, None, False)
        norm, _, norms = out or (torch.tensor(0.0), None, torch.zeros(0))
    if error_if_nonfinite:
        _check_finite(norm)
    return (norm, norms) if per_tensor else norm


@torch.compiler.disable
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
    one element (and no DTensor), is set to 1 if any element of the grads is
    inf or NaN, and left alone otherwise.  `error_if_nonfinite` and
    `process_group` are as in ``grad_norm``."""
    kind, bound = _kind(norm_type), _bound(max_norm)
    inv_scale = local_scalar(inv_scale, "inv_scale")
    found_inf = local_flag(found_inf, "found_inf")
    if process_group is not None:
        norm, coef = _over_ranks(grads, kind, process_group, bound, inv_scale, found_inf)
    else:
        out = _ops().norm(grads, kind, bound, False, inv_scale, found_inf, False)
        norm, coef, _ = out or (torch.tensor(0.0), _coef_of_nothing(bound, inv_scale), None)
    if error_if_nonfinite:
        _check_finite(norm)
    return norm, coef


@torch.compiler.disable
def scale_grads_(grads, coef) -> None:
    """Multiply every tensor in `grads` by `coef` in place: each element becomes
    ``round_to_its_type(fl32(g) * fl32(coef))``.  `coef` is a number or a
    one-element float32, bfloat16 or float16 tensor (of a DTensor, a replicated
    one; in host memory it is read at the call, and a captured call keeps that
    number); where it is 1 the grads are neither read nor written.  The tensors must not share memory."""
    _ops().scale(grads, local_scalar(coef, "coef"))


@torch.compiler.disable
def clip_grads_(grads, max_norm: float, norm_type: float = 2.0, *,
                error_if_nonfinite: bool = False, process_group=None) -> torch.Tensor:
    """Scale `grads` in place so that their norm is at most `max_norm`, and
    return the norm they had: ``norm, coef = clip_coef(...)``, then
    ``scale_grads_(grads, coef)``.  With `error_if_nonfinite` an inf or NaN norm
    raises before anything is written."""
    if process_group is None and not error_if_nonfinite:
        out = _ops().norm(grads, _kind(norm_type), _bound(max_norm), False, None, None, True)
        return torch.tensor(0.0) if out is None else out[0]
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    norm, coef = clip_coef(grads, max_norm, norm_type, error_if_nonfinite=error_if_nonfinite,
                           process_group=process_group)
    scale_grads_(grads, coef)
    return norm


@torch.compiler.disable
def accumulate_grads_(acc, grads, scale=1.0, *, overwrite: bool = False,
                      norm_type: float | None = None, max_norm: float | None = None):
    """``acc[i] += scale * grads[i]`` for every i, in a launch for each 960 pairs:
    a float32 product and a float32 sum per element, rounded to the accumulator's
    type.
    With `overwrite` it is ``acc[i] = scale * grads[i]`` (the first
    micro-batch), whatever `acc` held.

    `acc` are float32 or bfloat16 tensors, `grads` float32, bfloat16 or float16
    ones of the same shapes and dimension order (a DTensor and a DTensor also of
    the same mesh and placements; a plain tensor beside one is a buffer for this
    rank's part of it); `scale` is a number or a
    one-element tensor as in ``scale_grads_``.  ``grads[i]`` may be ``acc[i]``
    itself; other overlaps are refused.

    With `norm_type` (1, 2 or inf) the norm of the accumulators as they are
    afterwards is returned, from the same pass (and a launch that joins its sums);
    with `max_norm` it is ``(norm, coef)`` as of ``clip_coef(acc, max_norm,
    norm_type or 2)``, to the rounding of sums in another order.  Otherwise
    nothing is returned."""
    kind = _lib.NORM_NONE
    if norm_type is not None or max_norm is not None:
        kind = _kind(2.0 if norm_type is None else norm_type)
    bound = None if max_norm is None else _bound(max_norm)
    out = _ops().accumulate(acc, grads, local_scalar(scale, "scale"), overwrite, kind, bound)
    if kind == _lib.NORM_NONE:
        return None
    if out is None:
        norm, coef = torch.tensor(0.0), None if bound is None else _coef_of_nothing(bound)
    else:
        norm, coef = out
    return norm if bound is None else (norm, coef)
