"""``GradScaler.unscale_`` and the inf/NaN skip fused into the LUMA step.

Mixed-precision training with ``torch.amp.GradScaler`` runs, per iteration,
``scaler.step(opt)``: ``unscale_`` (one pass that reads and rewrites every
grad: ``g <- g * (1/scale)`` and a found-inf flag per device,
``torch._amp_foreach_non_finite_check_and_unscale_``), then a host read of the
flag, then ``opt.step()`` unless a grad was inf or NaN (reference usage:
IgorYashch/LUMA tests/test_mixed_precision.py:119-184).

``scaler_step(scaler, opt)`` gives the same results without the extra pass:
the LUMA step reads each grad as ``round_to_grad_dtype(fl32(g) * inv_scale)``
(what ``unscale_`` would have stored), its first pass raises the device flag
on any inf/NaN grad, and its second pass changes nothing when the flag is set.
The flag is recorded in the scaler's per-optimizer state, so
``scaler.update()`` backs off or grows the scale exactly as after
``scaler.step(opt)``.

``clip_step(scaler, opt, max_norm)`` is the same with the grads' norm clipped:
one pass over the grads takes the norm (of the unscaled values) and the
inf/NaN flag, and the step multiplies by one coefficient that holds both the
unscaling and the clipping.  In place of ``scaler.unscale_(opt)``, clipping,
``scaler.step(opt)``: two passes that rewrite the grads fewer.

Both rely on ``GradScaler``'s per-optimizer bookkeeping
(``_per_optimizer_states``, ``OptState``), which torch has kept since 1.6.
"""

from __future__ import annotations

import torch
from torch.amp.grad_scaler import OptState

from .grads import clip_coef

__all__ = ["clip_step", "scaler_step"]


def _scaled_grads(scaler, optimizer, kwargs):
    """(the optimizer's grads, its state in the scaler) of a step to take;
    raises what ``GradScaler.step`` raises."""
    if "closure" in kwargs:
        raise RuntimeError("Closure use is not currently supported if GradScaler is enabled.")
    state = scaler._per_optimizer_states[id(optimizer)]
    if state["stage"] is OptState.STEPPED:
        raise RuntimeError("step() has already been called since the last update().")
    grads = [p.grad for g in optimizer.param_groups for p in g["params"] if p.grad is not None]
    if state["stage"] is not OptState.UNSCALED and any(gr.dtype == torch.float16 for gr in grads):
        # GradScaler.unscale_ refuses fp16 grads (fp16 params): same error
        raise ValueError("Attempting to unscale FP16 gradients.")
    return grads, state


def _unscaling(scaler, grads):
    """(inv_scale, found_inf) on the grads' device, the flag 0."""
    scaler._check_scale_growth_tracker("step")
    # The reciprocal in float64, then float32: GradScaler.unscale_'s inv_scale.
    dev = grads[0].device if grads else scaler._scale.device
    inv_scale = scaler._scale.double().reciprocal().float().to(dev)
    return inv_scale, torch.full((), 0.0, dtype=torch.float32, device=dev)


def scaler_step(scaler: torch.amp.GradScaler, optimizer, *args, **kwargs):
    """Drop-in for ``scaler.step(optimizer)`` with a ``luma_b200.LUMA`` optimizer.

    Falls back to ``scaler.step`` when the fused path does not apply: the
    scaler is disabled, the caller already ran ``scaler.unscale_(optimizer)``
    (e.g. to clip), or the stepped params span several devices (a skip must
    cover all of them, which one device's flag cannot order).
    """
    if not scaler.is_enabled():
        return optimizer.step(*args, **kwargs)
    grads, state = _scaled_grads(scaler, optimizer, kwargs)
    if state["stage"] is OptState.UNSCALED or len({gr.device for gr in grads}) > 1:
        return scaler.step(optimizer, *args, **kwargs)
    inv_scale, found_inf = _unscaling(scaler, grads)
    retval = optimizer.step(*args, grad_scale=inv_scale, found_inf=found_inf, **kwargs)
    state["found_inf_per_device"] = {found_inf.device: found_inf}
    state["stage"] = OptState.STEPPED
    return retval


def clip_step(scaler: torch.amp.GradScaler, optimizer, max_norm: float, norm_type: float = 2.0,
              *, process_group=None, **kwargs) -> torch.Tensor:
    """``scaler_step`` with the unscaled grads clipped to `max_norm` (their
    ``clip_coef``); returns the norm they had, inf or NaN on a step that is
    skipped.  The grads themselves keep their values.  Also takes a disabled
    scaler (clip and step) and grads the caller already unscaled; the grads
    have to be on one device.  With sharded grads every rank of `process_group`
    calls, and the norm and the inf/NaN flag are those of all ranks' parts (as
    in ``clip_coef``; grads already unscaled have ``unscale_``'s flag).  A closure is refused: it would change the grads after
    their norm was taken."""
    over = {} if process_group is None else {"process_group": process_group}
    if not scaler.is_enabled():
        if kwargs.get("closure") is not None:
            raise RuntimeError("clip_step does not support a closure: it would change the grads "
                               "after their norm was taken.")
        grads = [p.grad for g in optimizer.param_groups for p in g["params"] if p.grad is not None]
        norm, coef = clip_coef(grads, max_norm, norm_type, **over)
        optimizer.step(grad_scale=coef, **kwargs)
        return norm
    grads, state = _scaled_grads(scaler, optimizer, kwargs)
    if state["stage"] is OptState.UNSCALED:
        norm, coef = clip_coef(grads, max_norm, norm_type, **over)
        scaler.step(optimizer, grad_scale=coef, **kwargs)
        return norm
    inv_scale, found_inf = _unscaling(scaler, grads)
    norm, coef = clip_coef(grads, max_norm, norm_type, inv_scale=inv_scale, found_inf=found_inf,
                           **over)
    optimizer.step(grad_scale=coef, found_inf=found_inf, **kwargs)
    state["found_inf_per_device"] = {found_inf.device: found_inf}
    state["stage"] = OptState.STEPPED
    return norm
