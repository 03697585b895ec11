"""Gradient operators and wrapper tensors (DTensors), without a GPU: what is
refused, which of a group's ranks counts a replicated gradient, and the
arguments around them."""

import math

import pytest
import torch

import luma_b200
from luma_b200 import amp


class OnCuda(torch.Tensor):
    """A wrapper that passes for a float32 CUDA tensor in the checks and has no
    memory; further attributes make it pass for a DTensor."""

    @staticmethod
    def __new__(cls, shape=(0,), strides=None, **attrs):
        t = torch.Tensor._make_wrapper_subclass(cls, shape, strides=strides, dtype=torch.float32,
                                                device="cuda:0")
        for k, v in attrs.items():
            setattr(t, k, v)
        return t

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        if func is torch.ops.aten.detach.default:
            return cls(args[0].shape)
        raise AssertionError(func)


class Place:
    """A DTensor placement as far as the operators look at it."""

    def __init__(self, kind):
        self.kind = kind

    def is_replicate(self):
        return self.kind == "replicate"

    def is_partial(self):
        return self.kind == "partial"

    def __eq__(self, other):
        return self.kind == other.kind

    def __hash__(self):
        return hash(self.kind)

    def __repr__(self):
        return self.kind


def like_dtensor(*kinds, shape=(0,), local=None, mesh="mesh"):
    return OnCuda(shape, _local_tensor=OnCuda() if local is None else local, device_mesh=mesh,
                  placements=tuple(Place(k) for k in kinds))


# -- factors and flags -----------------------------------------------------------

SCALARS = [("coef", lambda g, t: luma_b200.scale_grads_(g, t)),
           ("scale", lambda g, t: luma_b200.accumulate_grads_(g, [OnCuda()], t)),
           ("inv_scale", lambda g, t: luma_b200.clip_coef(g, 1.0, inv_scale=t)),
           ("found_inf", lambda g, t: luma_b200.clip_coef(g, 1.0, found_inf=t))]


@pytest.mark.parametrize("name,call", SCALARS, ids=[n for n, _ in SCALARS])
@pytest.mark.parametrize("kinds", [("shard",), ("partial",), ("replicate", "partial")])
def test_a_distributed_scalar_is_refused(name, call, kinds):
    """Its value is not this rank's part of it."""
    with pytest.raises(ValueError, match=f"{name} .*(replicated|DTensor)"):
        call([OnCuda()], like_dtensor(*kinds, shape=(1,), local=OnCuda((1,))))


def test_a_replicated_flag_is_refused():
    """Every rank would write its own copy only."""
    with pytest.raises(ValueError, match="found_inf .*DTensor"):
        luma_b200.clip_coef([OnCuda()], 1.0, found_inf=like_dtensor("replicate", shape=(1,),
                                                                    local=OnCuda((1,))))


@pytest.mark.parametrize("name,call", SCALARS, ids=[n for n, _ in SCALARS])
def test_a_scalar_without_memory_is_refused(name, call):
    """Its address is 0, which a kernel takes for "no factor"."""
    with pytest.raises(ValueError, match=f"{name} .*memory"):
        call([OnCuda()], OnCuda((1,)))
