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


# -- the norm over ranks -----------------------------------------------------------

class Ops:
    """The list module in elementary operations on CPU tensors; DTensors are
    left to the caller, who knows the ranks."""

    @staticmethod
    def power(grads, kind):
        if any(hasattr(g, "_local_tensor") for g in grads):
            return None
        x = torch.cat([torch.zeros(1, dtype=torch.float64), *(g.double().reshape(-1) for g in grads)])
        x = x.abs()
        return {1: x.sum(), 2: (x * x).sum(), 3: x.max()}[kind].reshape(1)

    @staticmethod
    def finish(power, kind, max_norm, inv_scale, found_inf):
        norm = (power.sqrt() if kind == 2 else power)[0]
        return norm, None if max_norm is None else torch.clamp(max_norm / (norm + 1e-6), max=1.0)

    @staticmethod
    def scale(grads, coef):
        for g in grads:
            g.to_local().mul_(coef)


def _rank(rank, store, ok):
    import torch.distributed as dist
    from torch.distributed.tensor import DTensor, Partial, Replicate, Shard, init_device_mesh
    from luma_b200 import grads as module
    module._ext = Ops
    dist.init_process_group("gloo", init_method=f"file://{store}", rank=rank, world_size=4)
    world = dist.group.WORLD
    mesh = init_device_mesh("cpu", (2, 2), mesh_dim_names=("copies", "shards"))
    row, col = mesh.get_coordinate()

    def tensor(value, *placements):
        return DTensor.from_local(torch.full((3,), float(value)), mesh, placements, run_check=False)

    both = tensor(2, Replicate(), Replicate())           # 3 elements of 2
    hybrid = tensor(3 + col, Replicate(), Shard(0))      # 3 of 3, 3 of 4
    split = tensor(1 + rank, Shard(0), Shard(0))         # 3 each of 1, 2, 3, 4
    plain = torch.full((2,), 10.0 * rank)                # 2 each of 0, 10, 20, 30
    everything = [both, hybrid, split, plain]
    powers = [3 * 4, 3 * (9 + 16), 3 * (1 + 4 + 9 + 16), 2 * (100 + 400 + 900)]
    for k in range(4):
        assert module.grad_norm([everything[k]], process_group=world) == math.sqrt(powers[k]), k
    assert module.grad_norm(both, process_group=world) == math.sqrt(12)
    assert module.grad_norm(iter(everything), process_group=world) == math.sqrt(sum(powers))
    assert module.grad_norm([both, hybrid], 1.0, process_group=world) == 6 + 21
    assert module.grad_norm([both, hybrid], math.inf, process_group=world) == 4.0
    norm, coef = module.clip_coef([hybrid], 1.0, process_group=world)
    assert norm == math.sqrt(75) and abs(coef * math.sqrt(75) - 1) < 1e-5
    # the ranks of one copy: a copy of everything
    copy = mesh["shards"].get_group()
    assert module.grad_norm([both, hybrid], process_group=copy) == math.sqrt(12 + 75)
    # the two copies of one shard: counted once
    assert module.grad_norm([hybrid], process_group=mesh["copies"].get_group()) == \
        math.sqrt(3 * (3 + col) ** 2)
    # clipping scales every copy
    norm = module.clip_grads_([both, hybrid], math.sqrt(87) / 2, process_group=world)
    assert norm == math.sqrt(87)
    assert (both.to_local() - 1).abs().max() < 1e-6
    assert (hybrid.to_local() - (3 + col) / 2).abs().max() < 1e-6
    # parts of a sum have no norm of their own
    for call in (module.grad_norm, lambda g, **kw: module.clip_coef(g, 1.0, **kw),
                 lambda g, **kw: module.clip_grads_(g, 1.0, **kw)):
        try:
            call([both, tensor(1, Shard(0), Partial())], process_group=world)
        except ValueError as e:
            assert "Partial" in str(e)
        else:
            raise AssertionError("no error")
    dist.destroy_process_group()
    ok[rank] = 1


def test_copies_of_a_gradient_count_once(tmp_path):
    ctx = torch.multiprocessing.get_context("spawn")
    ok = ctx.Array("i", 4)
    ranks = [ctx.Process(target=_rank, args=(r, tmp_path / "store", ok)) for r in range(4)]
    for p in ranks:
        p.start()
    for p in ranks:
        p.join(180)
        assert p.exitcode == 0
    assert list(ok) == [1] * 4


def test_sharded_lists_need_a_group():
    for call in (luma_b200.grad_norm, lambda g: luma_b200.clip_coef(g, 1.0),
                 lambda g: luma_b200.clip_grads_(g, 1.0)):
        with pytest.raises(ValueError, match="process_group"):
            call([like_dtensor("shard")])


# -- accumulation of DTensors --------------------------------------------------------

@pytest.mark.parametrize("acc,grad,word", [
    (like_dtensor("shard"), like_dtensor("replicate"), "placements"),
    (like_dtensor("partial"), like_dtensor("replicate"), "placements"),
    (like_dtensor("shard"), like_dtensor("shard", mesh="another"), "mesh"),
    (like_dtensor("shard", shape=(5,)), like_dtensor("shard", shape=(6,)), "shape"),
])
def test_accumulate_refuses_other_placements(acc, grad, word):
    """Parts of equal shape that are not the same part."""
    with pytest.raises(ValueError, match=rf"acc\[1\] and grads\[1\] differ in .*{word}"):
        luma_b200.accumulate_grads_([like_dtensor("shard"), acc], [like_dtensor("shard"), grad])


# -- the step's own factor -----------------------------------------------------------

def test_step_refuses_distributed_scalars():
    opt = luma_b200.LUMA([torch.nn.Parameter(torch.zeros(4))])
    for kinds in (("shard",), ("partial",)):
        with pytest.raises(ValueError, match="grad_scale .*replicated"):
            opt.step(grad_scale=like_dtensor(*kinds, shape=(1,), local=OnCuda((1,))))
    with pytest.raises(ValueError, match="found_inf .*DTensor"):
        opt.step(found_inf=like_dtensor("replicate", shape=(1,), local=OnCuda((1,))))


def test_step_refuses_scalars_without_memory(monkeypatch):
    monkeypatch.setattr(OnCuda, "reshape", lambda t, *shape: t)
    monkeypatch.setattr(OnCuda, "data_ptr", lambda t: 0)
    opt = luma_b200.LUMA([torch.nn.Parameter(torch.zeros(4))])
    for name in ("grad_scale", "found_inf"):
        with pytest.raises(ValueError, match=f"{name} .*memory"):
            opt.step(**{name: OnCuda((1,))})


# -- amp.clip_step -------------------------------------------------------------------

class Optimizer(torch.optim.Optimizer):
    def __init__(self, *grads):
        ps = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
        for p, g in zip(ps, grads):
            p.grad = g
        super().__init__(ps or [torch.nn.Parameter(torch.zeros(1))], {})
        self.calls = []

    def step(self, closure=None, *, grad_scale=None, found_inf=None):
        self.calls.append((closure, grad_scale, found_inf))


def test_clip_step_refuses_a_closure_with_a_disabled_scaler(monkeypatch):
    """It would run after the norm was taken: the coefficient would be that of
    other gradients."""
    monkeypatch.setattr(amp, "clip_coef", lambda *a, **kw: (torch.tensor(2.0), torch.tensor(0.5)))
    off = torch.amp.GradScaler("cpu", enabled=False)
    opt = Optimizer(torch.ones(4))
    with pytest.raises(RuntimeError, match="[Cc]losure"):
        amp.clip_step(off, opt, 1.0, closure=lambda: 1.0)
    assert opt.calls == []
    assert amp.clip_step(off, opt, 1.0, closure=None) == 2.0
    assert opt.calls == [(None, torch.tensor(0.5), None)]


# -- empty lists -----------------------------------------------------------------------

def test_coefficient_of_an_empty_list():
    """min(1, max_norm / 1e-6), times the unscaling."""
    inv = torch.tensor([0.125])
    norm, coef = luma_b200.clip_coef([], 1.0, inv_scale=inv)
    assert norm == 0.0 and coef == 0.125 and coef.shape == () and coef.dtype == torch.float32
    inv.fill_(1.0)
    assert coef == 0.125  # a value of its own
    assert luma_b200.clip_coef([], 0.0)[1] == 0.0
    assert luma_b200.clip_coef([], 2.5e-7)[1] == 0.25
    assert luma_b200.clip_coef([], math.inf)[1] == 1.0
    assert luma_b200.accumulate_grads_([], [], max_norm=0.0) == (0.0, 0.0)


# -- the module that was built for another torch ------------------------------------------

def test_module_of_another_torch_is_refused():
    import subprocess
    import sys
    code = """
import torch
torch.__version__ = "1.0.0"
import luma_b200
try:
    luma_b200.grad_norm([])
except ImportError as e:
    assert "luma_b200.build" in str(e) and "1.0.0" in str(e), e
else:
    raise AssertionError("loaded")
from luma_b200 import build
assert build.is_stale()
"""
    root = luma_b200.__path__[0].rsplit("/", 1)[0]
    subprocess.run([sys.executable, "-c", code], check=True, cwd=root, timeout=300)


def test_library_without_torch(monkeypatch, tmp_path):
    """A host of the C ABI alone builds the library and is told about the rest."""
    import builtins
    from luma_b200 import build
    real = builtins.__import__

    def none(name, *a, **kw):
        if name == "torch" or name.startswith("torch."):
            raise ImportError(name)
        return real(name, *a, **kw)
    monkeypatch.setattr(builtins, "__import__", none)
    ran = []
    monkeypatch.setattr(build, "OUT", str(tmp_path / "lib.so"))
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, check: (
        ran.append(cmd[0]), (tmp_path / "lib.so.tmp").write_bytes(b"")))
    assert build.build() == str(tmp_path / "lib.so")
    assert len(ran) == 1 and "nvcc" in ran[0]


def test_clip_step_over_ranks(monkeypatch):
    """Sharded gradients take the group that their norm is reduced over."""
    seen = []

    def coef(grads, max_norm, norm_type=2.0, *, inv_scale=None, found_inf=None, process_group=None):
        seen.append((max_norm, norm_type, inv_scale, found_inf, process_group))
        return torch.tensor(2.0), torch.tensor(0.5)
    monkeypatch.setattr(amp, "clip_coef", coef)
    group = object()
    for enabled, unscaled in ((False, False), (True, False), (True, True)):
        scaler = torch.amp.GradScaler("cpu", enabled=enabled, init_scale=4.0)
        scaler.scale(torch.ones(()))
        opt = Optimizer(torch.ones(4))
        if unscaled:
            scaler.unscale_(opt)
        assert amp.clip_step(scaler, opt, 0.5, math.inf, process_group=group) == 2.0
        max_norm, norm_type, inv_scale, found_inf, over = seen.pop()
        assert (max_norm, norm_type) == (0.5, math.inf) and over is group and not seen
        fused = enabled and not unscaled
        assert (inv_scale is not None) == fused and (found_inf is not None) == fused
        (_, gs, fi), = opt.calls
        assert gs == 0.5 and fi is found_inf
