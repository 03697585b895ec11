"""Gradient operators on the GPU with DTensors, host factors and views: the
calls whose answer depends on what a tensor object is, besides its elements.
Values are small integers and powers of two, so results are exact."""

import math

import pytest
import torch

import luma_b200
from luma_b200 import LUMA, accumulate_grads_, clip_coef, clip_grads_, grad_norm, scale_grads_

pytestmark = pytest.mark.gpu


@pytest.fixture
def mesh(tmp_path):
    """The device mesh of one rank."""
    import torch.distributed as dist
    from torch.distributed.tensor import init_device_mesh
    dist.init_process_group("gloo", init_method=f"file://{tmp_path}/store", rank=0, world_size=1)
    try:
        yield init_device_mesh("cuda", (1,))
    finally:
        dist.destroy_process_group()


def distributed(mesh, local, kind="replicate"):
    from torch.distributed.tensor import DTensor, Partial, Replicate, Shard
    placement = {"replicate": Replicate(), "shard": Shard(0), "partial": Partial()}[kind]
    return DTensor.from_local(local, mesh, [placement], run_check=False)


def full(value, n=1):
    return torch.full((n,), float(value), device="cuda")


# -- factors and flags -----------------------------------------------------------

def test_replicated_factors_count(mesh):
    """A replicated DTensor is the number it holds."""
    x, acc = full(8, 9), full(1, 9)
    scale_grads_([x], distributed(mesh, full(0.25)))
    assert (x == 2).all()
    scale_grads_([x], distributed(mesh, torch.tensor(0.5, device="cuda")))
    assert (x == 1).all()
    accumulate_grads_([acc], [x], distributed(mesh, full(3).bfloat16()))
    assert (acc == 4).all()
    norm, coef = clip_coef([acc], 1e9, inv_scale=distributed(mesh, full(0.125)))
    assert norm == 1.5 and coef == 0.125


def test_the_coefficient_of_sharded_gradients(mesh):
    """clip_grad_coef of DTensor gradients gives a DTensor; scaling by it clips."""
    ps = []
    for k in range(2):
        p = torch.nn.Parameter(distributed(mesh, full(0, 8), "shard"))
        p.grad = distributed(mesh, full(3 + k, 8), "shard")
        ps.append(p)
    norm, coef = luma_b200.clip_grad_coef(ps, 1.0)
    scale_grads_([p.grad for p in ps], coef)
    after = math.sqrt(sum(float(p.grad.to_local().double().square().sum()) for p in ps))
    assert abs(after - 1) < 1e-6  # a coefficient within 4 roundings, a product within one


@pytest.mark.parametrize("kind", ["shard", "partial"])
def test_parts_of_a_factor_are_refused(mesh, kind):
    x = full(8, 9)
    part = distributed(mesh, full(0.25), kind)
    for call in (lambda: scale_grads_([x], part), lambda: accumulate_grads_([x], [x], part),
                 lambda: clip_coef([x], 1.0, inv_scale=part),
                 lambda: clip_coef([x], 1.0, found_inf=part)):
        with pytest.raises(ValueError, match="replicated|DTensor"):
            call()
    with pytest.raises(ValueError, match="found_inf .*DTensor"):
        clip_coef([x], 1.0, found_inf=distributed(mesh, full(0)))
    assert (x == 8).all()


# -- lists of DTensors --------------------------------------------------------------

def test_norms_of_dtensors(mesh):
    import torch.distributed as dist
    world = dist.group.WORLD
    a, b = full(3, 9), full(2, 1000)
    for kinds in (("shard", "shard"), ("replicate", "shard"), ("replicate", "replicate")):
        ts = [distributed(mesh, t, k) for t, k in zip((a, b), kinds)]
        ts.append(full(6, 1))
        assert grad_norm(ts, process_group=world) == math.sqrt(81 + 4000 + 36)
        assert grad_norm(ts, math.inf, process_group=world) == 6.0
        norm, coef = clip_coef(ts, 1e9, process_group=world)
        assert norm == math.sqrt(81 + 4000 + 36) and coef == 1.0
        with pytest.raises(ValueError, match="process_group"):
            grad_norm(ts)
        with pytest.raises(ValueError, match="process_group"):
            clip_grads_(ts, 1.0)
    assert grad_norm(distributed(mesh, a), process_group=world) == 9.0
    ts = [distributed(mesh, a), distributed(mesh, b, "partial")]
    for call in (grad_norm, lambda g, **kw: clip_grads_(g, 1.0, **kw)):
        with pytest.raises(ValueError, match="Partial"):
            call(ts, process_group=world)
    assert (a == 3).all() and (b == 2).all()
    ts = [distributed(mesh, full(3, 16), "shard"), distributed(mesh, full(4, 16))]
    assert clip_grads_(ts, 10.0, process_group=world) == 20.0
    for t, want in zip(ts, (1.5, 2.0)):
        assert (t.to_local() / want - 1).abs().max() < 1e-6  # max_norm / (norm + 1e-6)


def test_accumulation_of_dtensors(mesh):
    acc, g = full(1, 9), full(2, 9)
    for kind in ("shard", "replicate", "partial"):
        x = distributed(mesh, acc, kind)
        accumulate_grads_([x], [distributed(mesh, g, kind)], 0.5, overwrite=kind == "partial")
    assert (acc == 1).all()  # written in place, the last time anew
    accumulate_grads_([acc], [distributed(mesh, g, "shard")], 0.5)  # a buffer of this rank's own
    assert (acc == 2).all()
    for other in ("replicate", "partial"):
        with pytest.raises(ValueError, match="placements"):
            accumulate_grads_([distributed(mesh, acc, "shard")], [distributed(mesh, g, other)])
    with pytest.raises(ValueError, match="sharded"):
        accumulate_grads_([distributed(mesh, acc)], [distributed(mesh, g)], norm_type=2.0)
    assert (acc == 2).all()


def test_written_dtensors_change_their_version(mesh):
    """Autograd looks at the version of the tensor it saved, the DTensor."""
    x = distributed(mesh, full(1, 9))
    before = x._version, x.to_local()._version
    scale_grads_([x], 0.5)
    assert x._version > before[0] and x.to_local()._version > before[1]


# -- the step's own factor ------------------------------------------------------------

def test_step_with_a_replicated_coefficient(mesh):
    ps = [torch.nn.Parameter(full(1, 100)) for _ in range(2)]
    opts = [LUMA([p], lr=0.1) for p in ps]
    opts[1]._base_seed = opts[0]._base_seed
    gen = torch.Generator(device="cuda").manual_seed(0)
    for _ in range(2):
        g = torch.randn(100, device="cuda", generator=gen)
        for p in ps:
            p.grad = g
        opts[0].step(grad_scale=full(0.01))
        opts[1].step(grad_scale=distributed(mesh, full(0.01)))
    assert torch.equal(*ps)
    with pytest.raises(ValueError, match="grad_scale .*replicated"):
        opts[0].step(grad_scale=distributed(mesh, full(1), "partial"))
    assert torch.equal(*ps)


def test_zero_step_with_a_replicated_coefficient(mesh):
    from luma_b200.zero import ZeroLUMA, plan_layout
    layout = plan_layout([1000, 7], world=1, buckets=1)
    flats = [torch.ones(layout.total, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    zs = [ZeroLUMA(f, layout, 0) for f in flats]
    gen = torch.Generator(device="cuda").manual_seed(0)
    for _ in range(2):
        grad = torch.randn(layout.shard, device="cuda", generator=gen)
        zs[0].step(grad, grad_scale=full(0.01))
        zs[1].step(grad, grad_scale=distributed(mesh, full(0.01)))
    assert torch.equal(*flats)
    with pytest.raises(ValueError, match="grad_scale .*replicated"):
        zs[1].step(grad, grad_scale=distributed(mesh, full(0.01), "shard"))


# -- factors in host memory --------------------------------------------------------------

FACTOR_CALLS = [lambda x, c: scale_grads_([x], c),
                lambda x, c: accumulate_grads_([x], [x.clone()], c, overwrite=True)]


@pytest.mark.parametrize("call", FACTOR_CALLS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_a_host_factor_is_read_at_the_call(call, dtype):
    """Pinned or not: what is written to it afterwards, with the call still
    queued behind other work, belongs to the next call."""
    for pin in (True, False):
        c = torch.full((1,), 0.5, dtype=dtype)
        c = c.pin_memory() if pin else c
        x = full(8, 1000)
        torch.cuda.synchronize()
        torch.cuda._sleep(100_000_000)
        call(x, c)
        c.fill_(4.0)
        torch.cuda.synchronize()
        assert (x == 4).all()


@pytest.mark.parametrize("pin", [True, False])
def test_a_host_factor_in_a_capture(pin):
    """A replay uses the number that was captured."""
    c = torch.full((), 0.5)
    c = c.pin_memory() if pin else c
    x = full(64, 1000)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        scale_grads_([x], c)
    c.fill_(100.0)
    graph.replay()
    graph.replay()
    assert (x == 16).all()


def test_step_reads_a_host_scale_at_the_call():
    ps = [torch.nn.Parameter(full(1, 100)) for _ in range(2)]
    opts = [LUMA([p], lr=0.1) for p in ps]
    opts[1]._base_seed = opts[0]._base_seed
    gen = torch.Generator(device="cuda").manual_seed(0)
    host = torch.ones(1).pin_memory()
    for _ in range(2):
        g = torch.randn(100, device="cuda", generator=gen)
        for p in ps:
            p.grad = g
        opts[0].step(grad_scale=full(0.01))
        host.fill_(0.01)
        torch.cuda.synchronize()
        torch.cuda._sleep(100_000_000)
        opts[1].step(grad_scale=host)
        host.fill_(100.0)
    assert torch.equal(*ps)


# -- views -------------------------------------------------------------------------------

def test_negated_views_as_scalars():
    """A view whose memory holds minus its value."""
    x = full(2, 16)
    norm, coef = clip_coef([x], 1e9, inv_scale=torch._neg_view(full(-0.25)))
    assert norm == 2.0 and coef == 0.25
    with pytest.raises(ValueError, match="found_inf .*negated"):
        clip_coef([x], 1.0, found_inf=torch._neg_view(full(0)))
    scale_grads_([x], torch._neg_view(full(-0.25)))
    assert (x == 0.5).all()


def test_step_with_a_negated_view():
    ps = [torch.nn.Parameter(full(1, 100)) for _ in range(2)]
    opts = [LUMA([p], lr=0.1) for p in ps]
    opts[1]._base_seed = opts[0]._base_seed
    gen = torch.Generator(device="cuda").manual_seed(0)
    for _ in range(2):
        g = torch.randn(100, device="cuda", generator=gen)
        for p in ps:
            p.grad = g
        opts[0].step(grad_scale=full(0.01))
        opts[1].step(grad_scale=torch._neg_view(full(-0.01)))
    assert torch.equal(*ps)
    with pytest.raises(ValueError, match="found_inf"):
        opts[0].step(found_inf=torch._neg_view(full(0)))


def test_strides_of_single_rows():
    """A dimension of size 1 has a stride and no place in the order."""
    a = torch.empty_strided((4, 1, 6), (1, 1, 4), device="cuda").fill_(1.0)
    for strides in ((1, 24, 4), (1, 4, 4), (1, 7, 4)):
        g = torch.empty_strided((4, 1, 6), strides, dtype=torch.bfloat16, device="cuda")
        g.copy_(torch.arange(24, device="cuda").view(4, 1, 6))
        assert not g.is_contiguous()
        before = a.clone()
        accumulate_grads_([a], [g], 2.0)
        assert torch.equal(a, before + 2 * g.float())
    with pytest.raises(ValueError, match="order"):
        accumulate_grads_([a], [torch.zeros(4, 1, 6, device="cuda")])


# -- mixed precision with sharded gradients --------------------------------------------------

def test_clip_step_of_dtensors(mesh):
    """The params of a step on the same gradients in plain tensors."""
    import torch.distributed as dist
    gen = torch.Generator(device="cuda").manual_seed(0)
    init = [torch.randn(n, device="cuda", generator=gen) for n in (1000, 7)]
    plain = [torch.nn.Parameter(t.clone()) for t in init]
    kinds = ("shard", "replicate")
    shards = [torch.nn.Parameter(distributed(mesh, t.clone(), k)) for t, k in zip(init, kinds)]
    opts = [LUMA(ps, lr=1e-2) for ps in (plain, shards)]
    opts[1]._base_seed = opts[0]._base_seed
    scalers = [torch.amp.GradScaler("cuda", init_scale=2.0 ** 12) for _ in opts]
    for it in range(4):
        raw = [torch.randn(t.shape, device="cuda", generator=gen) for t in init]
        if it == 2:
            raw[0][5] = math.inf
        norms = []
        for ps, opt, scaler, over in zip((plain, shards), opts, scalers, (None, dist.group.WORLD)):
            scale = scaler.scale(torch.ones((), device="cuda"))
            for p, g, k in zip(ps, raw, kinds):
                p.grad = g * scale if ps is plain else distributed(mesh, g * scale, k)
            norms.append(luma_b200.amp.clip_step(scaler, opt, 1.0, process_group=over))
            scaler.update()
        assert torch.equal(*norms) and math.isfinite(norms[0]) == (it != 2)
        assert scalers[0].get_scale() == scalers[1].get_scale()
        assert all(torch.equal(a, b.to_local()) for a, b in zip(plain, shards)), it
