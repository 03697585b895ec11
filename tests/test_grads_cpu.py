"""Gradient operators without a GPU: what they refuse, in Python and at the C
entries (checked on the host before any device call), empty lists, and the
dispatch of the fused GradScaler step with clipping."""

import ctypes
import math
from array import array

import pytest
import torch
from torch.amp.grad_scaler import OptState

import luma_b200
from luma_b200 import _lib, amp
from luma_b200.grads import _ops

from test_host_abi import _c_offsets


@pytest.fixture(autouse=True)
def _no_message_left():
    """The library keeps a thread's last message; later tests expect none."""
    yield
    _lib.lib().luma_step(ctypes.byref(_lib.LumaStepArgs()), None)


# -- the C entries -------------------------------------------------------------

def test_args_layout(tmp_path):
    fields = [f for f, _ in _lib.LumaGradArgs._fields_]
    size, offs = _c_offsets("LumaGradArgs", fields, tmp_path)
    assert size == ctypes.sizeof(_lib.LumaGradArgs)
    assert offs == [getattr(_lib.LumaGradArgs, f).offset for f in fields]
    out = (ctypes.c_int64 * 6)()
    assert _lib.lib().luma_struct_sizes(out, 6) == 6 and out[5] == size


class Call:
    """LumaGradArgs over made-up addresses: nothing here reaches a kernel."""

    def __init__(self, ptrs, numels, codes, accs=None, acc_codes=None, **kw):
        self.keep = [array("Q", ptrs), array("q", numels), bytes(codes)]
        self.args = a = _lib.LumaGradArgs()
        a.grads, a.numel = (x.buffer_info()[0] for x in self.keep[:2])
        a.dtypes = ctypes.cast(ctypes.c_char_p(self.keep[2]), ctypes.c_void_p)
        if accs is not None:
            self.keep += [array("Q", accs), bytes(acc_codes)]
            a.accs = self.keep[3].buffer_info()[0]
            a.acc_dtypes = ctypes.cast(ctypes.c_char_p(self.keep[4]), ctypes.c_void_p)
        a.n, a.host_scale, a.norm_kind = len(ptrs), 1.0, _lib.NORM_2
        a.partials, a.n_partials = 256, _lib.grad_partials(len(ptrs))
        for k, v in kw.items():
            setattr(a, k, v)

    def refused(self, name, *words):
        h = _lib.lib()
        assert getattr(h, name)(ctypes.byref(self.args), None) == _lib.LUMA_ERR_INVALID
        msg = h.luma_last_error().decode()
        assert all(w in msg for w in words), msg


F, B, H = _lib.F32, _lib.BF16, _lib.F16
LISTS = ("luma_grad_norm", "luma_grad_scale", "luma_grad_clip", "luma_grad_accumulate")


@pytest.mark.parametrize("name", LISTS)
def test_c_entries_refuse_bad_lists(name):
    assert getattr(_lib.lib(), name)(None, None) == _lib.LUMA_ERR_INVALID

    def call(*a, **kw):
        return Call(*a, accs=[1 << 20] * len(a[0]), acc_codes=[F] * len(a[0]), coef=64, **kw)
    call([4096], [-1], [F]).refused(name, "negative")
    call([4096], [8], [3]).refused(name, "type")
    call([0], [8], [F]).refused(name, "address")
    call([4098], [8], [F]).refused(name, "address")
    call([4097], [8], [B]).refused(name, "address")
    call([4096], [8], [F], n=-1).refused(name, "tensors")
    call([4096], [8], [F], n=(1 << 24) + 1).refused(name, "tensors")
    call([4096], [8], [F], device=-1).refused(name, "device")
    call([4096], [8], [F], grads=None).refused(name, "NULL")


@pytest.mark.parametrize("name", ["luma_grad_norm", "luma_grad_clip", "luma_grad_accumulate"])
def test_c_entries_refuse_bad_norms(name):
    def call(**kw):
        return Call([4096], [8], [F], accs=[1 << 20], acc_codes=[F], **{"coef": 64, **kw})
    call(norm_kind=4).refused(name, "norm kind")
    call(partials=None).refused(name, "workspace")
    call(n_partials=_lib.grad_partials(1) - 1).refused(name, "workspace")
    call(max_norm=-1.0).refused(name, "max_norm")
    call(max_norm=math.nan).refused(name, "max_norm")


def test_c_finish_refuses():
    c = Call([4096], [8], [F])
    c.args.partials = None
    c.refused("luma_grad_finish", "partials")
    Call([4096], [8], [F], norm_kind=0).refused("luma_grad_finish", "norm kind")
    Call([4096], [8], [F], coef=64, max_norm=-0.5).refused("luma_grad_finish", "max_norm")
    Call([4096], [8], [F]).refused("luma_grad_clip", "coef")


@pytest.mark.parametrize("name", ["luma_grad_scale", "luma_grad_clip"])
@pytest.mark.parametrize("ptrs,numels,codes", [
    ([4096, 4096], [8, 8], [F, F]),          # the same tensor twice
    ([4096, 4112], [8, 8], [F, F]),          # views that overlap
    ([8192, 4096, 8200], [8, 8, 2], [F, F, B]),  # found after sorting
    ([4096, 4124], [8, 8], [F, F]),          # by one element
])
def test_c_in_place_refuses_overlap(name, ptrs, numels, codes):
    Call(ptrs, numels, codes, coef=64).refused(name, "overlap")


@pytest.mark.parametrize("grads,codes,accs,acc_codes,words", [
    ([4096, 8192], [F, F], [65536, 65536], [F, F], "overlap"),      # an accumulator twice
    ([65552], [F], [65536], [F], "gradient 0 overlaps"),            # shifted by four elements
    ([65536], [B], [65536], [F], "gradient 0 overlaps"),            # the same address, another type
    ([4096, 65536], [F, F], [65536, 131072], [F, F], "gradient 1 overlaps accumulator 0"),
    ([4096, 8192], [F, F], [65536, 131072], [F, H], "float16"),
])
def test_c_accumulate_refuses_overlap(grads, codes, accs, acc_codes, words):
    n = len(grads)
    Call(grads, [8] * n, codes, accs, acc_codes).refused("luma_grad_accumulate", words)


@pytest.mark.parametrize("name", ["luma_grad_scale", "luma_grad_accumulate"])
@pytest.mark.parametrize("at", [65536, 65536 + 28, 65536 - 2])
def test_c_refuses_a_factor_inside_what_is_written(name, at):
    """Every CTA reads it while others write."""
    Call([65536 if name == "luma_grad_scale" else 4096], [8], [F], [65536], [F],
         scale=at).refused(name, "factor")


# -- Python --------------------------------------------------------------------

OPS = [lambda g: luma_b200.grad_norm(g), lambda g: luma_b200.clip_coef(g, 1.0),
       lambda g: luma_b200.clip_grads_(g, 1.0), lambda g: luma_b200.scale_grads_(g, 0.5),
       lambda g: luma_b200.accumulate_grads_(g, g)]


@pytest.mark.parametrize("op", OPS)
def test_refuses_what_is_no_dense_cuda_tensor(op):
    with pytest.raises(RuntimeError, match="requires CUDA"):
        op([torch.zeros(4)])
    with pytest.raises(TypeError, match="NoneType"):
        op([None])
    with pytest.raises(TypeError, match="float"):
        op([1.0])
    with pytest.raises(TypeError, match="must be tensors"):
        op(None)
    with pytest.raises(RuntimeError, match="sparse"):
        op([torch.zeros(4, 4).to_sparse()])
    with pytest.raises(ValueError, match="float64"):
        op([torch.zeros(4, dtype=torch.float64)])
    with pytest.raises(ValueError, match="int16"):
        op([torch.zeros(4, dtype=torch.int16)])


def test_refuses_bad_numbers():
    for bad in (0.0, 3.0, -1.0, math.nan, -math.inf):
        with pytest.raises(ValueError, match="norm_type"):
            luma_b200.grad_norm([], bad)
    for bad in (-1.0, math.nan, -math.inf):
        with pytest.raises(ValueError, match="max_norm"):
            luma_b200.clip_coef([], bad)
        with pytest.raises(ValueError, match="max_norm"):
            luma_b200.clip_grads_([], bad)
        with pytest.raises(ValueError, match="max_norm"):
            luma_b200.accumulate_grads_([], [], max_norm=bad)
    with pytest.raises(ValueError, match="as long as"):
        luma_b200.accumulate_grads_([], [_Fake()])


class _Fake(torch.Tensor):
    """Passes for an empty CUDA tensor in the checks."""

    @staticmethod
    def __new__(cls):
        return torch.Tensor._make_wrapper_subclass(cls, (0,), dtype=torch.float32, device="cuda")

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError(func)


def test_empty_lists():
    assert luma_b200.grad_norm([]) == 0.0
    norm, norms = luma_b200.grad_norm([], per_tensor=True)
    assert norm == 0.0 and norms.shape == (0,)
    norm, coef = luma_b200.clip_coef([], 1.0)
    assert norm == 0.0 and coef == 1.0
    assert luma_b200.clip_grads_([], 1.0) == 0.0
    assert luma_b200.scale_grads_([], 0.5) is None
    assert luma_b200.accumulate_grads_([], []) is None
    assert luma_b200.accumulate_grads_([], [], norm_type=2.0) == 0.0
    assert luma_b200.accumulate_grads_([], [], max_norm=1.0) == (0.0, 1.0)


def test_dense_layouts():
    _dense = _ops().dense
    x = torch.zeros(4, 6, 8)
    assert _dense(x.transpose(0, 2)) and _dense(x.permute(1, 2, 0))
    assert _dense(torch.zeros(2, 3, 4, 5).to(memory_format=torch.channels_last))
    assert _dense(torch.zeros(0, 3).t()) and _dense(torch.zeros(1).expand(1))
    assert not _dense(x[:, ::2]) and not _dense(x[:, :3]) and not _dense(torch.zeros(1).expand(5))
    assert not _dense(torch.zeros(3, 1).expand(3, 4)) and not _dense(torch.zeros(8).as_strided((4, 2), (1, 1)))


# -- over ranks ----------------------------------------------------------------

class FakeOps:
    """The list module in elementary operations on CPU tensors."""

    @staticmethod
    def power(grads, kind):
        x = torch.cat([torch.zeros(1, dtype=torch.float64), *(g.double().reshape(-1) for g in grads)])
        x = x.abs()
        return {1: x.sum(), 2: (x * x).sum(), 3: x.max()}[kind].reshape(1)

    @staticmethod
    def finish(power, kind, max_norm, inv_scale, found_inf):
        norm = (power.sqrt() if kind == 2 else power)[0]
        if found_inf is not None and not torch.isfinite(norm):
            found_inf.fill_(1.0)
        coef = None if max_norm is None else torch.clamp(max_norm / (norm + 1e-6), max=1.0)
        return norm, coef

    @staticmethod
    def scale(grads, coef):
        for g in grads:
            g.mul_(coef)


def _rank(rank, store, ok):
    import torch.distributed as dist
    from luma_b200 import grads as module
    module._ext = FakeOps
    dist.init_process_group("gloo", init_method=f"file://{store}", rank=rank, world_size=2)
    pg = dist.group.WORLD
    # rank 1 holds no shards of the second list
    mine = [torch.full((4 + rank,), 2.0 + rank)]
    none = mine if rank == 0 else []
    assert module.grad_norm(mine, process_group=pg) == math.sqrt(4 * 4 + 5 * 9)
    assert module.grad_norm(mine, 1.0, process_group=pg) == 23.0
    assert module.grad_norm(mine, math.inf, process_group=pg) == 3.0
    assert module.grad_norm(none, process_group=pg) == 4.0
    norm, coef = module.clip_coef(none, 2.0, process_group=pg)
    assert norm == 4.0 and abs(coef - 0.5) < 1e-6
    norm = module.clip_grads_(none, 2.0, process_group=pg)
    assert norm == 4.0 and all(abs(g[0] - 1) < 1e-6 for g in none)
    # a NaN on one rank is not lost, and raises the flag on both
    mine[0][0] = math.nan if rank else 1.0
    flag = torch.zeros(1)
    norm, _ = module.clip_coef(mine, 1.0, math.inf, found_inf=flag, process_group=pg)
    assert norm == math.inf and flag == 1.0
    assert math.isnan(module.grad_norm(mine, process_group=pg))
    for fn in (module.grad_norm, lambda g, **kw: module.clip_coef(g, 1.0, **kw)):
        try:
            fn(mine, process_group=pg, error_if_nonfinite=True)
        except RuntimeError as e:
            assert "not finite" in str(e)
        else:
            raise AssertionError("no error")
    dist.destroy_process_group()
    ok[rank] = 1


def test_norm_over_two_ranks(tmp_path):
    ctx = torch.multiprocessing.get_context("spawn")
    ok = ctx.Array("i", 2)
    ranks = [ctx.Process(target=_rank, args=(r, tmp_path / "store", ok)) for r in range(2)]
    for p in ranks:
        p.start()
    for p in ranks:
        p.join(120)
        assert p.exitcode == 0
    assert list(ok) == [1, 1]
    with pytest.raises(ValueError, match="whole tensors"):
        luma_b200.grad_norm([], per_tensor=True, process_group=object())


# -- GradScaler ----------------------------------------------------------------

class FakeLUMA(torch.optim.Optimizer):
    def __init__(self, params):
        super().__init__(params, {})
        self.calls = []

    def step(self, closure=None, *, grad_scale=None, found_inf=None):
        self.calls.append((grad_scale, found_inf))


def _scaler(**kw):
    s = torch.amp.GradScaler("cpu", **kw)
    s.scale(torch.ones(()))
    return s


def _optimizer():
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.ones(4)
    return FakeLUMA([p])


@pytest.fixture
def fake_coef(monkeypatch):
    """clip_coef in elementary operations: there is no GPU here."""
    def coef(grads, max_norm, norm_type=2.0, *, inv_scale=None, found_inf=None):
        inv = 1.0 if inv_scale is None else float(inv_scale)
        norm = torch.linalg.vector_norm(torch.cat([g.reshape(-1) for g in grads]).double()) * inv
        if found_inf is not None and not torch.isfinite(norm):
            found_inf.fill_(1.0)
        return norm.float(), (inv * torch.clamp(max_norm / (norm + 1e-6), max=1.0)).float()
    monkeypatch.setattr(amp, "clip_coef", coef)


def test_clip_step_passes_one_coefficient_and_the_flag(fake_coef):
    opt, scaler = _optimizer(), _scaler(init_scale=4.0)
    norm = amp.clip_step(scaler, opt, 0.125)
    (gs, fi), = opt.calls
    assert norm == 0.5 and abs(gs.item() - 0.25 * 0.125 / (0.5 + 1e-6)) < 1e-8 and fi == 0.0
    st = scaler._per_optimizer_states[id(opt)]
    assert st["stage"] is OptState.STEPPED and list(st["found_inf_per_device"].values()) == [fi]
    with pytest.raises(RuntimeError, match="already been called"):
        amp.clip_step(scaler, opt, 0.125)
    scaler.update()
    assert scaler.get_scale() == 4.0


def test_clip_step_skips_and_backs_off(fake_coef):
    opt, scaler = _optimizer(), _scaler(init_scale=4.0)
    opt.param_groups[0]["params"][0].grad[1] = math.inf
    assert amp.clip_step(scaler, opt, 1.0) == math.inf
    assert opt.calls[0][1] == 1.0
    scaler.update()
    assert scaler.get_scale() == 2.0


def test_clip_step_of_unscaled_grads_and_disabled_scaler(fake_coef):
    opt, scaler = _optimizer(), _scaler(init_scale=4.0)
    scaler.unscale_(opt)
    assert amp.clip_step(scaler, opt, 0.125) == 0.5
    (gs, fi), = opt.calls
    assert abs(gs.item() - 0.25) < 1e-6 and fi is None
    opt = _optimizer()
    assert amp.clip_step(torch.amp.GradScaler("cpu", enabled=False), opt, 1.0) == 2.0
    (gs, fi), = opt.calls
    assert abs(gs.item() - 0.5) < 1e-6 and fi is None


def test_clip_step_refuses_what_scaler_step_refuses(fake_coef):
    opt, scaler = _optimizer(), _scaler()
    with pytest.raises(RuntimeError, match="Closure"):
        amp.clip_step(scaler, opt, 1.0, closure=lambda: None)
    p = opt.param_groups[0]["params"][0]
    p.grad_dtype = None
    p.grad = torch.ones(4, dtype=torch.float16)
    with pytest.raises(ValueError, match="FP16"):
        amp.clip_step(scaler, opt, 1.0)
