"""Gradient operators on the GPU over every path that a list can take: one
cluster (up to 128 tensors and 512 KB), a norm and a finishing launch, and
several tables (more than 1,280 tensors).  Plain implementations in 64 bits;
tolerances as in test_gpu_grads.py, where they are derived."""

import math

import pytest
import torch

from luma_b200 import LUMA, accumulate_grads_, amp, clip_coef, clip_grads_, grad_norm, scale_grads_
from test_gpu_grads import (BF16, F16, F32, INF, NAN, NORM_TOL, TYPES, U, exact_coef, exact_norm, make,
                            near, plain_scale)

pytestmark = pytest.mark.gpu

PATHS = {
    "cluster": [5, 70_000, 9],
    "launches": [5, 1_000_003, 9],
    "tables": [3, 0, 17, 1] * 330 + [300_001] + [2] * 100,
}
# (tensor, element): the first, inner and last tile, and those of the first,
# inner and last table
SPOTS = {
    "cluster": [(0, 0), (1, 0), (1, 33_333), (1, 69_999), (2, 8)],
    "launches": [(0, 4), (1, 0), (1, 500_000), (1, 1_000_002), (2, 8)],
    "tables": [(0, 0), (1278, 16), (1282, 16), (1320, 0), (1320, 150_000), (1320, 300_000), (1420, 1)],
}
path = pytest.mark.parametrize("path", PATHS)
every_norm = pytest.mark.parametrize("p", [1.0, 2.0, INF])
every_type = pytest.mark.parametrize("dtype", TYPES)


@path
@every_norm
@every_type
def test_nonfinite(path, dtype, p):
    _, ts = make(PATHS[path], dtype, offset=1, seed=3)
    clean = [exact_norm([t], p) for t in ts]
    for k, (i, at) in enumerate(SPOTS[path]):
        bad = (INF, -INF, NAN)[k % 3]
        want = NAN if math.isnan(bad) else INF
        kept = ts[i][at].clone()
        ts[i][at] = bad
        norm, norms = grad_norm(ts, p, per_tensor=True)
        near(norm, want, 0)
        for j, got in enumerate(norms.tolist()):
            near(got, want if j == i else clean[j], 0 if j == i else NORM_TOL[p])
        near(grad_norm(ts, p), want, 0)
        flag = torch.zeros(1, device="cuda")
        norm, coef = clip_coef(ts, 1.0, p, found_inf=flag)
        near(norm, want, 0)
        near(coef, NAN if math.isnan(bad) else 0.0, 0)
        assert flag == 1.0
        acc = [torch.zeros_like(t, dtype=F32) for t in ts]
        near(accumulate_grads_(acc, ts, overwrite=True, norm_type=p), want, 0)
        ts[i][at] = kept
    flag = torch.zeros(1, device="cuda")
    near(clip_coef(ts, 1.0, p, found_inf=flag)[0], exact_norm(ts, p), NORM_TOL[p])
    assert flag == 0.0


@path
@every_norm
@every_type
def test_ends_of_the_range(path, dtype, p):
    """Squares that float32 cannot hold, everywhere and in one place."""
    fin = torch.finfo(dtype)
    flat, ts = make(PATHS[path], dtype)
    for value in (fin.max, fin.tiny, fin.tiny / 4, 3e-23 if dtype != F16 else 6e-8):
        flat.fill_(value)
        want = exact_norm(ts, p)
        norm, norms = grad_norm(ts, p, per_tensor=True)
        for got in (norm, grad_norm(ts, p)):
            near(got, INF if want > torch.finfo(F32).max else want, NORM_TOL[p])
        first = exact_norm(ts[:1], p)
        near(norms[0], INF if first > torch.finfo(F32).max else first, NORM_TOL[p])
    for big, small in ((fin.max / 2, 1.0), (1.0, fin.tiny)):
        for i, at in SPOTS[path]:
            flat.fill_(small)
            ts[i][at] = big
            near(grad_norm(ts, p), exact_norm(ts, p), NORM_TOL[p])


@path
@every_norm
@every_type
def test_coefficients_and_clipping(path, dtype, p):
    for offset, max_norm in ((0, 0.25), (1, 0.25), (1, 1e9), (0, 0.0)):
        flat, ts = make(PATHS[path], dtype, offset=offset, std=0.3, seed=offset)
        want = exact_norm(ts, p)
        inv = torch.full((1,), 2.0 ** -9, device="cuda")
        norm, coef = clip_coef(ts, max_norm, p, inv_scale=inv)
        near(norm, want * 2.0 ** -9, NORM_TOL[p] + U)
        near(coef, exact_coef(want * 2.0 ** -9, max_norm, 2.0 ** -9), NORM_TOL[p] + U)
        norm, coef = clip_coef(ts, max_norm, p)
        near(norm, want, NORM_TOL[p])
        near(coef, exact_coef(want, max_norm), NORM_TOL[p] + U)
        scaled = plain_scale(ts, coef)
        got = clip_grads_(ts, max_norm, p)
        assert torch.equal(got, norm)
        assert all(torch.equal(a, b) for a, b in zip(ts, scaled))


@path
def test_streams(path):
    """Calls queued on several streams at once, each with its own workspace."""
    lists = [make(PATHS[path], BF16, seed=k, std=0.1 * (k + 1))[1] for k in range(4)]
    want = [exact_norm(ts, 2.0) for ts in lists]
    each = [[exact_norm([t], 2.0) for t in ts] for ts in lists]
    streams = [torch.cuda.Stream() for _ in lists]
    accs = [[torch.zeros_like(t, dtype=F32) for t in ts] for ts in lists]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for st, ts, acc in zip(streams, lists, accs):
            with torch.cuda.stream(st):
                got.append((clip_coef(ts, 0.5), grad_norm(ts, per_tensor=True),
                            accumulate_grads_(acc, ts, overwrite=True, norm_type=2.0)))
    torch.cuda.synchronize()
    for k, ((norm, coef), (total, norms), summed) in enumerate(got):
        for v in (norm, total, summed):
            near(v, want[k % 4], NORM_TOL[2.0])
        near(coef, exact_coef(want[k % 4], 0.5), NORM_TOL[2.0] + U)
        for v, w in zip(norms.tolist(), each[k % 4]):
            near(v, w, NORM_TOL[2.0])


@path
def test_what_is_only_read_keeps_its_version(path):
    _, gs = make(PATHS[path], BF16)
    accs = [torch.zeros_like(g, dtype=F32) for g in gs]
    before = [g._version for g in gs], [a._version for a in accs]
    grad_norm(gs, per_tensor=True)
    clip_coef(gs, 1.0)
    accumulate_grads_(accs, gs, 0.5, max_norm=1.0)
    assert [g._version for g in gs] == before[0]
    assert all(a._version > v for a, v in zip(accs, before[1]))
    scale_grads_(gs, 0.5)
    assert all(g._version > v for g, v in zip(gs, before[0]))


@pytest.mark.parametrize("long", [40_000, 300_000], ids=["cluster", "launches"])
def test_clip_step_against_its_parts(long):
    """scaler.unscale_, a norm and a coefficient in 64 bits, scaling in place and
    scaler.step, one after the other.  Gradients are integers up to 8 times
    2^-10, so that their squares' sums are exact and both sides round the same
    coefficient; the loss scale is a power of two.  Equal bits."""
    shapes = [(65, 33), (1000,), (long,), (7,), (300, 100)]
    gen = torch.Generator(device="cuda").manual_seed(5)
    init = [torch.randn(s, device="cuda", generator=gen) * 0.02 for s in shapes]
    pa, pb = ([torch.nn.Parameter(t.clone()) for t in init] for _ in range(2))
    oa, ob = LUMA(pa, lr=1e-3), LUMA(pb, lr=1e-3)
    ob._base_seed = oa._base_seed
    sa, sb = (torch.amp.GradScaler("cuda", init_scale=2.0 ** 12, growth_interval=3) for _ in range(2))
    for it in range(7):
        max_norm = 0.25 if it % 3 else 1e9
        scale = float(sa.scale(torch.ones((), device="cuda")))
        assert float(sb.scale(torch.ones((), device="cuda"))) == scale
        raw = [torch.randint(-8, 9, s, device="cuda", generator=gen) * 2.0 ** -10 for s in shapes]
        if it == 4:
            raw[2][123] = INF
        for ps in (pa, pb):
            for p, g in zip(ps, raw):
                p.grad = g * scale
        norm = amp.clip_step(sa, oa, max_norm)
        sb.unscale_(ob)
        want = exact_norm([p.grad for p in pb], 2.0)
        if math.isfinite(want):
            assert float(norm) == float(torch.tensor(want, dtype=torch.float64).float())
        else:
            assert norm == INF
        coef = min(1.0, max_norm / (want + 1e-6))
        for p in pb:
            p.grad = plain_scale([p.grad], coef)[0]
        sb.step(ob)
        sa.update(), sb.update()
        assert sa.get_scale() == sb.get_scale()
        assert all(torch.equal(a, b) for a, b in zip(pa, pb)), it
    assert oa.state_dict()["state"][0]["step"] == 6
