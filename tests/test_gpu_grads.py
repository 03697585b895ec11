"""Gradient operators on the GPU against plain implementations in 64 bits.

Tolerances.  A rounding is off by at most u = 2^-24 (float32), 2^-8 (bf16) or
2^-11 (fp16) of the value.  Sums of non-negative terms: elements are squared
and added in float32 in chains of at most 16, joined by at most 4 more
additions, and in float64 from there on, so S is off by at most 20 u (each
element's term passes at most 20 roundings; float64's are below 2^-40 of it).
The root halves that and the result is rounded once: NORM2 = 11 u, NORM1 =
21 u; a maximum is exact.  The coefficient c * min(1, max_norm / (r + 1e-6)) is
taken in float64 from r before its rounding: COEF2 = NORM2, likewise.
Scaling is one float32 product and one rounding to the type, and the plain
form's is the same: equal bits.  acc + c * x rounds the product (off by
2^-24 |c x|), the sum (2^-24 of it, itself off from the result by the former:
2^-24 (|result| + 2^-24 |c x|)) and the value stored (the type's u of that): with
U = 2^-24, at most U |c x| + (u + U + u U) (|result| + U |c x|); a subnormal
value by half the smallest number there is, once for each rounding.
"""

import math

import numpy as np
import pytest
import torch

import luma_b200
from luma_b200 import LUMA, accumulate_grads_, clip_coef, clip_grads_, grad_norm, scale_grads_

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
NORM_TOL = {1.0: 21 * U, 2.0: 11 * U, math.inf: 0.0}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
F32, BF16, F16 = TYPES
INF, NAN = math.inf, math.nan


def make(sizes, dtype, *, offset=0, std=1e-2, seed=0, gap=0):
    """Views of one buffer: tensor i starts `gap` elements behind the one before."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    total = offset + sum(sizes) + gap * len(sizes)
    flat = torch.empty(total, dtype=torch.float32, device="cuda").normal_(0, std, generator=gen)
    flat = flat.to(dtype)
    out, at = [], offset
    for n in sizes:
        out.append(flat[at:at + n])
        at += n + gap
    return flat, out


def exact_power(t, p):
    x = t.detach().double().abs().reshape(-1)
    if x.numel() == 0:
        return 0.0
    return float(x.max()) if p == INF else float((x ** p).sum())


def exact_norm(ts, p):
    powers = [exact_power(t, p) for t in ts]
    if p == INF:
        return max(powers, default=0.0)
    return math.sqrt(math.fsum(powers)) if p == 2.0 else math.fsum(powers)


def near(got, want, tol):
    got, want = float(got), float(want)
    if math.isnan(want) or math.isinf(want):
        assert (math.isnan(got) and math.isnan(want)) or got == want, (got, want)
    else:
        assert abs(got - want) <= tol * abs(want) + 2.0 ** -150, (got, want, abs(got / want - 1) / U)


SIZES = {
    "one": [1], "few": [31, 33, 1, 2, 3], "empty between": [5, 0, 1024, 0, 0, 7, 0],
    "tile ends": [16383, 16384, 16385, 65536, 32768 + 1], "long": [1_000_003],
    "many": list(range(1, 300)), "more than a table": [3, 0, 17, 1] * 700, "none": [0, 0],
    # around the ends of what one cluster takes: 128 tensors, 512 KB
    "128 tensors": [1, 2, 40, 700] * 32, "129 tensors": [5] * 129,
    "uneven in a cluster": [1, 100_000, 0, 3] + [17] * 60 + [20_000, 0, 1],
    "512 KB of fp32": [65_536, 0, 65_536], "more than 512 KB": [131_073, 131_072],
}


@pytest.mark.parametrize("p", [1.0, 2.0, INF])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", SIZES.values(), ids=SIZES.keys())
def test_norms(sizes, dtype, p):
    for offset, gap in ((0, 0), (1, 0), (3, 5)):
        _, ts = make(sizes, dtype, offset=offset, gap=gap, seed=len(sizes) + offset)
        norm, norms = grad_norm(ts, p, per_tensor=True)
        assert norm.dtype == norms.dtype == torch.float32 and norm.shape == ()
        assert norm.device == ts[0].device and norms.shape == (len(ts),)
        near(norm, exact_norm(ts, p), NORM_TOL[p])
        for got, t in zip(norms.tolist(), ts):
            near(got, exact_norm([t], p), NORM_TOL[p])
        assert torch.equal(grad_norm(ts, p), norm)  # the same bits again


@pytest.mark.parametrize("p", [1.0, 2.0, INF])
def test_mixed_types_and_layouts(p):
    gen = torch.Generator(device="cuda").manual_seed(3)
    a = torch.randn(37, 65, device="cuda", generator=gen)
    b = torch.randn(8, 3, 5, 7, device="cuda", generator=gen).to(BF16)
    ts = [a.t(), b.to(memory_format=torch.channels_last), a.to(F16)[3:], torch.nn.Parameter(a * 2),
          b.permute(2, 0, 3, 1), torch.tensor(3.5, device="cuda")]
    near(grad_norm(ts, p), exact_norm(ts, p), NORM_TOL[p])
    near(grad_norm(t for t in ts), exact_norm(ts, 2.0), NORM_TOL[2.0])  # any iterable
    near(grad_norm(a), exact_norm([a], 2.0), NORM_TOL[2.0])  # a tensor alone
    near(grad_norm([a, a], p), exact_norm([a, a], p), NORM_TOL[p])  # twice counts twice


@pytest.mark.parametrize("p", [1.0, 2.0, INF])
@pytest.mark.parametrize("dtype", TYPES)
def test_norm_keeps_its_precision_at_the_ends_of_the_range(dtype, p):
    """Squares that float32 cannot hold; a result that it cannot hold is inf."""
    fin = torch.finfo(dtype)
    for value in (fin.max, fin.max / 4, fin.tiny, fin.tiny / 4, 1e-30 if dtype != F16 else 1e-7,
                  1e18 if dtype != F16 else 1e4, 3e-23 if dtype != F16 else 6e-8):
        ts = [torch.full((n,), value, dtype=dtype, device="cuda") for n in (1, 5, 70_001)]
        want = exact_norm(ts, p)
        got = grad_norm(ts, p)
        if want > torch.finfo(F32).max:
            assert got == INF
        else:
            near(got, want, NORM_TOL[p])
    # one large element among small ones and the other way round
    for big, small in ((fin.max / 2, 1.0), (1.0, fin.tiny), (fin.max / 2, fin.tiny)):
        t = torch.full((40_000,), small, dtype=dtype, device="cuda")
        t[12_345] = big
        near(grad_norm([t], p), exact_norm([t], p), NORM_TOL[p])
    assert grad_norm([torch.zeros(100_000, dtype=dtype, device="cuda")], p) == 0.0
    minus = torch.full((1000,), -0.0, dtype=dtype, device="cuda")
    assert math.copysign(1.0, float(grad_norm([minus], p))) == 1.0


@pytest.mark.parametrize("p", [1.0, 2.0, INF])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [INF, -INF, NAN])
def test_nonfinite_elements(bad, dtype, p):
    for at in (0, 1, 4097, 69_998, 69_999):
        _, ts = make([5, 70_000, 9], dtype, offset=1, seed=at)
        ts[1][at] = bad
        want = NAN if math.isnan(bad) else INF
        norm, norms = grad_norm(ts, p, per_tensor=True)
        near(norm, want, 0)
        near(norms[1], want, 0)
        near(norms[0], exact_norm(ts[:1], p), NORM_TOL[p])
        flag = torch.zeros(1, device="cuda")
        norm, coef = clip_coef(ts, 1.0, p, found_inf=flag)
        near(norm, want, 0)
        near(coef, NAN if math.isnan(bad) else 0.0, 0)
        assert flag == 1.0
        for fn in (grad_norm, lambda g, p, **kw: clip_coef(g, 1.0, p, **kw),
                   lambda g, p, **kw: clip_grads_(g, 1.0, p, **kw)):
            before = ts[1].clone()
            with pytest.raises(RuntimeError, match="not finite"):
                fn(ts, p, error_if_nonfinite=True)
            assert torch.equal(before.nan_to_num(), ts[1].nan_to_num())
    # an inf and a NaN together are a NaN
    t = torch.ones(50_000, dtype=dtype, device="cuda")
    t[7], t[40_000] = INF, NAN
    near(grad_norm([t], p), NAN, 0)


def test_norm_beyond_32_bit_offsets():
    n = (1 << 31) + 4099
    t = torch.zeros(n, dtype=BF16, device="cuda")
    t[0], t[1 << 31], t[n - 1] = 3.0, 4.0, 12.0
    assert grad_norm([t]) == 13.0
    assert grad_norm([t[1:]], INF) == 12.0
    scale_grads_([t[1:]], 0.5)
    assert t[0] == 3.0 and t[1 << 31] == 2.0 and t[n - 1] == 6.0
    acc = torch.zeros(n, dtype=BF16, device="cuda")
    norm = accumulate_grads_([acc], [t], 2.0, norm_type=2.0)
    assert acc[1 << 31] == 4.0 and acc[n - 1] == 12.0 and norm == math.sqrt(36 + 16 + 144)


# -- coefficients ----------------------------------------------------------------

def exact_coef(norm, max_norm, inv=1.0):
    return inv * min(1.0, max_norm / (norm + 1e-6))


@pytest.mark.parametrize("p", [1.0, 2.0, INF])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("max_norm", [0.0, 0.37, 1e9, INF])
def test_coefficients(max_norm, dtype, p):
    _, ts = make([3, 70_001, 1000], dtype, std=0.3)
    want = exact_norm(ts, p)
    norm, coef = clip_coef(ts, max_norm, p)
    near(norm, want, NORM_TOL[p])
    near(coef, exact_coef(want, max_norm), NORM_TOL[p] + U)
    if max_norm > 1e8:
        assert coef == 1.0
    for inv in (2.0 ** -16, 1.0 / 3.0, 0.0):
        inv_t = torch.tensor([inv], device="cuda")
        inv = float(inv_t)
        flag = torch.zeros((), device="cuda")
        norm, coef = clip_coef(ts, max_norm, p, inv_scale=inv_t, found_inf=flag)
        near(norm, want * inv, NORM_TOL[p] + U)
        near(coef, exact_coef(want * inv, max_norm, inv), NORM_TOL[p] + U)
        assert flag == 0.0
    flag = torch.ones((), device="cuda")
    clip_coef(ts, max_norm, p, found_inf=flag)
    assert flag == 1.0  # never cleared


def test_zero_norm_and_overflowing_norm():
    z = torch.zeros(10, device="cuda")
    norm, coef = clip_coef([z], 1.0)
    assert norm == 0.0 and coef == 1.0
    norm, coef = clip_coef([z, z[:0]], 0.0)
    assert norm == 0.0 and coef == 0.0
    big = torch.full((1 << 20,), 3e38, device="cuda")
    flag = torch.zeros(1, device="cuda")
    norm, coef = clip_coef([big], 1e30, found_inf=flag)
    assert norm == INF and flag == 0.0  # no element is inf: the step is not skipped
    near(coef, 1e30 / exact_norm([big], 2.0), NORM_TOL[2.0] + U)


# -- in place --------------------------------------------------------------------

def plain_scale(ts, c):
    return [(t.float() * torch.as_tensor(c, dtype=F32, device="cuda")).to(t.dtype) for t in ts]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [v for k, v in SIZES.items()], ids=SIZES.keys())
def test_scale_in_place(sizes, dtype):
    for offset, gap in ((0, 0), (1, 0), (3, 5)):
        flat, ts = make(sizes, dtype, offset=offset, gap=gap, std=1.0)
        for coef in (0.3, torch.tensor([0.7], device="cuda"), 1.0, torch.tensor(1.0, device="cuda"),
                     torch.tensor(0.5, dtype=BF16, device="cuda")):
            before = flat.clone()
            want = plain_scale(ts, coef.float() if isinstance(coef, torch.Tensor) else coef)
            scale_grads_(ts, coef)
            assert all(torch.equal(a, b) for a, b in zip(ts, want))
            # what lies before, between and behind the tensors stays as it was
            keep = torch.ones_like(flat, dtype=torch.bool)
            for t in ts:
                at = t.storage_offset()
                keep[at:at + t.numel()] = False
            assert torch.equal(flat[keep], before[keep])


@pytest.mark.parametrize("dtype", TYPES)
def test_scale_special_values(dtype):
    fin = torch.finfo(dtype)
    v = torch.tensor([0.0, -0.0, INF, -INF, NAN, fin.max, fin.tiny, fin.tiny / 2, -1.0] * 7001,
                     dtype=dtype, device="cuda")
    for c in (0.5, 0.0, -2.0, 1e-3, 3e38, INF, NAN):
        t = v.clone()
        scale_grads_([t[1:]], c)
        want = torch.cat([v[:1], plain_scale([v[1:]], c)[0]])
        assert torch.equal(t.isnan(), want.isnan())
        assert torch.equal(t.nan_to_num(7.0).view(torch.int16), want.nan_to_num(7.0).view(torch.int16))


@pytest.mark.parametrize("p", [1.0, 2.0, INF])
@pytest.mark.parametrize("dtype", TYPES)
def test_clip_in_place(dtype, p):
    sizes = [3, 70_001, 0, 1000, 16_384]
    for offset in (0, 1):
        for max_norm in (0.25, 1e9, 0.0):
            flat, ts = make(sizes, dtype, std=0.3, offset=offset)
            norm0, coef = clip_coef(ts, max_norm, p)
            want = plain_scale(ts, coef)
            versions = [t._version for t in ts]
            norm = clip_grads_(ts, max_norm, p)
            assert torch.equal(norm, norm0)
            assert all(torch.equal(a, b) for a, b in zip(ts, want))
            assert all(t._version > v for t, v in zip(ts, versions))
            assert torch.equal(clip_grads_(plain := [t.clone() for t in ts], 1e30,
                                           error_if_nonfinite=True), grad_norm(ts))
            assert all(torch.equal(a, b) for a, b in zip(ts, plain))


def test_clip_against_what_users_call():
    """The float32 result of PyTorch's own clipping, to the rounding of its norm
    (float32 throughout: a few hundred u) and of the product."""
    shapes = [(33, 65), (1000,), (7, 3, 5)]
    pa = [torch.nn.Parameter(torch.zeros(s, device="cuda")) for s in shapes]
    gen = torch.Generator(device="cuda").manual_seed(1)
    for p in pa:
        p.grad = torch.randn(p.shape, device="cuda", generator=gen)
    ours = [p.grad.clone() for p in pa]
    norm = torch.nn.utils.clip_grad_norm_(pa, 0.5)
    got = clip_grads_(ours, 0.5)
    assert abs(float(norm) / float(got) - 1) < 1e-5
    for p, g in zip(pa, ours):
        torch.testing.assert_close(p.grad, g, rtol=1e-5, atol=0)


# -- accumulation ----------------------------------------------------------------

def check_accumulated(acc, before, g, c, overwrite):
    """acc against c * g (+ before) in 64 bits, where c * g is exact."""
    product = g.double() * c
    want = product + (0.0 if overwrite else before.double())
    u = torch.finfo(acc.dtype).eps / 2
    tol = U * product.abs() + (want.abs() + U * product.abs()) * (u + U + u * U) + 2.0 ** -149
    if acc.dtype != F32:
        tol = tol + 2.0 ** -134  # half the smallest bf16 there is
    assert bool(((acc.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("acc_dtype", [F32, BF16])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [v for k, v in SIZES.items()], ids=SIZES.keys())
def test_accumulate(sizes, dtype, acc_dtype):
    for offset, acc_offset, gap in ((0, 0, 0), (1, 0, 0), (0, 1, 0), (3, 3, 5), (2, 6, 1)):
        _, gs = make(sizes, dtype, offset=offset, gap=gap, seed=5)
        flat, accs = make(sizes, acc_dtype, offset=acc_offset, gap=gap, seed=6)
        keep = torch.ones_like(flat, dtype=torch.bool)
        for t in accs:
            at = t.storage_offset()
            keep[at:at + t.numel()] = False
        outside = flat[keep].clone()
        for c, overwrite, p in ((1.0, True, None), (0.25, False, 2.0), (1 / 3, False, INF),
                                (-2.0, True, 1.0)):
            before = [t.clone() for t in accs]
            scale = c if overwrite else torch.tensor([c], device="cuda")
            norm = accumulate_grads_(accs, gs, scale, overwrite=overwrite, norm_type=p)
            for a, b, g in zip(accs, before, gs):
                check_accumulated(a, b, g, float(torch.tensor(c)), overwrite)
            if p is None:
                assert norm is None
            else:
                near(norm, exact_norm(accs, p), NORM_TOL[p])
        assert torch.equal(flat[keep], outside)


def test_accumulate_coefficient_types_and_layouts():
    gen = torch.Generator(device="cuda").manual_seed(3)
    gs = [torch.randn(37, 65, device="cuda", generator=gen).to(BF16).t(),
          torch.randn(8, 3, 5, 7, device="cuda", generator=gen).to(memory_format=torch.channels_last),
          torch.randn(100, device="cuda", generator=gen).to(F16), torch.randn((), device="cuda")]
    accs = [torch.zeros_like(g, dtype=F32) for g in gs]
    accs[3] = accs[3].to(BF16)
    accumulate_grads_(accs, gs)
    norm, coef = accumulate_grads_(accs, gs, 0.5, max_norm=2.0)
    for a, g in zip(accs, gs):
        check_accumulated(a, g.to(a.dtype), g, 0.5, False)
    norm2, coef2 = clip_coef(accs, 2.0)
    near(norm, float(norm2), 2 * NORM_TOL[2.0])
    near(coef, float(coef2), 2 * NORM_TOL[2.0] + 2 * U)
    norm, coef = accumulate_grads_(accs, gs, 0.0, norm_type=INF, max_norm=1.0)
    assert norm == grad_norm(accs, INF) and torch.equal(coef, clip_coef(accs, 1.0, INF)[1])
    # onto itself: x + c x
    x = torch.randn(70_001, device="cuda", generator=gen)
    y = x.clone()
    accumulate_grads_([x], [x], 0.5)
    check_accumulated(x, y, y, 0.5, False)
    for t in (gs[2], accs[0]):
        before = t._version
        accumulate_grads_([accs[0]], [gs[0]])
    assert accs[0]._version > before


def test_accumulate_ties():
    """A third of a multiple of three is a short number again, and where the sum
    lies half-way between two bfloat16 values the even one is stored."""
    k = torch.arange(1, 128, device="cuda", dtype=torch.float32)
    g = (3 * k).to(BF16)[(3 * k) == (3 * k).to(BF16).float()]  # 3 k that bf16 holds
    third = g.double() / 3
    for start in (256.0, 512.0, 1024.0):
        acc = [torch.full(g.shape, start, dtype=BF16, device="cuda")]
        accumulate_grads_(acc, [g], 1 / 3)
        assert torch.equal(acc[0], (start + third).to(BF16))
        assert ((start + third) % (start / 128) == start / 256).any()  # ties are among them


def test_accumulate_nonfinite():
    _, gs = make([40_000], BF16)
    gs[0][7], gs[0][30_000] = INF, NAN
    acc = [torch.ones(40_000, device="cuda")]
    norm = accumulate_grads_(acc, gs, norm_type=2.0)
    assert math.isnan(float(norm)) and acc[0][7] == INF and acc[0][30_000].isnan()
    acc = [torch.full((40_000,), NAN, device="cuda")]
    gs[0][7] = gs[0][30_000] = 1.0
    norm = accumulate_grads_(acc, gs, overwrite=True, norm_type=INF)  # what acc held does not count
    assert norm == gs[0].abs().max().float()


# -- refusals that need CUDA tensors -----------------------------------------------

def test_refusals():
    x = torch.zeros(64, 64, device="cuda")
    for op in (grad_norm, lambda g: clip_coef(g, 1.0), lambda g: clip_grads_(g, 1.0),
               lambda g: scale_grads_(g, 0.5), lambda g: accumulate_grads_(g, g)):
        with pytest.raises(ValueError, match="dense"):
            op([x[:, :32]])
        with pytest.raises(ValueError, match="dense"):
            op([x[0, :1].expand(8)])
        with pytest.raises(RuntimeError, match="CUDA"):
            op([x, torch.zeros(3)])
    for op in (lambda g: clip_grads_(g, 1.0), lambda g: scale_grads_(g, 0.5),
               lambda g: accumulate_grads_(g, [t.clone() for t in g])):
        with pytest.raises(ValueError, match="overlap"):
            op([x, x])
        with pytest.raises(ValueError, match="overlap"):
            op([x[:10], x[9:]])
    v = torch.zeros(64, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        accumulate_grads_([v[:32]], [v[1:33]])
    with pytest.raises(ValueError, match="factor"):
        scale_grads_([v], v[3])
    with pytest.raises(ValueError, match="factor"):
        accumulate_grads_([v], [v.clone()], v[63:])
    with pytest.raises(ValueError, match="shape"):
        accumulate_grads_([v], [x])
    with pytest.raises(ValueError, match="order"):
        accumulate_grads_([x], [torch.zeros(64, 64, device="cuda").t()])
    with pytest.raises(ValueError, match="float16"):
        accumulate_grads_([v.half()], [v])
    with pytest.raises(ValueError, match="as long as"):
        accumulate_grads_([v, v.clone()], [v.clone()])
    with pytest.raises(ValueError, match="negated"):
        accumulate_grads_([v], [torch._neg_view(torch.ones(64, device="cuda"))])
    for bad in (torch.zeros(2, device="cuda"), torch.zeros(1), torch.zeros(1, dtype=BF16, device="cuda")):
        with pytest.raises(ValueError, match="found_inf"):
            clip_coef([v], 1.0, found_inf=bad)
        with pytest.raises(ValueError, match="inv_scale"):
            clip_coef([v], 1.0, inv_scale=bad)
    with pytest.raises(ValueError, match="coef"):
        scale_grads_([v], torch.zeros(2, device="cuda"))
    with pytest.raises(ValueError, match="scale"):
        accumulate_grads_([v], [v.clone()], torch.zeros(1, dtype=torch.int32, device="cuda"))


# -- streams and graphs --------------------------------------------------------------

def test_streams_share_nothing():
    """Calls queued on several streams at once each get their own result."""
    lists = [make([100_003, 17, 4096], BF16, seed=k, std=0.1 * (k + 1))[1] for k in range(4)]
    want = [exact_norm(ts, 2.0) for ts in lists]
    streams = [torch.cuda.Stream() for _ in lists]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for st, ts in zip(streams, lists):
            with torch.cuda.stream(st):
                got.append(clip_coef(ts, 0.5))
    torch.cuda.synchronize()
    for k, (norm, coef) in enumerate(got):
        near(norm, want[k % 4], NORM_TOL[2.0])
        near(coef, exact_coef(want[k % 4], 0.5), NORM_TOL[2.0] + U)


def test_two_captured_graphs_replayed_at_once():
    lists = [make([200_003, 17, 4096, 70_001], BF16, seed=k)[1] for k in range(2)]
    accs = [[torch.zeros(t.shape, device="cuda") for t in ts] for ts in lists]
    graphs, outs = [], []
    for ts, acc in zip(lists, accs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            accumulate_grads_(acc, ts, overwrite=True)
            norm = clip_grads_(acc, 0.5)
            n2, norms = grad_norm(acc, per_tensor=True)
            n3, coef = accumulate_grads_(acc, ts, norm_type=1.0, max_norm=3.0)
        graphs.append(g)
        outs.append((norm, n2, norms, n3, coef))
    streams = [torch.cuda.Stream() for _ in graphs]
    for round_ in range(5):
        for k, ts in enumerate(lists):
            fresh = make([t.numel() for t in ts], BF16, seed=100 * round_ + k)[1]
            for t, f in zip(ts, fresh):
                t.copy_(f)
        torch.cuda.synchronize()
        for _ in range(3):
            for st, g in zip(streams, graphs):
                with torch.cuda.stream(st):
                    g.replay()
        grad_norm(lists[0])  # an eager call between them
        torch.cuda.synchronize()
        for ts, acc, (norm, n2, norms, n3, coef) in zip(lists, accs, outs):
            ref = [torch.zeros(t.shape, device="cuda") for t in ts]
            accumulate_grads_(ref, ts, overwrite=True)
            assert torch.equal(clip_grads_(ref, 0.5), norm)
            r2, rs = grad_norm(ref, per_tensor=True)
            assert torch.equal(r2, n2) and torch.equal(rs, norms)
            r3, rc = accumulate_grads_(ref, ts, norm_type=1.0, max_norm=3.0)
            assert torch.equal(r3, n3) and torch.equal(rc, coef)
            assert all(torch.equal(a, b) for a, b in zip(ref, acc))


def test_first_call_in_a_capture():
    """A process whose first calls are captured: nothing is left to be set up
    that a capture forbids."""
    import subprocess
    import sys
    code = """
import torch, luma_b200
x = [torch.full((n,), 2.0, device="cuda") for n in (9, 300_000)]
y = [torch.zeros_like(t) for t in x]
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    a = luma_b200.accumulate_grads_(y, x, 0.5, norm_type=2.0)
    b, c = luma_b200.grad_norm(x, per_tensor=True)
    d = luma_b200.clip_grads_(y, 1.0)
    e = luma_b200.clip_grads_(x[:1], 3.0)
g.replay()
torch.cuda.synchronize()
assert abs(float(a) - 300_009 ** 0.5) < 1e-3 and abs(float(b) - 2 * 300_009 ** 0.5) < 1e-3
assert float(c[0]) == 6.0 and torch.equal(a, d) and float(e) == 6.0
assert abs(float(luma_b200.grad_norm(y)) - 1) < 1e-5 and abs(float(x[0][0]) - 1) < 1e-5
"""
    root = luma_b200.__path__[0].rsplit("/", 1)[0]
    subprocess.run([sys.executable, "-c", code], check=True, cwd=root, timeout=300)


def test_c_entries_without_torch_lists():
    """The C ABI as another host uses it: its own arrays, a workspace of its
    own, the power of two halves reduced by the caller."""
    import ctypes
    from array import array
    from luma_b200 import _lib
    h = _lib.lib()
    flat, ts = make([1000, 0, 70_001, 5], BF16, offset=3)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    out = torch.full((8,), -1.0, dtype=torch.float64, device="cuda")
    powers = torch.full((2,), -1.0, dtype=torch.float64, device="cuda")
    for k, part in enumerate((ts[:2], ts[2:])):
        a = _lib.LumaGradArgs()
        ptrs = array("Q", [t.data_ptr() for t in part])
        numels = array("q", [t.numel() for t in part])
        codes = bytes([_lib.BF16] * len(part))
        a.grads, a.numel = ptrs.buffer_info()[0], numels.buffer_info()[0]
        a.dtypes = ctypes.cast(ctypes.c_char_p(codes), ctypes.c_void_p)
        a.n, a.norm_kind = len(part), _lib.NORM_2
        ws = torch.empty(_lib.grad_partials(len(part)), dtype=torch.float64, device="cuda")
        a.partials, a.n_partials = ws.data_ptr(), ws.numel()
        a.power = powers[k:].data_ptr()
        assert h.luma_grad_norm(ctypes.byref(a), stream) == _lib.LUMA_OK, h.luma_last_error()
    near(powers[0], exact_power(ts[0], 2.0), 20 * U)
    a = _lib.LumaGradArgs()
    a.partials, a.n_partials, a.norm_kind, a.max_norm = powers.data_ptr(), 2, _lib.NORM_2, 0.5
    norm, coef = out[:1].view(torch.float32)[:1], out[1:2].view(torch.float32)[:1]
    a.norm, a.coef = norm.data_ptr(), coef.data_ptr()
    assert h.luma_grad_finish(ctypes.byref(a), stream) == _lib.LUMA_OK, h.luma_last_error()
    near(norm, exact_norm(ts, 2.0), NORM_TOL[2.0])
    near(coef, exact_coef(exact_norm(ts, 2.0), 0.5), NORM_TOL[2.0] + U)
    assert (out[2:] == -1).all()
    a = _lib.LumaGradArgs()  # nothing to do
    assert h.luma_grad_scale(ctypes.byref(a), stream) == _lib.LUMA_OK
    assert h.luma_grad_accumulate(ctypes.byref(a), stream) == _lib.LUMA_OK


def test_compiled_callers():
    ts = make([1000, 17], F32)[1]

    @torch.compile(backend="eager")
    def f(x, y):
        return grad_norm([x, y]) * 2

    assert f(*ts) == grad_norm(ts) * 2


def test_inference_tensors():
    with torch.inference_mode():
        t = torch.ones(9, device="cuda")
        assert clip_grads_([t], 1.5) == 3.0
    near(t[0], exact_coef(3.0, 1.5), 2 * U)


# -- the run of a training step --------------------------------------------------------

def _model(seed, dtype=BF16):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shapes = [(65, 33), (1000,), (40_000,), (7,), (300, 100)]
    ps = [torch.nn.Parameter((torch.randn(s, device="cuda", generator=gen) * 0.02).to(dtype))
          for s in shapes]
    for p in ps:
        p.grad_dtype = None
    return ps


@pytest.mark.parametrize("capture", [False, True])
def test_micro_batches_clip_and_step(capture):
    """Two bf16 micro-batches into fp32 accumulators, norm and coefficient from
    the same pass, LUMA's step with the coefficient: the params of a step on
    accumulators that were clipped in place, bit for bit."""
    pa, pb = _model(0), _model(0)
    main = [torch.zeros(p.shape, device="cuda") for p in pa]
    opts = [LUMA(ps, lr=1e-2, capturable=capture) for ps in (pa, pb)]
    opts[1]._base_seed = opts[0]._base_seed
    micro = [[torch.zeros(p.shape, dtype=BF16, device="cuda") for p in pa] for _ in range(2)]
    for p, m in zip(pa, main):
        p.grad = m

    def train():
        accumulate_grads_(main, micro[0], 0.5, overwrite=True)
        norm, coef = accumulate_grads_(main, micro[1], 0.5, max_norm=0.5)
        opts[0].step(grad_scale=coef)
        return norm, coef

    gen = torch.Generator(device="cuda").manual_seed(9)
    graph = None
    for it in range(4):
        for m in micro:
            for t in m:
                t.normal_(0, 10.0 ** -it, generator=gen)
        if capture and it == 1:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = train()
        if graph is not None:
            graph.replay()
        else:
            out = train()
        norm, coef = out
        ref = [(a.float() * 0.5).double() for a in micro[0]]
        ref = [(r + b.double() * 0.5).float() for r, b in zip(ref, micro[1])]
        assert all(torch.equal(m, r) for m, r in zip(main, ref))  # halves and their sum: exact
        near(norm, exact_norm(ref, 2.0), NORM_TOL[2.0])
        for p, r in zip(pb, ref):
            p.grad = r
        assert (coef < 1) == (it < 3)
        scale_grads_([p.grad for p in pb], coef)
        opts[1].step()
        assert all(torch.equal(a, b) for a, b in zip(pa, pb)), it


def test_optimizer_clip_coef():
    ps = _model(1)
    for k, p in enumerate(ps[:-1]):
        p.grad = torch.randn(p.shape, device="cuda").to(TYPES[k % 3])
    opt = LUMA([{"params": ps[:2]}, {"params": ps[2:]}])
    norm, coef = opt.clip_coef(1.0)
    grads = [p.grad for p in ps[:-1]]
    near(norm, exact_norm(grads, 2.0), NORM_TOL[2.0])
    near(coef, exact_coef(exact_norm(grads, 2.0), 1.0), NORM_TOL[2.0] + U)
    assert opt.clip_coef(1.0, INF)[0] == max(float(g.abs().max()) for g in grads)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scaler_clip_step(dtype):
    """Against unscaling, clipping and stepping one after the other.  The loss
    scale is a power of two, so unscaling is exact and the steps differ by the
    rounding of the coefficient alone; skipped steps change nothing."""
    pa, pb = _model(2, F32), _model(2, F32)
    oa, ob = LUMA(pa, lr=1e-3), LUMA(pb, lr=1e-3)
    ob._base_seed = oa._base_seed
    sa = torch.amp.GradScaler("cuda", init_scale=2.0 ** 12, growth_interval=3)
    gen = torch.Generator(device="cuda").manual_seed(4)
    skipped = 0
    for it in range(8):
        scale = sa.scale(torch.ones((), device="cuda"))
        raw = [torch.randn(p.shape, device="cuda", generator=gen) * 0.01 for p in pa]
        if it in (0, 4):
            raw[2][123] = INF if it else NAN
        for p, g in zip(pa, raw):
            p.grad = (g * scale).to(dtype)
        before = [p.clone() for p in pa]
        kept = [p.grad.clone() for p in pa]
        norm = luma_b200.amp.clip_step(sa, oa, 0.25)
        assert all(torch.equal(p.grad.nan_to_num(), k.nan_to_num()) for p, k in zip(pa, kept))
        s0 = float(scale)
        sa.update()
        if it in (0, 4):
            skipped += 1
            assert not math.isfinite(float(norm)) and sa.get_scale() == s0 / 2
            assert all(torch.equal(a, b) for a, b in zip(pa, before))
            continue
        unscaled = [k.float() / s0 for k in kept]
        near(norm, exact_norm(unscaled, 2.0), NORM_TOL[2.0] + U)
        _, coef = clip_coef(kept, 0.25, inv_scale=torch.full((1,), 1 / s0, device="cuda"))
        for p, k in zip(pb, kept):
            p.grad = k
        ob.step(grad_scale=coef)
        assert all(torch.equal(a, b) for a, b in zip(pa, pb)), it
    assert skipped == 2 and oa.state_dict()["state"][0]["step"] == 6


def test_zero_shards():
    """The norm of a ZeRO shard leaves out the gaps between tensors."""
    from luma_b200.zero import ZeroLUMA, plan_layout
    layout = plan_layout([1000, 7, 33_333, 1], world=1, buckets=2)
    flat = torch.zeros(layout.total, dtype=BF16, device="cuda").normal_()
    z = ZeroLUMA(flat, layout, 0)
    grad = torch.full((layout.shard,), NAN, device="cuda")
    segs = [grad[s.local:s.local + s.length] for s in z.segments]
    for s in segs:
        s.normal_()
    assert sum(s.numel() for s in segs) == 1000 + 7 + 33_333 + 1
    want = exact_norm(segs, 2.0)
    near(z.grad_norm(grad), want, NORM_TOL[2.0])
    norm, coef = z.clip_coef(grad, 1.0)
    near(norm, want, NORM_TOL[2.0])
    near(coef, exact_coef(want, 1.0), NORM_TOL[2.0] + U)
    z.step(grad, grad_scale=coef)
    with pytest.raises(ValueError, match="grad_shard"):
        z.clip_coef(grad[1:], 1.0)


def test_process_group_of_one(tmp_path):
    """The reduction over ranks, with one rank: the same numbers, NaN as inf
    where a maximum is reduced."""
    import torch.distributed as dist
    dist.init_process_group("gloo", init_method=f"file://{tmp_path}/store", rank=0, world_size=1)
    try:
        pg = dist.group.WORLD
        for p in (1.0, 2.0, INF):
            _, ts = make([1000, 17], BF16)
            assert torch.equal(grad_norm(ts, p, process_group=pg), grad_norm(ts, p))
            flag = torch.zeros(1, device="cuda")
            inv = torch.full((1,), 0.125, device="cuda")
            got = clip_coef(ts, 0.01, p, process_group=pg, inv_scale=inv, found_inf=flag)
            want = clip_coef(ts, 0.01, p, inv_scale=inv)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and flag == 0
            a, b = [t.clone() for t in ts], [t.clone() for t in ts]
            assert torch.equal(clip_grads_(a, 0.01, p, process_group=pg), clip_grads_(b, 0.01, p))
            assert all(torch.equal(x, y) for x, y in zip(a, b))
            ts[0][3] = NAN
            near(grad_norm(ts, p, process_group=pg), INF if p == INF else NAN, 0)
            clip_coef(ts, 1.0, p, process_group=pg, found_inf=flag)
            assert flag == 1
        assert grad_norm([], process_group=pg) == 0.0  # a rank without shards
        norm, coef = clip_coef([], 1.0, process_group=pg)
        assert norm == 0.0 and coef == 1.0 and norm.is_cuda
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("seed", range(12))
def test_random_lists(seed):
    """Sizes, types, offsets and functions drawn together."""
    rng = np.random.default_rng(seed)
    count = int(np.exp(rng.uniform(0, np.log(1500))))
    sizes = [int(np.exp(rng.uniform(0, np.log(2e6 / count + 20)))) - 1 for _ in range(count)]
    ts, accs = [], []
    for k, n in enumerate(sizes):
        ts += make([n], TYPES[rng.integers(3)], offset=int(rng.integers(0, 17)), seed=k)[1]
        accs += make([n], TYPES[rng.integers(2)], offset=int(rng.integers(0, 17)), seed=k + 7)[1]
    p = [1.0, 2.0, INF][rng.integers(3)]
    norm, norms = grad_norm(ts, p, per_tensor=True)
    near(norm, exact_norm(ts, p), NORM_TOL[p])
    for got, t in zip(norms.tolist(), ts):
        near(got, exact_norm([t], p), NORM_TOL[p])
    before = [a.clone() for a in accs]
    norm, coef = accumulate_grads_(accs, ts, 0.5, norm_type=p, max_norm=0.1)
    for a, b, g in zip(accs, before, ts):
        check_accumulated(a, b, g, 0.5, False)
    near(norm, exact_norm(accs, p), NORM_TOL[p])
    want = plain_scale(accs, coef)
    scale_grads_(accs, coef)
    assert all(torch.equal(a, b) for a, b in zip(accs, want))
