"""Cases of the gradient operators: what runs between the backward pass and the optimizer step.

Norms over many tensors, the clip coefficient (with a loss scale's unscaling and its inf/NaN
flag), clipping in place, and the accumulation of micro-batches into wider buffers.

The operators take lists of tensors.  The plain form joins a list into a workspace first and works
on that as a whole, so it needs no launch per tensor.  The tensors of a list lie one behind the
other in a buffer, as in a data-parallel bucket or a ZeRO shard, so that what a pass writes to
them can be returned whole."""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_ROW = 4096  # buffers are padded to whole rows of this many elements


# -- sizes --------------------------------------------------------------------

def _layer(d, kv, ffn):
    return [d * d, kv * d, kv * d, d * d, ffn * d, ffn * d, d * ffn, d, d]


def _sizes(case):
    """Elements of each gradient tensor of the case (ragged: multiples of ``multiple``)."""
    kind = case["sizes"]
    if kind == "decoder":  # the benchmark's Llama-3-8B shapes, 291 tensors
        vocab, d = 128256, 4096
        return [vocab * d] + _layer(4096, 1024, 14336) * 32 + [d, vocab * d]
    if kind == "layer":  # one of its decoder layers, 9 tensors
        return _layer(4096, 1024, 14336)
    if kind == "cpu21m":  # the benchmark's 8 tensors, 20,971,520 elements
        return [1024 * 1024] * 4 + [4096 * 1024] * 4
    if kind == "ragged":  # log-uniform in [lo, hi]
        rng = np.random.default_rng(case["size_seed"])
        draw = np.exp(rng.uniform(math.log(case["lo"]), math.log(case["hi"]), case["count"]))
        m = case["multiple"]
        return [max(1, -(-int(round(v)) // m)) * m for v in draw]
    raise ValueError(kind)


# -- cases --------------------------------------------------------------------

def listed():
    return [
        # the smallest call: the norm of one bias gradient, where latency is all there is
        {"name": "norm_bias", "op": "norm", "sizes": "ragged", "count": 1, "lo": 4096, "hi": 4096,
         "size_seed": 0, "multiple": 8, "type": "bf16", "norm": 2.0, "std": 1e-3},
        # the global norm before every step of the benchmark's 8 G-parameter model: the largest
        {"name": "norm_decoder", "op": "norm", "sizes": "decoder", "type": "bf16",
         "norm": 2.0, "std": 1e-3},
        # largest magnitude of a small fp16 model's gradients, tensors at odd offsets
        {"name": "norm_max_f16", "op": "norm", "sizes": "ragged", "count": 147, "lo": 1,
         "hi": 3000017, "size_seed": 3, "multiple": 1, "type": "f16", "norm": math.inf, "std": 1e-2},
        # a norm for each of the 10,000 tensors of the ragged stress, as a training log wants them
        {"name": "norms_ragged", "op": "norms", "sizes": "ragged", "count": 10000, "lo": 1,
         "hi": 1 << 20, "size_seed": 0, "multiple": 1, "type": "f32", "norm": 2.0, "std": 1e-2},
        # a norm for each tensor of one decoder layer
        {"name": "norms_layer", "op": "norms", "sizes": "layer", "type": "bf16",
         "norm": 2.0, "std": 1e-3},
        # mixed precision: unscaling, inf/NaN flag, norm and clip coefficient of fp32 gradients
        {"name": "coef_21m", "op": "coef", "sizes": "cpu21m", "type": "f32",
         "norm": 2.0, "std": 1e-2, "loss_scale": 65536.0, "max_norm": 1.0},
        # the same for bf16 gradients of odd sizes at odd offsets
        {"name": "coef_odd", "op": "coef", "sizes": "ragged", "count": 148, "lo": 7,
         "hi": 2000003, "size_seed": 5, "multiple": 1, "type": "bf16", "norm": 2.0, "std": 1e-2,
         "loss_scale": 1024.0, "max_norm": 1.0},
        # clipping in place late in training: the norm is below the bound, nothing changes
        {"name": "clip_within", "op": "clip", "sizes": "layer", "type": "bf16",
         "norm": 2.0, "std": 1e-5, "max_norm": 1.0},
        # clipping a small adapter's gradients in place (the tensors are first filled from a
        # half-precision backward pass), clip active
        {"name": "clip_adapter", "op": "fill_clip", "sizes": "ragged", "count": 33, "lo": 5,
         "hi": 70001, "size_seed": 7, "multiple": 8, "type": "f16", "acc": "bf16", "norm": 2.0,
         "std": 1e-1, "max_norm": 1.0, "scale": 1.0},
        # clipping the 21 M fp32 gradients filled from a bf16 backward pass, clip active
        {"name": "clip_21m", "op": "fill_clip", "sizes": "cpu21m", "type": "bf16",
         "acc": "f32", "norm": 2.0, "std": 1e-2, "max_norm": 1.0, "scale": 1.0},
        # two micro-batches of one decoder layer into fp32, norm and clip coefficient of the sum
        {"name": "accumulate_layer", "op": "accumulate", "sizes": "layer",
         "type": "bf16", "acc": "f32", "norm": 2.0, "std": 1e-3, "max_norm": 1.0, "scale": 0.5},
        # the same for odd sizes at odd offsets, accumulated in bf16
        {"name": "accumulate_odd", "op": "accumulate", "sizes": "ragged", "count": 301, "lo": 1,
         "hi": 999983, "size_seed": 11, "multiple": 1, "type": "f32", "acc": "bf16", "norm": 2.0,
         "std": 1e-2, "max_norm": 1.0, "scale": 0.5},
    ]


def draw(rng):
    op = rng.choice(["norm", "norms", "coef", "clip", "fill_clip", "accumulate"])
    count = max(1, int(round(math.exp(rng.uniform(0.0, math.log(4000.0))))))
    # log-uniform sizes have a mean near hi / log(hi): bound the sum by about 3e8 elements
    most = min(float(1 << 27), max(64.0, 3e8 / count * 10.0))
    hi = int(math.exp(rng.uniform(math.log(16.0), math.log(most))))
    lo = rng.randint(1, max(1, min(hi, 1 + hi // 8)))
    case = {"op": op, "sizes": "ragged", "count": count, "lo": lo, "hi": hi,
            "size_seed": rng.randrange(1 << 20), "multiple": rng.choice([1, 8, 8, 64]),
            "type": rng.choice(["f32", "bf16", "bf16", "f16"]),
            "norm": rng.choice([2.0, 2.0, 2.0, 1.0, math.inf]),
            "std": round(10.0 ** rng.uniform(-4.0, -1.0), 7)}
    if op == "coef":
        case["type"] = rng.choice(["f32", "bf16"])
        case["loss_scale"] = float(1 << rng.randrange(4, 20))
    if op in ("fill_clip", "accumulate"):
        case["acc"] = rng.choice(["f32", "f32", "bf16"])
        case["scale"] = 1.0 / rng.choice([1, 2, 3, 8])
    if op in ("coef", "accumulate"):
        case["max_norm"] = rng.choice([0.1, 1.0, 1e4])
    if op == "clip":
        case["max_norm"] = 1e9  # within the bound, so that a pass leaves the gradients alone
    if op == "fill_clip":
        case["max_norm"] = round(10.0 ** rng.uniform(-3.0, 0.0), 6)
    return case


# -- inputs -------------------------------------------------------------------

def _fill(flat, case, gen):
    """Gradients N(0, std) with a spread of magnitudes from row to row, times the loss scale."""
    flat.normal_(0.0, case["std"] * case.get("loss_scale", 1.0), generator=gen)
    rows = flat.view(-1, _ROW)
    spread = torch.empty(rows.shape[0], 1, dtype=flat.dtype, device=flat.device)
    spread.log_normal_(0.0, 0.5, generator=gen)
    rows.mul_(spread)


def prepare(case, seed):
    dev = torch.device("cuda")
    sizes = _sizes(case)
    n = sum(sizes)
    total = -(-n // _ROW) * _ROW
    gen = torch.Generator(device=dev).manual_seed(seed)
    flats, grads = [], []
    for _ in range(2 if case["op"] == "accumulate" else 1):
        flat = torch.empty(total, dtype=_TYPES[case["type"]], device=dev)
        _fill(flat, case, gen)
        flats.append(flat[:n])
        grads.append(list(flat[:n].split(sizes)))
    # the plain form's workspace, zeros behind the last tensor
    s = {"case": case, "flats": flats, "grads": grads,
         "joined": torch.zeros(total, dtype=_TYPES[case["type"]], device=dev)}
    if case["op"] == "norms":
        # the joined list cut into pieces of at most a row, none of which holds two tensors
        room = np.array(sizes, dtype=np.int64)
        per = -(-room // _ROW)
        pieces = np.full(int(per.sum()), _ROW, dtype=np.int64)
        pieces[np.cumsum(per) - 1] = room - (per - 1) * _ROW
        s["pieces"] = torch.from_numpy(pieces).to(dev)
        s["pieces_of"] = torch.from_numpy(per).to(dev)
    if case["op"] == "coef":
        s["inv_scale"] = torch.full((1,), 1.0 / case["loss_scale"], device=dev)
        s["found_inf"] = torch.zeros(1, device=dev)
    if "acc" in case:
        acc = torch.zeros(total, dtype=_TYPES[case["acc"]], device=dev)
        s["wide"] = acc  # with zeros behind the last tensor
        s["acc"] = acc[:n]
        s["accs"] = list(acc[:n].split(sizes))
    return s


# -- the plain form -----------------------------------------------------------

def _rows_sum(x):
    """Sum of all elements: rows in 32 bits, their sums in 64."""
    return x.view(-1, _ROW).sum(1).double().sum()


def _plain_norm(flat, p):
    x = flat.to(torch.float32, copy=True).abs_()
    if math.isinf(p):
        return x.max()
    if p == 2.0:
        return _rows_sum(x.mul_(x)).sqrt().float()
    return _rows_sum(x).float()


def _plain_norms(flat, pieces, pieces_of, p):
    x = flat.double().abs_()
    how = "max" if math.isinf(p) else "sum"
    x = torch.segment_reduce(x.mul_(x) if p == 2.0 else x, how, lengths=pieces)
    x = torch.segment_reduce(x, how, lengths=pieces_of)
    return (x.sqrt() if p == 2.0 else x).float()


def _plain_coef(norm, max_norm):
    return (max_norm / (norm + 1e-6)).clamp(max=1.0)


def _plain(s):
    case, p = s["case"], s["case"]["norm"]
    joined, op = s["joined"], case["op"]
    n = s["flats"][0].numel()
    flat = joined[:n]
    torch.cat(s["grads"][0], out=flat)
    if op == "norm":
        return {"norm": _plain_norm(joined, p)}
    if op == "norms":
        norms = _plain_norms(flat, s["pieces"], s["pieces_of"], p)
        x = norms.double()
        total = x.max() if math.isinf(p) else x.square().sum().sqrt() if p == 2.0 else x.sum()
        return {"norm": total.float(), "norms": norms}
    if op == "coef":
        inv = s["inv_scale"][0]
        norm = _plain_norm(joined, p) * inv
        found = s["found_inf"]
        found.fill_(0.0)
        found.copy_(torch.maximum(found, (~torch.isfinite(flat)).any().float()))
        return {"norm": norm, "coef": _plain_coef(norm, case["max_norm"]) * inv, "found_inf": found}
    if op == "clip":
        norm = _plain_norm(joined, p)
        grads = s["flats"][0]
        grads.copy_(flat.float().mul_(_plain_coef(norm, case["max_norm"])))
        return {"norm": norm, "grads": grads}
    acc, wide = s["acc"], s["wide"]
    acc.copy_(flat.float().mul_(case["scale"]))
    if op == "fill_clip":
        norm = _plain_norm(wide, p)
        acc.copy_(acc.float().mul_(_plain_coef(norm, case["max_norm"])))
        return {"norm": norm, "grads": acc}
    torch.cat(s["grads"][1], out=flat)
    acc.copy_(acc.float().add_(flat.float().mul_(case["scale"])))
    norm = _plain_norm(wide, p)
    return {"norm": norm, "coef": _plain_coef(norm, case["max_norm"]), "grads": acc}


# -- a pass -------------------------------------------------------------------

def run(s):
    if not own:
        return _plain(s)
    import luma_b200
    case = s["case"]
    op, p, grads = case["op"], case["norm"], s["grads"][0]
    if op == "norm":
        return {"norm": luma_b200.grad_norm(grads, p)}
    if op == "norms":
        norm, norms = luma_b200.grad_norm(grads, p, per_tensor=True)
        return {"norm": norm, "norms": norms}
    if op == "coef":
        found = s["found_inf"]
        found.zero_()
        norm, coef = luma_b200.clip_coef(grads, case["max_norm"], p, inv_scale=s["inv_scale"],
                                         found_inf=found)
        return {"norm": norm, "coef": coef, "found_inf": found}
    if op == "clip":
        norm = luma_b200.clip_grads_(grads, case["max_norm"], p)
        return {"norm": norm, "grads": s["flats"][0]}
    accs = s["accs"]
    luma_b200.accumulate_grads_(accs, grads, case["scale"], overwrite=True)
    if op == "fill_clip":
        norm = luma_b200.clip_grads_(accs, case["max_norm"], p)
        return {"norm": norm, "grads": s["acc"]}
    norm, coef = luma_b200.accumulate_grads_(accs, s["grads"][1], case["scale"], norm_type=p,
                                             max_norm=case["max_norm"])
    return {"norm": norm, "coef": coef, "grads": s["acc"]}


# -- what a pass cannot do without --------------------------------------------

def work(case):
    sizes = _sizes(case)
    n, count = sum(sizes), len(sizes)
    size = _TYPES[case["type"]].itemsize
    op = case["op"]
    if op == "norm":
        return {"bytes": n * size + 4, "flops": 2 * n}
    if op == "norms":
        return {"bytes": n * size + 4 * count + 4, "flops": 2 * n}
    if op == "coef":
        return {"bytes": n * size + 16, "flops": 2 * n}
    if op == "clip":  # within the bound: the gradients stay as they are
        return {"bytes": n * size + 4, "flops": 2 * n}
    wide = _TYPES[case["acc"]].itemsize
    if op == "fill_clip":
        return {"bytes": n * (size + wide) + 4, "flops": 4 * n}
    return {"bytes": n * (2 * size + wide) + 8, "flops": 6 * n}


# -- the definition in 64 bits ------------------------------------------------

def _power(x, p):
    x = x.to(torch.float64)
    if math.isinf(p):
        return x.abs().max()
    return (x * x).sum() if p == 2.0 else x.abs().sum()


def _exact_norm(flat, p):
    """Norm of a buffer piece by piece (a whole copy in 64 bits may not fit)."""
    parts = torch.stack([_power(piece, p) for piece in flat.split(1 << 26)])
    if math.isinf(p):
        return parts.max()
    return parts.sum().sqrt() if p == 2.0 else parts.sum()


def exact(case, seed):
    s = prepare(case, seed)
    p, op = case["norm"], case["op"]
    flat = s["flats"][0]
    if op in ("norm", "clip"):
        norm = _exact_norm(flat, p)
        if op == "norm":
            return {"norm": norm}
        c = torch.clamp(case["max_norm"] / (norm + 1e-6), max=1.0)
        return {"norm": norm, "grads": flat.double() * c}
    if op == "norms":
        parts = torch.stack([_power(g, p) for g in s["grads"][0]])
        if math.isinf(p):
            return {"norm": parts.max(), "norms": parts}
        root = torch.sqrt if p == 2.0 else (lambda v: v)
        return {"norm": root(parts.sum()), "norms": root(parts)}
    if op == "coef":
        inv = 1.0 / case["loss_scale"]
        norm = _exact_norm(flat, p) * inv
        coef = torch.clamp(case["max_norm"] / (norm + 1e-6), max=1.0) * inv
        finite = bool(torch.isfinite(norm))
        return {"norm": norm, "coef": coef,
                "found_inf": torch.full((1,), 0.0 if finite else 1.0, dtype=torch.float64)}
    # what an accumulator holds between two calls is rounded to its type
    x = (flat.double() * case["scale"]).to(_TYPES[case["acc"]]).double()
    if op == "accumulate":
        x = (x + s["flats"][1].double() * case["scale"]).to(_TYPES[case["acc"]]).double()
        norm = _exact_norm(x, p)
        return {"norm": norm, "coef": torch.clamp(case["max_norm"] / (norm + 1e-6), max=1.0),
                "grads": x}
    norm = _exact_norm(x, p)
    return {"norm": norm, "grads": x * torch.clamp(case["max_norm"] / (norm + 1e-6), max=1.0)}
