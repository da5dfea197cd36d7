"""Cases of a layer's quantised work: rows in 8 bits, weights in 4.

A case is a dict of plain values; ``kind`` names the operator:

* ``norm8``: the residual's addition and RMSNorm with the result in 8 bits,
  a scale for each row and group of columns (``PreparedAddRMSNormInt8``);
* ``silu8``: SiLU(gate) * up with the result in 8 bits (``PreparedSiluMulInt8``);
* ``rows8``: rows brought to 8 bits (``PreparedQuantizeRowsInt8``);
* ``linear``: 16-bit rows times 4-bit weights with a scale, and where given a
  zero point, for each output column and group (``PreparedInt4Linear``), with
  the residual's addition or SiLU(gate) * up behind it;
* ``linear8``: the same over rows in 8 bits.

Where ``own`` is false the operators run in their plain form: elementary torch
operations in 32 bits, rounded once at the end. Rows in 8 bits are returned as
the values that they stand for, in the type of the rows that they came from.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
DEVICE = "cuda"
EPS = 1e-6


def listed():
    return [
        # The smallest call: one token of a small model's decode step.
        _norm8("norm8_t1", 1, 2048, "bf16", 128),
        # The rows of a batched prefill.
        _norm8("norm8_t8192", 8192, 4096, "bf16", 128),
        # A batch of decoding requests, an odd number of them.
        _silu8("silu8_t61", 61, 5632, "fp16", 64),
        # The gated activation of a long prefill chunk, the widest rows.
        _silu8("silu8_t4096", 4096, 14336, "bf16", 128),
        # Attention output of a decode batch, before the o projection.
        _rows8("rows8_t32", 32, 4096, "bf16", 128),
        # A ragged prefill chunk's, short groups.
        _rows8("rows8_t4099", 4099, 2048, "fp16", 32),
        # One request's gate and up projections with the activation: latency.
        _linear("linear_b1_silu", 1, 2048, 2 * 5632, "bf16", 128, epilogue="silu"),
        # A decode batch's o projection and its residual, weights with zero points.
        _linear("linear_b16_residual", 16, 4096, 4096, "fp16", 64, zeros=True, epilogue="residual"),
        # A short chunk of prompts, 16-bit rows.
        _linear("linear_t517", 517, 5632, 2048, "bf16", 128, zeros=True, epilogue="residual"),
        # A large model's gate projection for a whole decode batch.
        _linear("linear8_b32", 32, 4096, 14336, "bf16", 128),
        # A ragged prefill chunk, an odd number of columns, zero points.
        _linear("linear8_t2047", 2047, 2048, 5001, "fp16", 64, zeros=True),
        # The largest: a batched prefill through a large model's up projection.
        _linear("linear8_t8192", 8192, 4096, 14336, "bf16", 128),
    ]


def draw(rng):
    kind = rng.choice(("norm8", "silu8", "rows8", "linear", "linear", "linear8", "linear8"))
    group = rng.choice((32, 64, 128, 128))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if kind in ("norm8", "rows8", "silu8"):
        most = 14336 if kind == "silu8" else 8192
        cols = rng.choice((_spread(rng, group, most) // group * group, 2048, 4096))
        rows = _spread(rng, 1, min(8192, (1 << 25) // cols))
        make = {"norm8": _norm8, "silu8": _silu8, "rows8": _rows8}[kind]
        return make(None, rows, cols, dtype, group)
    cols = rng.choice((_spread(rng, 256, 14336) // group * group, 2048, 4096, 5632))
    outs = rng.choice((_spread(rng, 33, 14336), _spread(rng, 33, 14336), 4096))
    rows = rng.choice((_spread(rng, 1, 64), _spread(rng, 1, 8192)))
    epilogue = rng.choice(("none", "residual", "silu"))
    if epilogue == "silu":
        outs += outs % 2
    dearest = 1 << 36  # products of one row and one column, at most
    rows = max(1, min(rows, dearest // (cols * outs)))
    return _linear(None, rows, cols, outs, dtype, group, zeros=rng.random() < 0.4, epilogue=epilogue,
                   kind=kind)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    state = _PREPARE[case["kind"]](case, gen)
    if own:
        _bind(case, state)
    return {"case": case, **state}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["kind"]](state)


def work(case):
    rows, cols, eb = case["rows"], case["cols"], DTYPES[case["dtype"]].itemsize
    n, groups = rows * cols, rows * cols // case["group"]
    if case["kind"] == "norm8":  # x, delta and the weight; the sum, the codes and their scales
        return {"bytes": (3 * eb + 1) * n + eb * cols + 4 * groups, "flops": 7.0 * n}
    if case["kind"] == "silu8":
        return {"bytes": (2 * eb + 1) * n + 4 * groups, "flops": 8.0 * n}
    if case["kind"] == "rows8":
        return {"bytes": (eb + 1) * n + 4 * groups, "flops": 3.0 * n}
    outs = case["outs"]
    weight = outs * cols / 2 + outs * cols / case["group"] * (2.5 if case["zeros"] else 2)
    x = n + 4 * groups if case["kind"] == "linear8" else eb * n
    y = eb * rows * outs * {"none": 1, "residual": 2, "silu": 0.5}[case["epilogue"]]
    return {"bytes": weight + x + y, "flops": 2.0 * n * outs}


def exact(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    return _EXACT[case["kind"]](_PREPARE[case["kind"]](case, gen), case)


# ------------------------------------------------------------------ the cases
def _spread(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _case(name, kind, rows, cols, dtype, group, **more):
    case = {"kind": kind, "rows": rows, "cols": cols, "dtype": dtype, "group": group, **more}
    return case if name is None else {"name": name, **case}


def _norm8(name, rows, cols, dtype, group):
    return _case(name, "norm8", rows, cols, dtype, group)


def _silu8(name, rows, cols, dtype, group):
    return _case(name, "silu8", rows, cols, dtype, group)


def _rows8(name, rows, cols, dtype, group):
    return _case(name, "rows8", rows, cols, dtype, group)


def _linear(name, rows, cols, outs, dtype, group, *, zeros=False, epilogue="none", kind=None):
    kind = kind or ("linear8" if name.startswith("linear8") else "linear")
    return _case(name, kind, rows, cols, dtype, group, outs=outs, zeros=zeros, epilogue=epilogue)


# ----------------------------------------------------------------- the inputs
def _rows(gen, rows, cols, dtype, loudness=12.0):
    """Normal rows with a few columns that are larger throughout, as a model's residual stream has."""
    x = torch.randn(rows, cols, generator=gen, device=DEVICE)
    loud = torch.randint(0, cols, (max(1, cols // 256),), generator=gen, device=DEVICE)
    x[:, loud] *= loudness
    return x.to(DTYPES[dtype])


def _inputs_norm8(case, gen):
    rows, cols, dtype = case["rows"], case["cols"], case["dtype"]
    weight = (1 + 0.1 * torch.randn(cols, generator=gen, device=DEVICE)).to(DTYPES[dtype])
    return {"x": _rows(gen, rows, cols, dtype), "delta": _rows(gen, rows, cols, dtype), "weight": weight}


def _inputs_silu8(case, gen):
    both = _rows(gen, case["rows"], 2 * case["cols"], case["dtype"], 3.0)  # the gate and up projections' one result
    return {"gate": both[:, :case["cols"]], "up": both[:, case["cols"]:]}


def _inputs_rows8(case, gen):
    return {"x": _rows(gen, case["rows"], case["cols"], case["dtype"])}


def _inputs_linear(case, gen):
    rows, cols, outs, group, dtype = (case[k] for k in ("rows", "cols", "outs", "group", "dtype"))
    # codes of a normal weight: the middle ones are the most frequent
    codes = (torch.randn(outs, cols, generator=gen, device=DEVICE) * 2.5 + 8).round_().clamp_(0, 15).to(torch.uint8)
    step = torch.rand(outs, cols // group, generator=gen, device=DEVICE) + 0.5
    state = {"codes": codes, "scales": (step * (0.4 * cols ** -0.5)).to(DTYPES[dtype]), "zeros": None,
             "residual": None}
    if case["zeros"]:
        state["zeros"] = torch.randint(5, 12, (outs, cols // group), generator=gen, device=DEVICE).to(torch.uint8)
    if case["epilogue"] == "residual":
        state["residual"] = _rows(gen, rows, outs, dtype)
    x = _rows(gen, rows, cols, dtype)
    if case["kind"] == "linear":
        return state | {"x": x}
    grouped = x.float().view(rows, -1, group)
    scales = grouped.abs().amax(-1) / 127
    return state | {"x_scales": scales,
                    "x_codes": (grouped / scales[..., None]).round_().to(torch.int8).view(rows, cols)}


_PREPARE = {"norm8": _inputs_norm8, "silu8": _inputs_silu8, "rows8": _inputs_rows8, "linear": _inputs_linear,
            "linear8": _inputs_linear}


# ------------------------------------------------------------ the plain forms
def _in_8_bits(values, group, dtype):
    """What the rows' codes stand for: the nearest of 255 even steps up to each group's largest magnitude."""
    grouped = values.view(values.shape[0], -1, group)
    scale = grouped.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100) / 127
    return ((grouped / scale).round() * scale).view_as(values).to(dtype)


def _plain_norm8(state):
    x = state["x"]
    total = (x.float() + state["delta"].float()).to(x.dtype)
    t = total.float()
    t = t * torch.rsqrt((t * t).mean(-1, keepdim=True) + EPS) * state["weight"].float()
    return {"sum": total, "values": _in_8_bits(t, state["case"]["group"], x.dtype)}


def _plain_silu8(state):
    gate = state["gate"].float()
    values = gate / (1 + torch.exp(-gate)) * state["up"].float()
    return {"values": _in_8_bits(values, state["case"]["group"], state["gate"].dtype)}


def _plain_rows8(state):
    return {"values": _in_8_bits(state["x"].float(), state["case"]["group"], state["x"].dtype)}


def _plain_linear(state):
    group, codes, scales = state["case"]["group"], state["codes"], state["scales"]
    zeros = 8.0 if state["zeros"] is None else state["zeros"].float()[..., None]
    weight = ((codes.float().view(codes.shape[0], -1, group) - zeros) * scales.float()[..., None]).view_as(codes)
    if state["case"]["kind"] == "linear":
        x = state["x"].float()
    else:
        x = state["x_codes"]
        x = (x.float().view(x.shape[0], -1, group) * state["x_scales"][..., None]).view_as(x)
    y = x @ weight.t()
    if state["case"]["epilogue"] == "silu":
        gate, up = y.chunk(2, -1)
        y = gate / (1 + torch.exp(-gate)) * up
    if state["residual"] is not None:
        y = y + state["residual"].float()
    return y.to(scales.dtype)


_PLAIN = {"norm8": _plain_norm8, "silu8": _plain_silu8, "rows8": _plain_rows8, "linear": _plain_linear,
          "linear8": _plain_linear}


# ---------------------------------------------------- the definitions, 64 bits
def _stepped(v, group):
    """Each value on its group's grid."""
    parts = []
    for part in v.split(group, dim=1):
        largest = part.abs().max(dim=1, keepdim=True).values.clamp(min=2.0 ** -100)
        parts.append(torch.round(part * 127.0 / largest) * largest / 127.0)
    return torch.cat(parts, 1)


def _exact_norm8(state, case):
    total = (state["x"].double() + state["delta"].double()).to(DTYPES[case["dtype"]]).double()
    root = ((total ** 2).sum(1, keepdim=True) / case["cols"] + EPS).sqrt()
    return {"sum": total, "values": _stepped(total / root * state["weight"].double(), case["group"])}


def _exact_silu8(state, case):
    gate = state["gate"].double()
    return {"values": _stepped(gate * torch.sigmoid(gate) * state["up"].double(), case["group"])}


def _exact_rows8(state, case):
    return {"values": _stepped(state["x"].double(), case["group"])}


def _exact_linear(state, case):
    """Group by group of the contraction."""
    g, sums = case["group"], torch.zeros(case["rows"], case["outs"], dtype=torch.float64, device=DEVICE)
    for i in range(case["cols"] // g):
        at = slice(i * g, (i + 1) * g)
        zero = 8 if state["zeros"] is None else state["zeros"][:, i:i + 1].double()
        w = (state["codes"][:, at].double() - zero) * state["scales"][:, i:i + 1].double()
        if case["kind"] == "linear":
            part = state["x"][:, at].double()
        else:
            part = state["x_codes"][:, at].double() * state["x_scales"][:, i:i + 1].double()
        sums += torch.mm(part, w.t().contiguous())
    if case["epilogue"] == "silu":
        half = case["outs"] // 2
        sums = sums[:, :half] * torch.sigmoid(sums[:, :half]) * sums[:, half:]
    if case["epilogue"] == "residual":
        sums += state["residual"].double()
    return sums


_EXACT = {"norm8": _exact_norm8, "silu8": _exact_silu8, "rows8": _exact_rows8, "linear": _exact_linear,
          "linear8": _exact_linear}


# ----------------------------------------------------- the framework's calls
def _bind(case, state):
    """The weights as a serving program keeps them, and its handles on the step's buffers."""
    import inferkernellab_amd as ikl

    kind, group = case["kind"], case["group"]
    if kind == "norm8":
        state["call"] = ikl.PreparedAddRMSNormInt8(state["x"], state["delta"], state["weight"], eps=EPS,
                                                   group_size=group)
    elif kind == "silu8":
        state["call"] = ikl.PreparedSiluMulInt8(state["gate"], state["up"], group_size=group)
    elif kind == "rows8":
        state["call"] = ikl.PreparedQuantizeRowsInt8(state["x"], group_size=group)
    else:
        weight = ikl.pack_int4_weight(state["codes"], state["scales"], state["zeros"], group_size=group,
                                      gated=case["epilogue"] == "silu")
        x = state["x"] if kind == "linear" else ikl.Int8Rows(state["x_codes"], state["x_scales"], group,
                                                             dtype=DTYPES[case["dtype"]])
        state["call"] = ikl.PreparedInt4Linear(x, weight, residual=state["residual"])
    if kind in ("norm8", "silu8", "rows8"):
        state["values"] = torch.empty(case["rows"], case["cols"], dtype=DTYPES[case["dtype"]], device=DEVICE)


def _own(state):
    kind = state["case"]["kind"]
    if kind in ("linear", "linear8"):
        return state["call"]()
    if kind == "norm8":
        total, rows = state["call"]()
        return {"sum": total, "values": rows.dequantize(out=state["values"])}
    return {"values": state["call"]().dequantize(out=state["values"])}
