"""Cases of the operators around the routed experts of a decoder layer whose
weights are e4m3 with a scale for each 128x128 block.

Such a layer first adds the residual stream and normalises it, with an output
in 16 bits for the router and the routed experts and one in 8 bits for the
dense products (``fused_rms_norm``); multiplies 8-bit activations by 8-bit
weights in the shared expert and the projections (``fp8_block_matmul``); and
between the shared expert's two products applies the gated activation and
returns to 8 bits (``silu_and_mul_quant``). Decode steps of one to a few dozen
tokens and prefill chunks of up to 8192 are both in.
"""

import math
import os
import sys

import torch

own = False

_package = None


def _fgs():
    """The framework, imported where ``own`` is true only."""
    global _package
    if _package is None:
        path = os.path.join(os.getcwd(), "flaggems-sglang_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import flaggems_sglang

        _package = flaggems_sglang
    return _package


_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_FP8 = torch.float8_e4m3fn


# ------------------------------------------------------------------ cases ---
def _norm(name, dtype, rows, cols, **more):
    case = dict(name=name, op="norm", dtype=dtype, rows=rows, cols=cols, residual=True,
                quant="fp8", norm_out=True, offset=0.0, column=False, gap=0)
    case.update(more)
    return case


def _act(name, dtype, rows, cols, **more):
    case = dict(name=name, op="act", dtype=dtype, rows=rows, cols=cols, quant="fp8",
                gelu=False, column=False)
    case.update(more)
    return case


def _product(name, m, n, k, **more):
    case = dict(name=name, op="product", dtype="bf16", m=m, n=n, k=k, bias=False, column=False)
    case.update(more)
    return case


def listed():
    return [
        # the norm before an fp8 layer: one token of a chat request (latency),
        # and the largest prefill chunk
        _norm("norm_decode", "bf16", 1, 7168),
        _norm("norm_prefill", "bf16", 8192, 7168, column=True),
        # a decode batch on a layer without 8-bit products, whose weight is
        # stored about zero
        _norm("norm_plain", "fp16", 61, 4096, quant="none", offset=1.0),
        # a prefill chunk before int8 products, the first norm of a model: no
        # residual yet
        _norm("norm_int8", "bf16", 1021, 3584, quant="int8", residual=False, norm_out=False),
        # the shared expert's middle: a decode batch, a prefill chunk with a
        # wide intermediate size, an odd int8 one
        _act("act_decode", "bf16", 8, 2048),
        _act("act_prefill", "bf16", 8192, 14336, column=True),
        _act("act_int8", "bf16", 999, 2560, quant="int8"),
        # the shared expert's gate and up product of one token: the weights'
        # bytes and the launch
        _product("product_decode", 1, 4096, 7168),
        # its down product in a decode batch
        _product("product_batch", 48, 7168, 2048),
        # a projection whose sizes end inside a block, on an odd chunk
        _product("product_ragged", 333, 2112, 1552, bias=True),
        # prefill chunks: the shared expert, and a wide dense layer
        _product("product_prefill", 4096, 4096, 7168, column=True),
        _product("product_large", 8192, 14336, 7168, column=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "act", "product", "product"])
    column = rng.random() < 0.5
    if op == "product":
        m = _log_int(rng, 1, 8192)
        n = _log_int(rng, 16, 16384)
        if rng.random() < 0.5:  # whole blocks about half of the time
            n = max(128, n // 128 * 128)
        k = 16 * _log_int(rng, 8, 1024)
        if rng.random() < 0.5:
            k = max(128, k // 128 * 128)
        while m * n * k > 8192 * 14336 * 7168:
            m = max(1, m // 2)
        case = _product("", m, n, k, bias=rng.random() < 0.3, column=column,
                        dtype=rng.choice(["bf16", "bf16", "fp16"]))
    else:
        rows = _log_int(rng, 1, 8192)
        cols = _log_int(rng, 64, 16384)
        step = rng.choice([1, 8, 128, 128])  # odd sizes, whole vectors, whole groups
        cols = max(step, cols // step * step)
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        quant = rng.choice(["fp8", "fp8", "int8"])
        if op == "norm":
            case = _norm("", dtype, rows, cols, quant=rng.choice([quant, quant, "none"]),
                         residual=rng.random() < 0.7, norm_out=rng.random() < 0.6,
                         offset=rng.choice([0.0, 0.0, 1.0]), column=column,
                         gap=rng.choice([0, 0, 64]))  # rows of a wider tensor
            case["norm_out"] = case["norm_out"] or case["quant"] == "none"
        else:
            case = _act("", dtype, rows, cols, quant=quant, gelu=rng.random() < 0.2,
                        column=column)
    del case["name"]
    return case


# ----------------------------------------------------------------- inputs ---
def _activations(rows, cols, gen, dtype):
    """Rows of a hidden state: token norms that differ, a few loud channels."""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    loud = torch.rand(cols, generator=gen, device="cuda") < 0.01
    x *= torch.where(loud, 8.0, 1.0)
    x *= 0.5 + torch.rand(rows, 1, generator=gen, device="cuda")
    return x.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    s = {"case": dict(case)}
    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        s["x"] = _activations(rows, cols + case["gap"], gen, dtype)[:, :cols]
        s["residual"] = _activations(rows, cols, gen, dtype) if case["residual"] else None
        weight = 1.0 - case["offset"] + 0.1 * torch.randn(cols, generator=gen, device="cuda")
        s["weight"] = weight.to(dtype)
        s["eps"] = 1e-6
    elif case["op"] == "act":
        s["x"] = _activations(case["rows"], 2 * case["cols"], gen, dtype)
    else:
        m, n, k = case["m"], case["n"], case["k"]
        kb = -(-k // 128)
        # what a quantiser gives: each group's largest value is 448
        x = _activations(m, kb * 128, gen, torch.float32)
        x[:, k:] = 0
        x = x.reshape(m, kb, 128)
        scale = x.abs().amax(-1).clamp(min=1e-10) / 448
        s["a"] = (x / scale[..., None]).clamp(-448, 448).to(_FP8).reshape(m, -1)[:, :k].contiguous()
        s["a_scale"] = scale.t().contiguous().t() if case["column"] else scale
        nb = -(-n // 128)
        w = torch.randn(n, k, generator=gen, device="cuda")
        s["w"] = (w * 90).clamp(-448, 448).to(_FP8)
        s["w_scale"] = (0.02 / 90) * (0.5 + torch.rand(nb, kb, generator=gen, device="cuda"))
        s["bias"] = None
        if case["bias"]:
            s["bias"] = torch.randn(n, generator=gen, device="cuda").to(dtype)
    return s


# ------------------------------------------------------------------- runs ---
def _quantised(v, quant):
    """(values of the codes, scales) of the rows of ``v`` in 32 bits."""
    rows, cols = v.shape
    if quant == "int8":
        scale = v.abs().amax(-1, keepdim=True).clamp(min=1e-10) / 127
        q = torch.round(v / scale).clamp(-127, 127) * scale
        return q.to(torch.bfloat16), scale[:, 0]
    groups = -(-cols // 128)
    g = torch.nn.functional.pad(v, (0, groups * 128 - cols)).reshape(rows, groups, 128)
    scale = g.abs().amax(-1).clamp(min=1e-10) / 448
    q = (g / scale[..., None]).clamp(-448, 448).to(_FP8)
    return q.reshape(rows, -1)[:, :cols], scale


def _values(q, scales):
    """int8 codes as the values that they stand for; e4m3 ones are values."""
    if q.dtype == torch.int8:
        values = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
        return torch.mul(q, scales[:, None], out=values)
    return q


def _run_norm(s):
    c = s["case"]
    quant = None if c["quant"] == "none" else c["quant"]
    if own:
        o = _fgs().fused_rms_norm(s["x"], s["weight"], s["eps"], s["residual"],
                                  weight_offset=c["offset"], quant=quant,
                                  return_norm=c["norm_out"], column_major_scales=c["column"])
        out = {"norm": o.norm, "residual": o.residual, "scales": o.scales}
        if quant:
            out["q"] = _values(o.q, o.scales)
    else:
        h = s["x"].float()
        out = {}
        if s["residual"] is not None:
            h = h + s["residual"].float()
            out["residual"] = h.to(s["x"].dtype)
        n = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + s["eps"])
        n = n * (s["weight"].float() + c["offset"])
        if c["norm_out"]:
            out["norm"] = n.to(s["x"].dtype)
        if quant:
            out["q"], out["scales"] = _quantised(n, quant)
    return {k: v for k, v in out.items() if v is not None}


def _run_act(s):
    c = s["case"]
    if own:
        q, scales = _fgs().silu_and_mul_quant(
            s["x"], c["quant"], activation="gelu" if c["gelu"] else "silu",
            column_major_scales=c["column"])
        return {"q": _values(q, scales), "scales": scales}
    x = s["x"].float()
    gate, up = x[:, :c["cols"]], x[:, c["cols"]:]
    if c["gelu"]:
        gate = 0.5 * gate * (1 + torch.erf(gate * math.sqrt(0.5)))
    else:
        gate = gate / (1 + torch.exp(-gate))
    q, scales = _quantised(gate * up, c["quant"])
    return {"q": q, "scales": scales}


def _run_product(s):
    c = s["case"]
    dtype = _TYPES[c["dtype"]]
    if own:
        return _fgs().fp8_block_matmul(s["a"], s["a_scale"], s["w"], s["w_scale"],
                                       bias=s["bias"], out_dtype=dtype)
    spread = torch.repeat_interleave
    a = s["a"].float() * spread(s["a_scale"], 128, 1)[:, :c["k"]]
    w = spread(spread(s["w_scale"], 128, 1)[:, :c["k"]], 128, 0)[:c["n"]] * s["w"].float()
    out = a @ w.t()
    if s["bias"] is not None:
        out = out + s["bias"].float()
    return out.to(dtype)


def run(s):
    return {"norm": _run_norm, "act": _run_act, "product": _run_product}[s["case"]["op"]](s)


# ------------------------------------------------------------------- work ---
def work(case):
    size = _TYPES[case["dtype"]].itemsize
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        kb, nb = -(-k // 128), -(-n // 128)
        return {"bytes": m * k + n * k + 4 * kb * (m + nb) + size * m * n
                + (size * n if case["bias"] else 0), "flops": 2 * m * n * k}
    rows, cols = case["rows"], case["cols"]
    values = rows * cols
    scales = 4 * rows * {"none": 0, "int8": 1, "fp8": -(-cols // 128)}[case["quant"]]
    codes = 0 if case["quant"] == "none" else values
    if case["op"] == "act":
        return {"bytes": 2 * size * values + codes + scales, "flops": 10 * values}
    moved = 1 + 2 * case["residual"] + case["norm_out"]
    return {"bytes": size * (moved * values + cols) + codes + scales, "flops": 8 * values}


# ------------------------------------------------------------------ exact ---
def _exact_codes(v, quant):
    """The codes' values and scales of ``v`` (64 bits), from the formats'
    definitions: int8 counts steps of the scale; an e4m3 value has three bits
    behind its leading one, and steps of 2^-9 below 2^-6."""
    rows, cols = v.shape
    if quant == "int8":
        scale = v.abs().max(-1, keepdim=True).values.clamp(min=1e-10) / 127
        return {"q": torch.round(v / scale) * scale, "scales": scale[:, 0]}
    groups = (cols + 127) // 128
    scales = torch.stack([v[:, 128 * g:128 * g + 128].abs().max(-1).values for g in range(groups)],
                         1).clamp(min=1e-10) / 448
    t = v / scales[:, torch.arange(cols, device=v.device) // 128]
    step = torch.exp2(torch.frexp(t.abs().clamp(min=2.0 ** -6)).exponent.double() - 4)
    return {"q": (torch.round(t / step) * step).clamp(-448, 448), "scales": scales}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = s["x"].double()
        out = {}
        if s["residual"] is not None:
            h = h + s["residual"].double()
            out["residual"] = h
        root = torch.sqrt(torch.sum(h ** 2, -1, keepdim=True) / case["cols"] + s["eps"])
        n = h / root * (s["weight"].double() + case["offset"])
        if case["norm_out"]:
            out["norm"] = n
        if case["quant"] != "none":
            out.update(_exact_codes(n, case["quant"]))
        return out
    if case["op"] == "act":
        gate, up = s["x"].double().chunk(2, -1)
        if case["gelu"]:
            gate = gate * 0.5 * torch.erfc(-gate / math.sqrt(2))
        else:
            gate = gate * torch.sigmoid(gate)
        return _exact_codes(gate * up, case["quant"])
    m, n, k = case["m"], case["n"], case["k"]
    a, w = s["a"].double(), s["w"].double()
    for b in range((k + 127) // 128):
        at = slice(128 * b, min(k, 128 * b + 128))
        a[:, at] *= s["a_scale"][:, b:b + 1].double()
        w[:, at] *= s["w_scale"][torch.arange(n, device=w.device) // 128, b].double()[:, None]
    out = torch.matmul(a, w.t())
    return out if s["bias"] is None else out + s["bias"].double()
