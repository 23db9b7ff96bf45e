"""Plain forms in 64 bits of the routed layer's steps and their gradients, with
bounds on how far a kernel may be off that follow from the operators' definitions:

* h: half a step of the output's type, once for each rounding;
* a sum of n products in fp32: each of at most n additions is off by 2^-24 of a
  partial sum, which is at most the sum of the magnitudes;
* what is kept between the passes is off by its own rounding (z in fp32, dz by h), and
  that passes on through the derivative of what is taken of it.
"""

import math

import torch

F32 = 2.0 ** -24
# |act'| <= 1.13, and |act''| at most (silu 1/2, gelu 2 phi(0) = 0.798, relu 0)
SLOPE = 1.13
CURVE = {None: 0.0, "relu": 0.0, "silu": 0.5, "gelu": 0.8}


def half(dtype):
    return torch.finfo(dtype).eps / 2


def act(z, kind):
    """(act(z), act'(z)) in 64 bits."""
    if kind is None:
        return z, torch.ones_like(z)
    if kind == "relu":
        return z.clamp(min=0), (z > 0).double()
    if kind == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    phi = 0.5 * torch.erfc(-z / math.sqrt(2))
    return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def product(x, w, bias=None, kind=None, gated=False, residual=None, dout=None):
    """{name: (value, bound)} of one group: out and, with dout, dx, dw, dbias,
    dresidual."""
    h = half(x.dtype)
    x, w = x.double(), w.double()
    rows, k = x.shape
    n = w.shape[0] // (2 if gated else 1)
    z = x @ w.t()
    zmag = x.abs() @ w.abs().t()
    if bias is not None:
        z = z + bias.double()
        zmag = zmag + bias.double().abs()
    ez = (k + 1) * F32 * zmag
    # the activation's own steps: fp32 exp, reciprocal and products, whose
    # arguments (at most 90 in magnitude before exp leaves fp32) are off by 2^-24
    fn = 0.0 if kind in (None, "relu") else 2.0 ** -16
    if gated:
        a, slope = act(z[:, :n], kind)
        u = z[:, n:]
        y = a * u
        ey = u.abs() * (SLOPE * ez[:, :n] + fn * a.abs()) + a.abs() * ez[:, n:] + 2 * F32 * y.abs()
    else:
        y, slope = act(z, kind)
        ey = (SLOPE if kind else 1) * ez + fn * y.abs()
    if residual is not None:
        y = y + residual.double()
        ey = ey + F32 * y.abs()
    out = {"out": (y, ey + h * y.abs() + tiny(x, h))}
    if dout is None:
        return out
    d = dout.double()
    # z is kept in fp32: the slope is taken there, off by what |act''| makes of it
    if gated:
        zg, zu = F32 * z[:, :n].abs() + ez[:, :n], F32 * u.abs() + ez[:, n:]
        dz = torch.cat([d * u * slope, d * a], 1)
        e = torch.cat([d.abs() * (zu * (SLOPE + CURVE[kind] * zg) + u.abs() * CURVE[kind] * zg),
                       d.abs() * SLOPE * zg], 1)
        e = e + fn * torch.cat([d.abs() * u.abs() * SLOPE, d.abs() * (a.abs() + 1)], 1)
        e = e + h * (dz.abs() + e)
    elif kind:
        dz = d * slope
        e = d.abs() * (CURVE[kind] * (F32 * z.abs() + ez) + fn * SLOPE)
        e = e + h * (dz.abs() + e)
    else:
        dz, e = d, torch.zeros_like(d)
    m = dz.abs() + e
    wide = w.shape[0]

    def bound(value, passed, mag, length):
        b = passed + (length + 1) * F32 * mag
        return value, b + h * (value.abs() + b) + tiny(x, h)

    out["dx"] = bound(dz @ w, e @ w.abs(), m @ w.abs(), wide)
    out["dw"] = bound(dz.t() @ x, e.t() @ x.abs(), m.t() @ x.abs(), rows)
    if bias is not None:
        out["dbias"] = bound(dz.sum(0), e.sum(0), m.sum(0), rows)
    if residual is not None:
        out["dresidual"] = d, torch.zeros_like(d)
    return out


def tiny(x, h):
    """Half the smallest step of a 16-bit type (fp16's subnormals; bf16's are
    fp32's)."""
    return 2.0 ** -25 if h == 2.0 ** -11 else 2.0 ** -134


def grouped(x, w, counts, bias=None, kind=None, gated=False, residual=None, dout=None):
    """The same for rows sorted by group."""
    rows, n = x.shape[0], w.shape[1] // (2 if gated else 1)
    dev, f = x.device, torch.float64

    def none(*shape):
        return torch.zeros(*shape, dtype=f, device=dev), torch.zeros(*shape, dtype=f, device=dev)

    names = {"out": none(rows, n)}
    if residual is not None:
        names["out"] = residual.double(), names["out"][1]
    if dout is not None:
        names.update(dx=none(*x.shape), dw=none(*w.shape))
        if bias is not None:
            names["dbias"] = none(*bias.shape)
        if residual is not None:
            names["dresidual"] = dout.double(), none(rows, n)[1]
    at = 0
    for e, c in enumerate(counts):
        c = min(max(int(c), 0), rows - at)
        if c == 0:
            continue
        s = slice(at, at + c)
        at += c
        one = product(x[s], w[e], None if bias is None else bias[e], kind, gated,
                      None if residual is None else residual[s], None if dout is None else dout[s])
        for name, pair in one.items():
            for whole, part in zip(names[name], pair):
                if name in ("dw", "dbias"):
                    whole[e] = part
                else:
                    whole[s] = part
    return names


def order(ids, experts):
    """(counts, row_of_slot, slot_of_row) of ids [tokens, topk], slot by slot."""
    flat = [int(i) for i in ids.reshape(-1).tolist()]
    slots = [s for e in range(experts) for s, i in enumerate(flat) if i == e]
    counts = torch.zeros(experts, dtype=torch.int32)
    rows = torch.full((len(flat),), -1, dtype=torch.int32)
    back = torch.full((len(flat),), -1, dtype=torch.int32)
    for r, s in enumerate(slots):
        counts[flat[s]] += 1
        rows[s] = r
        back[r] = s
    return counts, rows.view(ids.shape), back


def close(what, got, value, bound):
    """Fails, and names the worst value, where one is off by more than its bound."""
    assert got.shape == value.shape, (what, got.shape, value.shape)
    off = (got.double() - value).abs()
    bad = ~(off <= bound)
    if bool(bad.any()):
        i = int(torch.where(bad, off / bound.clamp(min=1e-300), 0).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values are off, value {i}: "
                             f"{float(got.reshape(-1)[i])} for {float(value.reshape(-1)[i])} "
                             f"+- {float(bound.reshape(-1)[i])}")
