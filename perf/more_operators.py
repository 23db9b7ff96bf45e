"""Cases of the steps of a routed layer, with their gradients: the router's
weights (``fused_topk``), tokens sorted by expert and back (``moe_permute``,
``moe_unpermute``), and the products in between and beside them with bias,
activation and residual in the epilogue (``grouped_linear`` of the experts,
``fused_linear`` of the shared expert and the projections).

Serving takes them forward, from a token to chunks of thousands; training takes
each with its gradients. Sizes are those of the layers in
``flaggems_sglang.testing.CONFIGS`` and odd ones about them.
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


# ------------------------------------------------------------------ cases ---
def _router(name, m, experts, topk, **more):
    case = dict(name=name, op="router", dtype="fp32", m=m, experts=experts, topk=topk,
                scoring="softmax", renormalize=True)
    case.update(more)
    return case


def _move(name, op, m, cols, experts, topk, **more):
    """``dropped``: the share of slots that other GPUs' experts have."""
    case = dict(name=name, op=op, dtype="bf16", m=m, cols=cols, experts=experts, topk=topk,
                dropped=0.0, train=False)
    case.update(more)
    return case


def _product(name, m, n, k, **more):
    """``experts`` 0: one matrix; else ``m`` rows sorted by expert, of which
    ``behind`` belong to none. A gated product has 2n weight rows."""
    case = dict(name=name, op="product", dtype="bf16", m=m, n=n, k=k, experts=0, act="none",
                gated=False, bias=False, residual=False, train=False, behind=0)
    case.update(more)
    return case


def listed():
    return [
        # the router of a small batch, and of a training step's tokens; both with
        # the weights' gradient
        _router("router_batch", 61, 256, 8, scoring="sigmoid"),
        _router("router_train", 8192, 128, 8),
        # one token's rows for its experts' GPUs (latency); a training step's
        # tokens sorted by expert, with the gradient's way back
        _move("permute_decode", "permute", 1, 7168, 256, 8),
        _move("permute_train", "permute", 8192, 2048, 128, 8, train=True),
        # a decode batch's results back in token order; an odd chunk of a GPU
        # that has three quarters of the experts, trained
        _move("unpermute_decode", "unpermute", 16, 4096, 8, 2),
        _move("unpermute_train", "unpermute", 4093, 7168, 256, 8, dropped=0.25, train=True),
        # one token through an output projection, onto the residual stream
        _product("linear_decode", 1, 4096, 4096, residual=True),
        # a layer whose sizes end inside every tile, trained
        _product("linear_ragged", 333, 2112, 1552, dtype="fp16", act="gelu", bias=True,
                 residual=True, train=True),
        # the gate and up product of a wide dense layer over a training step
        _product("linear_train", 8192, 14336, 4096, act="silu", gated=True, train=True),
        # the gate and up products of a decode batch's experts: the weights' bytes
        _product("experts_decode", 128, 768, 2048, experts=128, act="silu", gated=True),
        # the down products of a prefill chunk
        _product("experts_prefill", 8192, 4096, 14336, experts=8),
        # many small experts over a training step
        _product("experts_train", 65536, 768, 2048, experts=128, act="silu", gated=True,
                 train=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_LARGEST = 3 * 2 * 8192 * 2 * 14336 * 4096


def draw(rng):
    op = rng.choice(["router", "permute", "unpermute", "product", "product", "product"])
    experts = rng.choice([8, 16, 61, 64, 128, 256])
    if op == "router":
        case = _router("", _log_int(rng, 1, 8192), experts, rng.choice([1, 2, 4, 8]),
                       dtype=rng.choice(["fp32", "fp32", "bf16"]),
                       scoring=rng.choice(["softmax", "softmax", "sigmoid"]),
                       renormalize=rng.random() < 0.6)
    elif op != "product":
        step = rng.choice([1, 8, 128])  # odd sizes, whole vectors
        cols = max(step, _log_int(rng, 64, 7168) // step * step)
        m, topk = _log_int(rng, 1, 8192), rng.choice([1, 2, 5, 8])
        while m * topk * cols > 8192 * 8 * 4096:
            m //= 2
        case = _move("", op, m, cols, experts, topk,
                     dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                     dropped=rng.choice([0.0, 0.0, 0.5]), train=rng.random() < 0.5)
    else:
        grouped = rng.random() < 0.5
        m = _log_int(rng, 1, 16384)
        n, k = 8 * _log_int(rng, 8, 1024), 8 * _log_int(rng, 8, 1024)
        if rng.random() < 0.5:  # whole tiles about half of the time
            n, k = max(128, n // 128 * 128), max(128, k // 128 * 128)
        gated, train = rng.random() < 0.4, rng.random() < 0.5
        experts = experts if grouped else 0
        while experts > 8 and experts * n * k > 1 << 28:
            experts //= 2
        while m * n * k * (1 + gated) * (1 + 2 * train) * 2 > _LARGEST:
            m = max(1, m // 2)
        act = rng.choice(["silu", "gelu"] if gated else ["none", "none", "relu", "silu", "gelu"])
        case = _product("", m, n, k, experts=experts, act=act, gated=gated, train=train,
                        bias=rng.random() < 0.4, residual=rng.random() < 0.4,
                        dtype=rng.choice(["bf16", "bf16", "fp16"]),
                        behind=m // 3 if grouped and rng.random() < 0.3 else 0)
    del case["name"]
    return case


# ----------------------------------------------------------------- inputs ---
def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _activations(rows, cols, gen, dtype):
    """Rows of a hidden state: token norms that differ, a few loud channels."""
    x = _randn(gen, rows, cols)
    loud = torch.rand(cols, generator=gen, device="cuda") < 0.01
    x *= torch.where(loud, 4.0, 1.0)
    x *= 0.5 + torch.rand(rows, 1, generator=gen, device="cuda")
    return x.to(dtype)


def _logits(m, experts, gen):
    """A router's: some experts are liked by most tokens."""
    return _randn(gen, m, experts) + 0.5 * _randn(gen, experts)


def _ids(case, gen):
    ids = torch.topk(_logits(case["m"], case["experts"], gen), case["topk"], dim=1).indices
    ids = ids.to(torch.int32)
    if case["dropped"]:
        here = torch.rand(ids.shape, generator=gen, device="cuda") >= case["dropped"]
        ids = torch.where(here, ids, -1)
    return ids


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    s = {"case": dict(case)}
    train = case.get("train", True)

    def leaf(t):
        return t.requires_grad_() if train else t

    if case["op"] == "router":
        m = case["m"]
        s["logits"] = leaf(_logits(m, case["experts"], gen).to(dtype))
        s["hidden"] = torch.empty(m, 8, dtype=torch.bfloat16, device="cuda")
        s["dweights"] = _randn(gen, m, case["topk"])
    elif case["op"] == "permute":
        m, topk, cols = case["m"], case["topk"], case["cols"]
        s["ids"] = _ids(case, gen)
        s["x"] = leaf(_activations(m, cols, gen, dtype))
        if train:
            s["drows"] = _randn(gen, m * topk, cols).to(dtype)
    elif case["op"] == "unpermute":
        m, topk, cols = case["m"], case["topk"], case["cols"]
        s["ids"] = _ids(case, gen)
        # the order that sorting the tokens left
        if own:
            s["order"] = _fgs().moe_permute(torch.zeros(m, 8, device="cuda"), s["ids"],
                                            case["experts"])[1]
        else:
            s["order"] = _sorted(s["ids"], case["experts"])
        s["rows"] = leaf(_activations(m * topk, cols, gen, dtype))
        s["weights"] = leaf(torch.softmax(_randn(gen, m, topk), 1))
        if train:
            s["dout"] = _randn(gen, m, cols).to(dtype)
    else:
        m, n, k = case["m"], case["n"], case["k"]
        rows = n * (1 + case["gated"])
        s["x"] = leaf(_activations(m, k, gen, dtype))
        shape = (case["experts"], rows) if case["experts"] else (rows,)
        w = torch.empty(*shape, k, dtype=dtype, device="cuda")
        for part in (w if case["experts"] else [w]):
            part.copy_(_randn(gen, rows, k) / math.sqrt(k))
        s["w"] = leaf(w)
        s["bias"] = leaf(_randn(gen, *shape).to(dtype)) if case["bias"] else None
        s["residual"] = leaf(_activations(m, n, gen, dtype)) if case["residual"] else None
        s["counts"], s["sizes"] = None, [m]
        if case["experts"]:
            here = m - case["behind"]
            share = torch.softmax(0.5 * _randn(gen, case["experts"]), 0)
            of = torch.multinomial(share, here, replacement=True, generator=gen)
            s["counts"] = torch.bincount(of, minlength=case["experts"]).to(torch.int32)
            s["sizes"] = s["counts"].tolist()
        if train:
            s["dout"] = _randn(gen, m, n).to(dtype)
    return s


# ------------------------------------------------------------------- runs ---
def _run_router(s):
    c = s["case"]
    topk, renormalize = c["topk"], c["renormalize"]
    if own:
        weights, ids = _fgs().fused_topk(s["hidden"], s["logits"], topk, renormalize, c["scoring"])
        grad, = torch.autograd.grad(weights, s["logits"], s["dweights"])
        return {"weights": weights.detach(), "ids": ids, "dlogits": grad}
    logits, d = s["logits"].detach().float(), s["dweights"]
    ids = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :topk]
    if c["scoring"] == "softmax":
        scores = torch.exp(logits - logits.amax(1, keepdim=True))
        scores = scores / scores.sum(1, keepdim=True)
    else:
        scores = 1 / (1 + torch.exp(-logits))
    weights = torch.gather(scores, 1, ids)
    total = weights.sum(1, keepdim=True)
    if renormalize:
        weights = weights / total
        d = (d - (d * weights).sum(1, keepdim=True)) / total
    dscores = torch.zeros_like(scores).scatter(1, ids, d)
    if c["scoring"] == "softmax":
        grad = scores * (dscores - (dscores * scores).sum(1, keepdim=True))
    else:
        grad = dscores * scores * (1 - scores)
    return {"weights": weights, "ids": ids.to(torch.int32), "dlogits": grad.to(s["logits"].dtype)}


def _sorted(ids, experts):
    """(rows per expert, each slot's row, each row's slot), slots that no expert
    here has last; -1 for those."""
    flat = ids.reshape(-1).long()
    group = torch.where((flat >= 0) & (flat < experts), flat, experts)
    slots = torch.sort(group, stable=True).indices
    rows = torch.empty_like(slots)
    rows[slots] = torch.arange(slots.numel(), device=ids.device)
    counts = torch.zeros(experts + 1, dtype=torch.int32, device=ids.device)
    counts.scatter_add_(0, group, torch.ones_like(group, dtype=torch.int32))
    kept = group < experts
    rows = torch.where(kept, rows, -1).to(torch.int32).view(ids.shape)
    slots = torch.where(kept[slots], slots, -1).to(torch.int32)
    return counts[:-1], rows, slots


def _run_permute(s):
    c = s["case"]
    topk = c["topk"]
    if own:
        rows, order = _fgs().moe_permute(s["x"], s["ids"], c["experts"])
        out = {"rows": rows.detach(), "counts": order.counts, "row_of_slot": order.row_of_slot,
               "slot_of_row": order.slot_of_row}
        if c["train"]:
            out["dx"], = torch.autograd.grad(rows, s["x"], s["drows"])
        return out
    x = s["x"].detach()
    counts, row_of_slot, slot_of_row = _sorted(s["ids"], c["experts"])
    kept = slot_of_row >= 0
    rows = torch.where(kept[:, None], x[slot_of_row.clamp(min=0) // topk], 0)
    out = {"rows": rows, "counts": counts, "row_of_slot": row_of_slot, "slot_of_row": slot_of_row}
    if c["train"]:
        dx = torch.zeros(x.shape, dtype=torch.float32, device=x.device)
        for j in range(topk):
            r = row_of_slot[:, j]
            dx += torch.where((r >= 0)[:, None], s["drows"][r.clamp(min=0)].float(), 0)
        out["dx"] = dx.to(x.dtype)
    return out


def _run_unpermute(s):
    c = s["case"]
    if own:
        out = _fgs().moe_unpermute(s["rows"], s["order"], s["weights"])
        if not c["train"]:
            return {"out": out}
        drows, dweights = torch.autograd.grad(out, (s["rows"], s["weights"]), s["dout"])
        return {"out": out.detach(), "drows": drows, "dweights": dweights}
    rows, weights = s["rows"].detach(), s["weights"].detach()
    _, row_of_slot, slot_of_row = s["order"]
    acc = torch.zeros(c["m"], c["cols"], dtype=torch.float32, device=rows.device)
    dweights = torch.zeros_like(weights)
    for j in range(c["topk"]):
        r = row_of_slot[:, j]
        part = torch.where((r >= 0)[:, None], rows[r.clamp(min=0)].float(), 0)
        acc += weights[:, j:j + 1] * part
        if c["train"]:
            dweights[:, j] = (part * s["dout"].float()).sum(1)
    if not c["train"]:
        return {"out": acc.to(rows.dtype)}
    slot = slot_of_row.clamp(min=0)
    drows = weights.reshape(-1)[slot][:, None] * s["dout"][slot // c["topk"]].float()
    drows = torch.where((slot_of_row >= 0)[:, None], drows, 0).to(rows.dtype)
    return {"out": acc.to(rows.dtype), "drows": drows, "dweights": dweights}


def _activate(z, act):
    """act(z) and its derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return torch.where(z > 0, z, 0), (z > 0).to(z.dtype)
    if act == "silu":
        e = 1 / (1 + torch.exp(-z))
        return z * e, e * (1 + z * (1 - e))
    cdf = 0.5 * torch.erfc(-z * math.sqrt(0.5))
    return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))


def _groups(s):
    """(row range, weights, bias) of each group of rows."""
    w = s["w"].detach()
    bias = None if s["bias"] is None else s["bias"].detach()
    if not s["case"]["experts"]:
        return [(slice(0, s["sizes"][0]), w, bias)]
    at, parts = 0, []
    for e, size in enumerate(s["sizes"]):
        parts.append((slice(at, at + size), w[e], None if bias is None else bias[e]))
        at += size
    return parts


def _run_product(s):
    c = s["case"]
    act = None if c["act"] == "none" else c["act"]
    x, w, bias, residual = s["x"], s["w"], s["bias"], s["residual"]
    names = [k for k in ("x", "w", "bias", "residual") if s[k] is not None]
    if own:
        options = dict(bias=bias, activation=act, gated=c["gated"], residual=residual)
        if c["experts"]:
            out = _fgs().grouped_linear(x, w, s["counts"], **options)
        else:
            out = _fgs().fused_linear(x, w, **options)
        if not c["train"]:
            return {"out": out}
        grads = torch.autograd.grad(out, [s[k] for k in names], s["dout"])
        return {"out": out.detach(), **{"d" + k: g for k, g in zip(names, grads)}}
    dtype, n = x.dtype, c["n"]
    x = x.detach()
    out = torch.zeros(c["m"], n, dtype=dtype, device=x.device)
    if residual is not None:
        out.copy_(residual.detach())
    r = {"out": out}
    if c["train"]:
        r["dx"], r["dw"] = torch.zeros_like(x), torch.zeros_like(w, requires_grad=False)
        if bias is not None:
            r["dbias"] = torch.zeros_like(bias, requires_grad=False)
        if residual is not None:
            r["dresidual"] = s["dout"]
    for e, (rows, we, be) in enumerate(_groups(s)):
        if rows.start == rows.stop:
            continue
        xe, we = x[rows].float(), we.float()
        z = xe @ we.t()
        if be is not None:
            z = z + be.float()
        if c["gated"]:
            a, slope = _activate(z[:, :n], c["act"])
            y = a * z[:, n:]
        else:
            y, slope = _activate(z, c["act"])
        if residual is not None:
            y = y + residual[rows].detach().float()
        out[rows] = y.to(dtype)
        if not c["train"]:
            continue
        d = s["dout"][rows].float()
        dz = torch.cat([d * z[:, n:] * slope, d * a], 1) if c["gated"] else d * slope
        r["dx"][rows] = (dz @ we).to(dtype)
        dw = (dz.t() @ xe).to(dtype)
        db = dz.sum(0).to(dtype)
        if c["experts"]:
            r["dw"][e] = dw
            if bias is not None:
                r["dbias"][e] = db
        else:
            r["dw"] = dw
            if bias is not None:
                r["dbias"] = db
    return r


def run(s):
    return {"router": _run_router, "permute": _run_permute, "unpermute": _run_unpermute,
            "product": _run_product}[s["case"]["op"]](s)


# ------------------------------------------------------------------- work ---
def work(case):
    size = _TYPES[case["dtype"]].itemsize
    if case["op"] == "router":
        values, slots = case["m"] * case["experts"], case["m"] * case["topk"]
        return {"bytes": 2 * size * values + 12 * slots, "flops": 8 * values + 8 * slots}
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        wide, groups = n * (1 + case["gated"]), max(1, case["experts"])
        used = min(groups, m - case["behind"])  # experts that have rows
        weights = wide * k + case["bias"] * wide
        moved = m * k + used * weights + m * n * (1 + case["residual"])
        if case["train"]:
            moved += m * k + groups * weights + m * n * (1 + case["residual"])
        rows = m - case["behind"]
        return {"bytes": size * moved + 4 * case["experts"],
                "flops": 2 * rows * wide * k * (3 if case["train"] else 1)}
    m, cols, slots = case["m"], case["cols"], case["m"] * case["topk"]
    kept = int(slots * (1 - case["dropped"]))
    if case["op"] == "permute":
        moved = m * cols + slots * cols + (kept * cols + m * cols if case["train"] else 0)
        return {"bytes": size * moved + 12 * slots + 4 * case["experts"],
                "flops": kept * cols if case["train"] else 0}
    moved = kept * cols + m * cols + (slots * cols + m * cols if case["train"] else 0)
    return {"bytes": size * moved + 8 * slots + (8 * slots if case["train"] else 0),
            "flops": kept * cols * (5 if case["train"] else 2)}


# ------------------------------------------------------------------ exact ---
def _exact_router(s, c):
    logits = s["logits"].detach().double().requires_grad_()
    ids = torch.sort(logits.detach(), dim=1, descending=True, stable=True).indices[:, :c["topk"]]
    scores = logits.softmax(1) if c["scoring"] == "softmax" else logits.sigmoid()
    weights = scores.gather(1, ids)
    if c["renormalize"]:
        weights = weights / weights.sum(1, keepdim=True)
    weights.backward(s["dweights"].double())
    return {"weights": weights.detach(), "ids": ids.to(torch.int32), "dlogits": logits.grad}


def _exact_order(c, ids):
    """By expert, then by slot: one list a group."""
    flat = ids.reshape(-1).cpu()
    slots = torch.cat([torch.nonzero(flat == e)[:, 0] for e in range(c["experts"])])
    row_of_slot = torch.full((flat.numel(),), -1, dtype=torch.int32)
    row_of_slot[slots] = torch.arange(slots.numel(), dtype=torch.int32)
    slot_of_row = torch.full((flat.numel(),), -1, dtype=torch.int32)
    slot_of_row[:slots.numel()] = slots.to(torch.int32)
    counts = torch.tensor([int((flat == e).sum()) for e in range(c["experts"])],
                          dtype=torch.int32)
    return counts.cuda(), row_of_slot.view(ids.shape).cuda(), slot_of_row.cuda()


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "router":
        return _exact_router(s, c)
    if c["op"] == "product":
        return _exact_product(s, c)
    counts, row_of_slot, slot_of_row = _exact_order(c, s["ids"])
    used = row_of_slot.reshape(-1) >= 0
    slots = torch.nonzero(used)[:, 0]          # the kept slots,
    at = row_of_slot.reshape(-1)[slots].long()  # their rows
    token = slots // c["topk"]                  # and tokens
    total = c["m"] * c["topk"]
    if c["op"] == "permute":
        rows = torch.zeros(total, c["cols"], dtype=torch.float64, device="cuda")
        rows[at] = s["x"].detach().double()[token]
        out = {"rows": rows, "counts": counts, "row_of_slot": row_of_slot,
               "slot_of_row": slot_of_row}
        if c["train"]:
            dx = torch.zeros(c["m"], c["cols"], dtype=torch.float64, device="cuda")
            out["dx"] = dx.index_add_(0, token, s["drows"].double()[at])
        return out
    weights = s["weights"].detach().double().reshape(-1)[slots, None]
    rows = s["rows"].detach().double()
    out = torch.zeros(c["m"], c["cols"], dtype=torch.float64, device="cuda")
    out.index_add_(0, token, weights * rows[at])
    if not c["train"]:
        return {"out": out}
    dout = s["dout"].double()
    drows = torch.zeros_like(rows)
    drows[at] = weights * dout[token]
    dweights = torch.zeros(total, dtype=torch.float64, device="cuda")
    dweights[slots] = torch.linalg.vecdot(rows[at], dout[token])
    return {"out": out, "drows": drows, "dweights": dweights.view(c["m"], c["topk"])}


def _exact_product(s, c):
    def wide(t):
        return None if t is None else t.detach().double().requires_grad_(c["train"])

    acts = {"none": lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu,
            "gelu": torch.nn.functional.gelu}
    many = c["experts"] > 0
    x, residual = wide(s["x"]), wide(s["residual"])
    # a group at a time, so that only its weights are held in 64 bits
    out = torch.zeros(c["m"], c["n"], dtype=torch.float64, device="cuda")
    dw, db, at = [], [], 0
    for e, size in enumerate(s["sizes"]):
        w = wide(s["w"][e] if many else s["w"])
        b = None if s["bias"] is None else wide(s["bias"][e] if many else s["bias"])
        z = torch.matmul(x[at:at + size], w.transpose(0, 1))
        z = z if b is None else z + b
        if c["gated"]:
            gate, up = z.chunk(2, 1)
            y = acts[c["act"]](gate) * up
        else:
            y = acts[c["act"]](z)
        out[at:at + size] = y.detach()
        if c["train"]:
            y.backward(s["dout"][at:at + size].double())
            dw.append(w.grad)
            if b is not None:
                db.append(b.grad)
        at += size
    if residual is not None:
        out += residual.detach()
    r = {"out": out}
    if c["train"]:
        r["dx"] = x.grad
        r["dw"] = torch.stack(dw) if many else dw[0]
        if db:
            r["dbias"] = torch.stack(db) if many else db[0]
        if residual is not None:
            r["dresidual"] = s["dout"].double()
    return r
