"""moe_permute, moe_unpermute and the gradient of fused_topk against plain forms in
64 bits, and the routed layer of these steps, on the GPU."""

import pytest
import torch

import flaggems_sglang as fgs
import steps_ref as ref
from flaggems_sglang import _capi

pytestmark = pytest.mark.gpu

F32 = ref.F32
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def generator(*numbers):
    return torch.Generator(device="cuda").manual_seed(sum(7 ** i * n for i, n in enumerate(numbers)))


def make_ids(gen, m, topk, experts, dropped=0.0):
    ids = torch.rand(m, max(experts, topk), generator=gen, device="cuda").argsort(1)[:, :topk] % experts
    ids = ids.to(torch.int32)
    out = torch.rand(m, topk, generator=gen, device="cuda") < dropped
    stray = torch.tensor([-1, experts, -2 ** 31, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    return torch.where(out, stray[torch.randint(4, (m, topk), generator=gen, device="cuda")], ids)


CASES = [(1, 1, 1, 1), (1, 7168, 256, 8), (3, 5, 7, 2), (64, 128, 8, 1), (65, 8, 16, 5),
         (37, 1001, 61, 8), (600, 40, 64, 8), (700, 24, 1022, 6), (1500, 16, 8, 3), (20, 2050, 4, 17)]


@pytest.mark.parametrize("dropped", [0.0, 0.4, 1.0])
@pytest.mark.parametrize("m, cols, experts, topk", CASES)
@pytest.mark.parametrize("dtype", TYPES)
def test_permute(gpu, dtype, m, cols, experts, topk, dropped):
    gen = generator(m, cols, experts, topk)
    ids = make_ids(gen, m, topk, experts, dropped)
    x = torch.randn(m, cols, generator=gen, device="cuda").to(TYPES[dtype]).requires_grad_()
    rows, order = fgs.moe_permute(x, ids, experts)
    counts, row_of_slot, slot_of_row = ref.order(ids, experts)
    assert torch.equal(order.counts.cpu(), counts)
    assert torch.equal(order.row_of_slot.cpu(), row_of_slot)
    assert torch.equal(order.slot_of_row.cpu(), slot_of_row)
    slots = slot_of_row.long().cuda()
    want = torch.where(slots[:, None] >= 0, x.detach()[slots.clamp(min=0) // topk], 0)
    assert torch.equal(rows.detach(), want)
    # the same rows by the order
    again, same = fgs.moe_permute(x, order=order)
    assert same is order and torch.equal(again.detach(), want)

    drows = torch.randn(m * topk, cols, generator=gen, device="cuda").to(TYPES[dtype])
    drows[int(counts.sum()):] = float("nan")  # (rows of no slot)
    value = torch.zeros(m, cols, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(value)
    for k in range(topk):
        r = row_of_slot[:, k].long().cuda()
        part = torch.where(r[:, None] >= 0, drows.double()[r.clamp(min=0)], 0)
        value += part
        mag += part.abs()
    bound = topk * F32 * mag
    bound = bound + ref.half(TYPES[dtype]) * (value.abs() + bound) + ref.tiny(x, ref.half(TYPES[dtype]))
    for out in (rows, again):
        dx, = torch.autograd.grad(out, x, drows)
        ref.close("dx", dx, value, bound)


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float8_e5m2, torch.int8, torch.uint8,
                                   torch.int32, torch.int64])
def test_permute_other_types(gpu, dtype):
    gen = generator(5)
    ids = make_ids(gen, 90, 4, 16, 0.2)
    for cols in (1, 3, 17, 256):
        x = (60 * torch.randn(90, cols, generator=gen, device="cuda")).to(dtype)
        rows, order = fgs.moe_permute(x, ids, 16)
        slots = order.slot_of_row.long()
        raw, got = x.view(torch.uint8), rows.view(torch.uint8)
        assert torch.equal(got, torch.where(slots[:, None] >= 0, raw[slots.clamp(min=0) // 4], 0))


@pytest.mark.parametrize("slots", [1, 2, 63, 64, 65])
@pytest.mark.parametrize("experts", [1, 8, 1022])
def test_permute_few_slots(gpu, slots, experts):
    """Up to 64 slots and one more: all of one expert, of none, of the first and the
    last; rows of 1 to 33 bytes and of several workgroups."""
    gen = generator(slots, experts)
    first_last = torch.arange(slots, dtype=torch.int32, device="cuda") % 2 * (experts - 1)
    stray = torch.where(first_last == 0, first_last, experts)
    for flat in (torch.zeros_like(first_last), torch.full_like(first_last, -1), first_last, stray):
        for topk in {1, slots}:
            ids = flat.view(-1, topk)
            counts, row_of_slot, slot_of_row = ref.order(ids, experts)
            at = slot_of_row.long().cuda()
            for cols in (1, 2, 3, 4, 7, 15, 16, 17, 33, 9001):
                x = torch.randint(256, (ids.shape[0], cols), generator=gen, device="cuda").byte()
                rows, order = fgs.moe_permute(x, ids, experts)
                assert torch.equal(order.counts.cpu(), counts)
                assert torch.equal(order.row_of_slot.cpu(), row_of_slot)
                assert torch.equal(order.slot_of_row.cpu(), slot_of_row)
                assert torch.equal(rows, torch.where(at[:, None] >= 0, x[at.clamp(min=0) // topk], 0))


def test_permute_ids_of_64_bits_and_strides(gpu):
    gen = generator(6)
    ids = make_ids(gen, 50, 3, 10, 0.3)
    x = torch.randn(50, 70, generator=gen, device="cuda").bfloat16()
    want, order = fgs.moe_permute(x[:, 1:66], ids, 10)
    far = ids.long()
    far[ids < 0] = 2 ** 32 + 3  # outside, though not in 32 bits
    for i in (far, ids.t().contiguous().t()):
        rows, again = fgs.moe_permute(x[:, 1:66].contiguous(), i, 10)
        assert torch.equal(rows, want) and all(torch.equal(a, b) for a, b in zip(order, again))
    rows, _ = fgs.moe_permute(x.t()[:50], ids, 10)  # columns that lie apart
    assert torch.equal(rows, fgs.moe_permute(x.t()[:50].contiguous(), ids, 10)[0])


@pytest.mark.parametrize("dropped", [0.0, 0.4, 1.0])
@pytest.mark.parametrize("m, cols, experts, topk", CASES)
@pytest.mark.parametrize("dtype", TYPES)
def test_unpermute(gpu, dtype, m, cols, experts, topk, dropped):
    gen = generator(m, cols, experts, topk)
    t = TYPES[dtype]
    h = ref.half(t)
    ids = make_ids(gen, m, topk, experts, dropped)
    _, order = fgs.moe_permute(torch.zeros(m, 1, device="cuda"), ids, experts)
    rows = torch.randn(m * topk, cols, generator=gen, device="cuda").to(t)
    rows[int(order.counts.sum()):] = float("nan")  # (rows of no slot)
    weights = torch.rand(m, topk, generator=gen, device="cuda")
    weights[order.row_of_slot < 0] = float("inf")  # (slots of no row)
    dout = torch.randn(m, cols, generator=gen, device="cuda").to(t)
    rows.requires_grad_()
    weights.requires_grad_()
    out = fgs.moe_unpermute(rows, order, weights)
    drows, dweights = torch.autograd.grad(out, (rows, weights), dout)

    r = order.row_of_slot.long()
    kept = (r >= 0)[..., None]
    parts = torch.where(kept, rows.detach().double()[r.clamp(min=0)], 0)  # [m, topk, cols]
    w = torch.where(kept, weights.detach().double()[..., None], 0)
    value, mag = (w * parts).sum(1), (w * parts).abs().sum(1)
    bound = topk * F32 * mag
    ref.close("out", out.detach(), value, bound + h * (value.abs() + bound) + ref.tiny(rows, h))
    value = (parts * dout.double()[:, None]).sum(2)
    mag = (parts * dout.double()[:, None]).abs().sum(2)
    ref.close("dweights", dweights, value, (cols + 1) * F32 * mag)
    want = torch.zeros(m * topk, cols, dtype=torch.float64, device="cuda")
    want[r[r >= 0]] = (w * dout.double()[:, None])[r >= 0]
    bound = (F32 + h + F32 * h) * want.abs() + ref.tiny(rows, h)
    ref.close("drows", drows, want, bound)

    # ones for weights; a gradient of one alone
    plain = fgs.moe_unpermute(rows, order)
    ones = fgs.moe_unpermute(rows, order, torch.ones_like(weights))
    assert torch.equal(plain.detach(), ones.detach())
    d1, = torch.autograd.grad(plain, rows, dout)
    d2, = torch.autograd.grad(ones, rows, dout)
    assert torch.equal(d1, d2)
    only, = torch.autograd.grad(fgs.moe_unpermute(rows.detach(), order, weights), weights, dout)
    assert torch.equal(only, dweights)


def test_unpermute_rows_out_of_range(gpu):
    """An order's rows are looked at: those outside add nothing."""
    rows = torch.ones(8, 24, device="cuda", dtype=torch.bfloat16)
    at = torch.tensor([[0, 8], [-3, 7], [2 ** 31 - 1, -2 ** 31], [1, 1]], dtype=torch.int32, device="cuda")
    order = fgs.moe_permute(rows[:4], torch.zeros_like(at), 1)[1]._replace(row_of_slot=at)
    out = fgs.moe_unpermute(rows, order)
    assert out[:, 0].tolist() == [1, 1, 0, 2]


def test_weights_of_other_types(gpu):
    gen = generator(8)
    ids = make_ids(gen, 30, 4, 8)
    _, order = fgs.moe_permute(torch.zeros(30, 1, device="cuda"), ids, 8)
    rows = torch.randn(120, 40, generator=gen, device="cuda").bfloat16()
    w = torch.rand(30, 4, generator=gen, device="cuda").bfloat16().requires_grad_()
    out = fgs.moe_unpermute(rows, order, w)
    assert torch.equal(out, fgs.moe_unpermute(rows, order, w.detach().float()))
    g, = torch.autograd.grad(out.float().sum(), w)
    assert g.dtype == torch.bfloat16 and g.shape == w.shape


def test_no_tokens(gpu):
    x = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    rows, order = fgs.moe_permute(x, torch.empty(0, 4, dtype=torch.int32, device="cuda"), 9)
    assert rows.shape == (0, 64) and order.counts.tolist() == [0] * 9
    w = torch.empty(0, 4, device="cuda", requires_grad=True)
    out = fgs.moe_unpermute(rows, order, w)
    dx, dw = torch.autograd.grad(out, (x, w), torch.empty_like(out))
    assert out.shape == dx.shape == (0, 64) and dw.shape == (0, 4)


# ----------------------------------------------------------------- router ---
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("m, experts, topk", [(1, 1, 1), (1, 8, 2), (7, 64, 8), (300, 61, 4), (33, 256, 8),
                                              (5, 1000, 64), (9, 5, 5)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32", "fp16"])
def test_router_gradient(gpu, dtype, m, experts, topk, scoring, renormalize):
    gen = generator(m, experts, topk)
    logits = (2 * torch.randn(m, experts, generator=gen, device="cuda")).to(TYPES[dtype])
    logits.requires_grad_()
    d = torch.randn(m, topk, generator=gen, device="cuda")
    weights, ids = fgs.fused_topk(torch.empty(m, 1, device="cuda"), logits, topk, renormalize, scoring)
    assert not ids.requires_grad
    got, = torch.autograd.grad(weights, logits, d)
    with torch.no_grad():  # what a call without gradients returns
        w2, ids2 = fgs.fused_topk(torch.empty(m, 1, device="cuda"), logits, topk, renormalize, scoring)
    assert torch.equal(weights, w2) and torch.equal(ids, ids2)

    x = logits.detach().double().requires_grad_()
    score = x.softmax(1) if scoring == "softmax" else x.sigmoid()
    picked = score.gather(1, ids.long())
    w = picked / picked.sum(1, keepdim=True) if renormalize else picked
    want, = torch.autograd.grad(w, x, d.double())
    # weights are off by at most 2^-17 of themselves (exp of arguments up to 16, two
    # sums of up to 1000 terms of one sign, a quotient); the gradient is a product of
    # two or three of them with differences of d, each term's error a few of these
    w = w.detach()
    mean = (d.double() * w).abs().sum(1, keepdim=True)
    mag = torch.zeros_like(want).scatter(1, ids.long(), w * (d.double().abs() + mean))
    if scoring == "softmax" and not renormalize:
        mag += score.detach() * mean
    # (the 64-bit form's own roundings: where the picks' sum cancels, an expert that was
    # not picked has 0, and there it has a few 2^-53 of the terms that cancel)
    terms = score.detach() * d.double().abs().sum(1, keepdim=True)
    terms = terms / picked.detach().sum(1, keepdim=True) if renormalize else terms
    h = ref.half(TYPES[dtype])
    bound = 2.0 ** -14 * mag + 2.0 ** -48 * terms
    ref.close("dlogits", got, want, bound + h * (want.abs() + bound) + ref.tiny(logits, h))


@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_router_gradient_of_masked_experts(gpu, scoring, renormalize):
    """Experts masked with -inf or the type's lowest value, fewer left than are picked,
    have gradients of 0; a NaN stays in its token's row."""
    gen = generator(11)
    logits = torch.randn(6, 70, generator=gen, device="cuda")
    logits[1, 5:] = float("-inf")
    logits[2, 3:] = torch.finfo(torch.float32).min
    logits[3, 17] = float("nan")
    logits.requires_grad_()
    d = torch.randn(6, 8, generator=gen, device="cuda")
    weights, _ = fgs.fused_topk(torch.empty(6, 1, device="cuda"), logits, 8, renormalize, scoring)
    got, = torch.autograd.grad(weights, logits, d)
    assert not bool(got[1, 5:].any()) and not bool(got[2, 3:].any())
    rows = [0, 1, 2, 4, 5]
    assert bool(got[rows].isfinite().all()) and bool(got[1, :5].any()) and bool(got[2, :3].any())
    again = logits.detach()[rows].requires_grad_()
    weights, _ = fgs.fused_topk(torch.empty(5, 1, device="cuda"), again, 8, renormalize, scoring)
    assert torch.equal(torch.autograd.grad(weights, again, d[rows])[0], got[rows])


def test_router_gradient_of_ids_that_are_none(gpu):
    """The C entry: an id outside the experts has no gradient and reads nothing."""
    gen = generator(12)
    logits = torch.randn(4, 16, generator=gen, device="cuda")
    w, d = torch.rand(2, 4, 2, generator=gen, device="cuda")
    ids = torch.tensor([[0, -1], [16, 5], [-2 ** 31, 2 ** 31 - 1], [3, 15]], dtype=torch.int32, device="cuda")
    lib = _capi.load()
    for scoring in (0, 1):
        for renormalize in (0, 1):
            out = torch.full_like(logits, float("nan"))
            rc = lib.fgs_moe_topk_gating_grad(
                logits.data_ptr(), 0, 4, 16, 2, scoring, renormalize, w.data_ptr(), ids.data_ptr(),
                d.data_ptr(), out.data_ptr(), torch.cuda.current_stream().cuda_stream)
            assert rc == 0 and bool(out.isfinite().all()) and not bool(out[2].any())


# ------------------------------------------------------------------ layer ---
@pytest.mark.parametrize("m, k, n, experts, topk", [(1, 128, 64, 8, 2), (33, 256, 136, 16, 4),
                                                   (300, 264, 72, 61, 8), (520, 512, 264, 8, 2)])
@pytest.mark.parametrize("graph", [False, True])
def test_routed_layer(gpu, m, k, n, experts, topk, graph):
    """A routed layer of the steps, trained: outputs and gradients against the same
    layer in 64 bits on the same picks. Every step's output and gradient is rounded
    to bf16 between the steps, h each; the bound counts the roundings on the longest
    way (forward: x in; h, y, out rounded: backward: z, dz, dh, dy, drows, dx and the
    forward values that they meet) at the magnitudes of the terms, in the norm over a
    tensor: independent roundings add up to at most their number."""
    gen = generator(m, k, n, experts)

    def leaf(*shape, scale=1.0, dtype=torch.bfloat16):
        return (scale * torch.randn(*shape, generator=gen, device="cuda")).to(dtype).requires_grad_()

    x, logits = leaf(m, k), leaf(m, experts, dtype=torch.float32)
    w13, w2 = leaf(experts, 2 * n, k, scale=k ** -0.5), leaf(experts, k, n, scale=n ** -0.5)
    dout = torch.randn(m, k, generator=gen, device="cuda").bfloat16()
    leaves = [x, logits, w13, w2]

    def step():
        weights, ids = fgs.fused_topk(x, logits, topk)
        rows, order = fgs.moe_permute(x, ids, experts)
        h = fgs.grouped_linear(rows, w13, order.counts, activation="silu", gated=True)
        y = fgs.grouped_linear(h, w2, order.counts)
        out = fgs.moe_unpermute(y, order, weights)
        return (ids, out.detach(), *torch.autograd.grad(out, leaves, dout))

    if graph:
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step()
        torch.cuda.current_stream().wait_stream(stream)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            captured = step()
        for _ in range(3):
            with torch.no_grad():
                for t in leaves:
                    t.mul_(0.9)
            g.replay()
            torch.cuda.synchronize()
            got = [c.clone() for c in captured]
            for a, b in zip(got, step()):
                assert torch.equal(a, b)
    else:
        got = step()
    ids, out, *grads = got
    # with the layer's own forward call: the same products, rounded alike
    with torch.no_grad():
        weights, same = fgs.fused_topk(x, logits, topk)
    assert torch.equal(ids, same)

    d = [t.detach().double().requires_grad_() for t in leaves]
    p = d[1].softmax(1).gather(1, ids.long())
    p = p / p.sum(1, keepdim=True)
    want = torch.zeros(m, k, dtype=torch.float64, device="cuda")
    for e in range(experts):
        t, j = (ids == e).nonzero(as_tuple=True)
        z = d[0][t] @ d[2][e].t()
        y = (torch.nn.functional.silu(z[:, :n]) * z[:, n:]) @ d[3][e].t()
        want = want.index_add(0, t, p[t, j][:, None] * y)
    expect = [want.detach(), *torch.autograd.grad(want, d, dout.double())]
    h = 2.0 ** -8
    for name, a, b, roundings in zip(("out", "dx", "dlogits", "dw13", "dw2"), (out, *grads), expect,
                                     (3, 8, 5, 7, 5)):
        off = float((a.double() - b).norm())
        assert off <= roundings * h * float(b.norm()) + 1e-12, (name, off / float(b.norm()))


def test_matches_fused_moe(gpu):
    """The steps' forward pass against the layer's one call: both round the
    activation's output to bf16, the call its input too, so each value is within a
    few roundings at the terms' magnitude."""
    gen = generator(11)
    m, k, n, experts, topk = 200, 256, 128, 16, 4
    x = torch.randn(m, k, generator=gen, device="cuda").bfloat16()
    w13 = (torch.randn(experts, 2 * n, k, generator=gen, device="cuda") / 16).bfloat16()
    w2 = (torch.randn(experts, k, n, generator=gen, device="cuda") / 11).bfloat16()
    weights, ids = fgs.fused_topk(x, torch.randn(m, experts, generator=gen, device="cuda"), topk)
    rows, order = fgs.moe_permute(x, ids, experts)
    h = fgs.grouped_linear(rows, w13, order.counts, activation="silu", gated=True)
    out = fgs.moe_unpermute(fgs.grouped_linear(h, w2, order.counts), order, weights)
    whole = fgs.fused_moe(x, w13, w2, weights, ids)
    assert float((out.double() - whole.double()).norm()) <= 4 * 2.0 ** -8 * float(whole.double().norm())


# ---------------------------------------------------------- graphs, streams ---
def test_graph_of_permute_and_back(gpu):
    """Captured with dropped slots; every replay of new ids against the eager call."""
    gen = generator(21)
    m, topk, experts = 700, 8, 64  # (the alignment's counting kernels, with their scratch)
    x = torch.randn(m, 72, generator=gen, device="cuda").bfloat16()
    w = torch.rand(m, topk, generator=gen, device="cuda")
    ids = make_ids(gen, m, topk, experts, 0.3)

    def step():
        rows, order = fgs.moe_permute(x, ids, experts)
        again, _ = fgs.moe_permute(w, order=order)
        return rows, again, *order, fgs.moe_unpermute(rows, order, w)

    step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        captured = step()
    for i in range(4):
        ids.copy_(make_ids(gen, m, topk, experts, 0.25 * i))
        x.copy_(torch.randn(m, 72, generator=gen, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got = [c.clone() for c in captured]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_two_graphs_replay_side_by_side(gpu):
    """Each capture has its own workspaces."""
    gen = generator(22)
    sides = []
    for seed in (1, 2):
        x = torch.randn(5000, 64, generator=gen, device="cuda").bfloat16()
        ids = make_ids(gen, 5000, 2, 16)
        stream = torch.cuda.Stream()
        fgs.moe_permute(x, ids, 16)
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            rows, order = fgs.moe_permute(x, ids, 16)
        sides.append((graph, stream, rows, order, fgs.moe_permute(x, ids, 16), (x, ids)))
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, stream, *_ in sides:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, _, rows, order, (want, want_order), _ in sides:
            assert torch.equal(rows, want)
            assert all(torch.equal(a, b) for a, b in zip(order, want_order))


def test_capture_beside_an_eager_graph_is_refused(gpu):
    """A leaf whose eager graph, recorded on another stream, is still alive is refused
    while a stream is captured; without that graph it is taken."""
    x = torch.ones(4, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    w = torch.ones(32, 64, dtype=torch.bfloat16, device="cuda")
    alive = fgs.fused_linear(x, w)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        graph.capture_begin()
        try:
            with pytest.raises(RuntimeError, match="still alive"):
                fgs.fused_linear(x, w)
            out = fgs.fused_linear(x.detach(), w)
        finally:
            graph.capture_end()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, alive)
    del alive
    with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):
        out = fgs.fused_linear(x, w)
        torch.autograd.grad(out, x, torch.ones_like(out))


def test_steps_on_another_stream(gpu):
    gen = generator(23)
    x = torch.randn(900, 136, generator=gen, device="cuda").bfloat16()
    ids = make_ids(gen, 900, 4, 32, 0.2)
    w = torch.rand(900, 4, generator=gen, device="cuda")

    def step():
        leaf, lw = x.detach().requires_grad_(), w.detach().requires_grad_()
        rows, order = fgs.moe_permute(leaf, ids, 32)
        out = fgs.moe_unpermute(rows, order, lw)
        return (out.detach(), *torch.autograd.grad(out, (leaf, lw), torch.ones_like(out)))

    want = step()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = step()
    stream.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_long_rows_and_offsets_past_32_bits(gpu):
    """More than 2^31 values in rows: 2^17 slots of 2^14 + 8 columns (4.3 GB)."""
    m, topk, cols = 1 << 14, 8, (1 << 14) + 8
    x = torch.arange(m, device="cuda", dtype=torch.float32).to(torch.bfloat16)[:, None].expand(m, cols)
    ids = torch.arange(m * topk, device="cuda", dtype=torch.int32).view(m, topk) % 4
    rows, order = fgs.moe_permute(x, ids, 4)
    assert rows.numel() > 1 << 31
    slots = order.slot_of_row.long()
    assert torch.equal(rows[:, 0], x[:, 0][slots // topk])
    assert torch.equal(rows[:, -1], x[:, 0][slots // topk])
    out = fgs.moe_unpermute(rows, order, torch.full((m, topk), 1 / topk, device="cuda"))
    assert torch.equal(out[:, 0], x[:, 0]) and torch.equal(out[:, -1], x[:, 0])


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("strided", [False, True])
def test_router_takes_lazily_negated_logits(gpu, strided, dtype):
    """With and without a gradient: the values, not what memory holds of them."""
    gen = generator(31)
    values = torch.randn(2, 9, 20, generator=gen, device="cuda").to(TYPES[dtype]).unbind(0)
    d = torch.randn(9, 4, generator=gen, device="cuda")
    hidden = torch.empty(9, 1, device="cuda")
    base = torch.stack(values, -1)[..., 0] if strided else values[0]
    assert base.is_contiguous() != strided
    got, want = [], []
    for to, make in ((got, lambda t: torch._neg_view(t)), (want, lambda t: -t)):
        leaf = base.detach().requires_grad_()
        assert make(leaf).is_neg() == (to is got)
        w, ids = fgs.fused_topk(hidden, make(leaf), 4)
        to.extend([w.detach(), ids, torch.autograd.grad(w, leaf, d)[0]])
        with torch.no_grad():
            to.extend(fgs.fused_topk(hidden, make(leaf), 4))
    for a, b in zip(got, want):
        assert torch.equal(a, b)
