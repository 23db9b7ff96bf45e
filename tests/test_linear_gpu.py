"""fused_linear and grouped_linear with their gradients against plain forms in 64
bits, on the GPU."""

import pytest
import torch

import flaggems_sglang as fgs
import steps_ref as ref
from flaggems_sglang import _capi

pytestmark = pytest.mark.gpu

def flags(form):
    """Form ``form`` - 1 of each pass, or its last one; 0: the call's own choice."""
    return sum(min(form, _capi.LINEAR_FORMS[p]) << (8 * i)
               for i, p in enumerate(("forward", "input", "weight")))


FORMS = [flags(f) for f in range(max(_capi.LINEAR_FORMS.values()) + 1)]
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def rand(gen, *shape, dtype=torch.bfloat16, scale=1.0):
    return (scale * torch.randn(*shape, generator=gen, device="cuda")).to(dtype)


def generator(*numbers):
    return torch.Generator(device="cuda").manual_seed(sum(7 ** i * n for i, n in enumerate(numbers)))


def inputs(rows, n, k, dtype, gated, bias, residual, groups=None, seed=0):
    gen = generator(rows, n, k, seed)
    wide = n * (2 if gated else 1)
    lead = () if groups is None else (groups,)
    return dict(
        x=rand(gen, rows, k, dtype=dtype), w=rand(gen, *lead, wide, k, dtype=dtype, scale=k ** -0.5),
        bias=rand(gen, *lead, wide, dtype=dtype) if bias else None,
        residual=rand(gen, rows, n, dtype=dtype) if residual else None), rand(gen, rows, n, dtype=dtype)


def run(t, counts=None, dout=None, **options):
    """out and the gradients of what is given, by their names."""
    leaves = {k: v.detach().requires_grad_() for k, v in t.items() if v is not None}
    args = [leaves["x"], leaves["w"]] + ([] if counts is None else [counts])
    f = fgs.fused_linear if counts is None else fgs.grouped_linear
    out = f(*args, leaves.get("bias"), residual=leaves.get("residual"), **options)
    got = {"out": out.detach()}
    if dout is not None:
        grads = torch.autograd.grad(out, list(leaves.values()), dout)
        got.update({"d" + k: g for k, g in zip(leaves, grads)})
    return got


def compare(got, want):
    assert set(got) == set(want)
    for name, (value, bound) in want.items():
        ref.close(name, got[name], value, bound)


SIZES = [(1, 8, 8), (7, 24, 40), (33, 264, 72), (64, 128, 64), (129, 136, 200), (300, 520, 328),
         (513, 1032, 192), (257, 256, 1000)]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows, n, k", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
def test_dense(gpu, dtype, rows, n, k, form):
    t, dout = inputs(rows, n, k, TYPES[dtype], False, True, True)
    got = run(t, dout=dout, _flags=form)
    compare(got, ref.product(**t, dout=dout))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("kind", ["relu", "silu", "gelu"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows, n, k", [(5, 8, 24), (70, 200, 136), (270, 392, 80)])
def test_activations(gpu, rows, n, k, gated, kind, form):
    for bias, residual, dtype in [(True, True, "bf16"), (False, False, "fp16")]:
        t, dout = inputs(rows, n, k, TYPES[dtype], gated, bias, residual)
        got = run(t, dout=dout, activation=kind, gated=gated, _flags=form)
        compare(got, ref.product(**t, kind=kind, gated=gated, dout=dout))


COUNTS = {
    "even": [64, 64, 64, 64], "ragged": [1, 0, 130, 7, 0, 118], "one of many": [0, 0, 0, 256],
    "rows behind": [30, 5, 0, 91], "none": [0, 0, 0], "negative": [-5, 40, -1, 100],
    "past the end": [200, 100, 50], "empty first and last": [0, 100, 156, 0],
    "many": [3 * (i % 3) + (i == 77) * 40 for i in range(130)],
}


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("n, k, gated, kind", [(136, 72, False, None), (264, 200, True, "silu"),
                                               (40, 136, False, "gelu")])
def test_groups(gpu, n, k, gated, kind, counts, form):
    c = COUNTS[counts]
    rows = 500 if counts == "many" else 256
    t, dout = inputs(rows, n, k, torch.bfloat16, gated, True, True, groups=len(c))
    on_gpu = torch.tensor(c, dtype=torch.int32, device="cuda")
    got = run(t, on_gpu, dout, activation=kind, gated=gated, _flags=form)
    compare(got, ref.grouped(**t, counts=c, kind=kind, gated=gated, dout=dout))


@pytest.mark.parametrize("form", FORMS)
def test_rows_of_no_group_are_not_read(gpu, form):
    """NaN and infinities behind the last group's rows reach no output."""
    c = [20, 0, 60]
    t, dout = inputs(200, 72, 136, torch.bfloat16, True, True, False, groups=3)
    t["x"][80:] = float("nan")
    dout[80:140] = float("inf")
    dout[140:] = float("nan")
    counts = torch.tensor(c, dtype=torch.int32, device="cuda")
    got = run(t, counts, dout, activation="silu", gated=True, _flags=form)
    t["x"][80:] = 0
    dout[80:] = 0
    compare(got, ref.grouped(**t, counts=c, kind="silu", gated=True, dout=dout))


@pytest.mark.parametrize("form", FORMS)
def test_nan_stays_in_its_row(gpu, form):
    """A NaN of x is in its output row, its dx's and (through x) the weights'
    column, no neighbour's; zeros stand behind every sum's end."""
    t, dout = inputs(100, 136, 104, torch.bfloat16, False, False, False)
    clean = run(t, dout=dout, _flags=form)
    t["x"][41, 103] = float("nan")
    got = run(t, dout=dout, _flags=form)
    assert bool(got["out"][41].isnan().all())
    keep = torch.arange(100, device="cuda") != 41
    assert torch.equal(got["out"][keep], clean["out"][keep])
    assert torch.equal(got["dx"], clean["dx"])
    assert bool(got["dw"][:, 103].isnan().all())
    assert torch.equal(got["dw"][:, :103], clean["dw"][:, :103])


@pytest.mark.parametrize("kind", ["relu", "silu", "gelu"])
@pytest.mark.parametrize("gated", [False, True])
def test_nan_passes_activations(gpu, kind, gated):
    """A NaN row reaches its own output and the weights, and no other row."""
    t, dout = inputs(20, 72, 64, torch.bfloat16, gated, False, False)
    t["x"][7] = float("nan")
    got = run(t, dout=dout, activation=kind, gated=gated)
    assert bool(got["out"][7].isnan().all()) and bool(got["dw"].isnan().all())
    keep = torch.arange(20, device="cuda") != 7
    assert bool(got["out"][keep].isfinite().all()) and bool(got["dx"][keep].isfinite().all())


@pytest.mark.parametrize("form", FORMS)
def test_strides_and_shapes(gpu, form):
    """Slices of wider tensors, leading sizes, other strides, offsets that leave
    rows unaligned: the values of contiguous copies."""
    gen = generator(3)
    wide = rand(gen, 90, 200)
    w_wide = rand(gen, 100, 136, scale=0.1)
    for x, w in [(wide[:, 8:80], w_wide[:72, 64:]), (wide[:, 3:75], w_wide[1:97:2, 5:77]),
                 (wide[:72].t()[8:], w_wide[:72, :72].t()), (wide[:1, :72].expand(40, 72), w_wide[:96, :72])]:
        a, b = fgs.fused_linear(x, w, _flags=form), fgs.fused_linear(x.contiguous(), w.contiguous(),
                                                                    _flags=form)
        assert torch.equal(a, b)
    x = rand(gen, 2, 3, 5, 64)
    w = rand(gen, 40, 64)
    out = fgs.fused_linear(x, w, residual=rand(gen, 2, 3, 5, 40), _flags=form)
    assert out.shape == (2, 3, 5, 40)
    assert fgs.fused_linear(x[:0], w).shape == (0, 3, 5, 40)
    # stepped groups, and a gradient whose rows all lie at one address
    w = rand(gen, 6, 80, 72, scale=0.1)
    counts = torch.tensor([30, 20, 40], dtype=torch.int32, device="cuda")
    leaf, copy = (v.detach().requires_grad_() for v in (w[::2, :64], w[::2, :64].contiguous()))
    for grad in (rand(gen, 1, 1).expand(90, 64), rand(gen, 90, 72)[:, 8:]):
        a, = torch.autograd.grad(fgs.grouped_linear(wide[:, :72], leaf, counts), leaf, grad)
        b, = torch.autograd.grad(fgs.grouped_linear(wide[:, :72], copy, counts), copy, grad.contiguous())
        assert torch.equal(a, b)


def test_no_rows(gpu):
    """No rows: empty outputs, and weights' gradients of zeros."""
    x = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    w = torch.randn(3, 32, 64, device="cuda").bfloat16().requires_grad_()
    b = torch.zeros(3, 32, device="cuda").bfloat16().requires_grad_()
    counts = torch.zeros(3, dtype=torch.int32, device="cuda")
    out = fgs.grouped_linear(x, w, counts, b, activation="gelu")
    assert out.shape == (0, 32)
    dx, dw, db = torch.autograd.grad(out, (x, w, b), torch.empty_like(out))
    assert dx.shape == x.shape and not bool(dw.any()) and not bool(db.any())


@pytest.mark.parametrize("kind, gated", [("silu", True), ("gelu", False)])
def test_gradients_against_differences(gpu, kind, gated):
    """fp16 gradients against differences of the plain form in 64 bits: the same
    bound as against its derivative, and the differences' own error, at most the
    third derivative's (4 is above any here) times the step squared."""
    t, dout = inputs(6, 16, 24, torch.float16, gated, True, False)
    got = run(t, dout=dout, activation=kind, gated=gated)
    want = ref.product(**t, kind=kind, gated=gated, dout=dout)
    step = 2.0 ** -12

    def loss(**changed):
        v = {k: q.double() for k, q in t.items() if q is not None} | changed
        z = v["x"] @ v["w"].t() + v["bias"]
        y = ref.act(z[:, :16], kind)[0] * z[:, 16:] if gated else ref.act(z, kind)[0]
        return float((y * dout.double()).sum())

    for name in ("x", "w", "bias"):
        base = t[name].double()
        for i in range(0, base.numel(), 1 + base.numel() // 9):
            sides = []
            for sign in (1, -1):
                moved = base.clone()
                moved.view(-1)[i] += sign * step
                sides.append(loss(**{name: moved}))
            diff = (sides[0] - sides[1]) / (2 * step)
            bound = float(want["d" + name][1].reshape(-1)[i])
            assert abs(float(got["d" + name].reshape(-1)[i]) - diff) <= bound + 400 * step ** 2, name


def test_needs_of_gradients(gpu):
    """Only the gradients that are asked for are made; x's alone, the bias's alone."""
    t, dout = inputs(40, 64, 32, torch.bfloat16, False, True, True)
    want = ref.product(**t, kind="silu", dout=dout)
    for name in t:
        leaf = t[name].detach().requires_grad_()
        args = t | {name: leaf}
        out = fgs.fused_linear(args["x"], args["w"], args["bias"], activation="silu",
                               residual=args["residual"])
        g, = torch.autograd.grad(out, leaf, dout)
        ref.close(name, g, *want["d" + name])


def test_no_second_derivative(gpu):
    t, dout = inputs(8, 16, 16, torch.bfloat16, False, False, False)
    x = t["x"].requires_grad_()
    g, = torch.autograd.grad(fgs.fused_linear(x, t["w"]).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


def test_same_inputs_same_bits(gpu):
    t, dout = inputs(777, 264, 520, torch.bfloat16, True, True, False, groups=5)
    counts = torch.tensor([100, 300, 0, 277, 90], dtype=torch.int32, device="cuda")
    first = run(t, counts, dout, activation="silu", gated=True)
    for _ in range(3):
        again = run(t, counts, dout, activation="silu", gated=True)
        for name in first:
            assert torch.equal(first[name], again[name]), name


def test_graph(gpu):
    """Forward and backward captured, replayed on new inputs."""
    t, dout = inputs(200, 72, 136, torch.bfloat16, True, True, False, groups=4)
    counts = torch.tensor([50, 0, 100, 50], dtype=torch.int32, device="cuda")
    leaves = [v.requires_grad_() for v in (t["x"], t["w"], t["bias"])]

    def step():
        out = fgs.grouped_linear(leaves[0], leaves[1], counts, leaves[2], activation="silu", gated=True)
        return (out.detach(), *torch.autograd.grad(out, leaves, dout))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        captured = step()
    gen = generator(9)
    for sizes in ([50, 0, 100, 50], [0, 200, 0, 0], [10, 20, 30, 40]):
        with torch.no_grad():
            counts.copy_(torch.tensor(sizes, dtype=torch.int32))
            for v in leaves:
                v.copy_(rand(gen, *v.shape))
            dout.copy_(rand(gen, *dout.shape))
        graph.replay()
        torch.cuda.synchronize()
        got = [c.clone() for c in captured]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_other_stream(gpu):
    t, dout = inputs(300, 200, 72, torch.bfloat16, False, True, False)
    want = run(t, dout=dout, activation="gelu")
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = run(t, dout=dout, activation="gelu")
    stream.synchronize()
    for name in want:
        assert torch.equal(got[name], want[name])


# (rows, n, k, counts): more than a round of 256 x 256 tiles, the last of which leaves
# CUs without one: for the forward product and, with n and k swapped, each gradient
CUT = [(2100, 8200, 72, None), (2304, 8192, 64, None), (2100, 8200, 72, [700, 0, 33, 900, 1, 400]),
       (2600, 8200, 40, [256] * 9)]


@pytest.mark.parametrize("which", ["forward", "gated", "input", "weight"])
@pytest.mark.parametrize("rows, n, k, counts", CUT)
def test_last_round_in_quarters(gpu, rows, n, k, counts, which):
    large = sum(_capi.LINEAR_FORMS[p] << (8 * i) for i, p in enumerate(("forward", "input", "weight")))
    if which == "input":
        n, k = k, n
    if which == "weight":
        rows, n, k = k, 2104, n
        counts = None if counts is None else [30, 0, k]  # (cut at the last row)
    gated = which == "gated"
    if gated:
        n = (n // 2 + 7) // 8 * 8
    groups = None if counts is None else len(counts)
    t, dout = inputs(rows, n, k, torch.bfloat16, gated, which in ("forward", "gated"), False, groups)
    on_gpu = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    options = dict(kind="silu" if gated else None, gated=gated,
                   dout=dout if which in ("input", "weight") else None)
    want = ref.product(**t, **options) if counts is None else ref.grouped(**t, counts=counts, **options)
    got = run(t, on_gpu, options["dout"], activation=options["kind"], gated=gated, _flags=large)
    compare(got, want)


@pytest.mark.parametrize("which", ["forward", "gated", "input"])
@pytest.mark.parametrize("rows, counts", [
    (256 * 18 + 1, None), (256 * 18 + 128, None), (256 * 18 + 129, None), (100, None),
    (2560, [1, 128, 129, 255, 256, 257, 0, 384, 385, 640]), (2560, [128] * 18 + [100]),
    (2560, [0, 640, -5, 513, 128]), (2561, [255] * 9 + [385]), (2500, [2200, 400, 100])])
def test_rows_past_whole_tiles(gpu, rows, counts, which):
    """More than a round of 256 x 256 tiles: groups (and products) that end in each part
    of a tile; rows of no group are 0."""
    large = sum(_capi.LINEAR_FORMS[p] << (8 * i) for i, p in enumerate(("forward", "input", "weight")))
    wide = 4136 if rows > 256 else 66056
    n, k = (40, wide) if which == "input" else (wide, 40)
    gated = which == "gated"
    if gated:
        n //= 2
        n = n // 8 * 8
    groups = None if counts is None else len(counts)
    t, dout = inputs(rows, n, k, torch.bfloat16, gated, which != "input", False, groups)
    on_gpu = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    options = dict(kind="silu" if gated else None, gated=gated, dout=dout if which == "input" else None)
    if counts is not None:  # (as the kernels cut them)
        left, cut = rows, []
        for c in counts:
            cut.append(min(max(c, 0), left))
            left -= cut[-1]
        counts = cut
    want = ref.product(**t, **options) if counts is None else ref.grouped(**t, counts=counts, **options)
    got = run(t, on_gpu, options["dout"], activation=options["kind"], gated=gated, _flags=large)
    compare(got, want)


@pytest.mark.parametrize("which", ["input", "weight"])
@pytest.mark.parametrize("sums", [8, 64, 72, 136, 520])
@pytest.mark.parametrize("dtype", TYPES)
def test_several_tiles_of_a_workgroup(gpu, dtype, sums, which):
    """The gradients in 256 x 256 tiles, each workgroup with several of them, some of a
    stage or none: the same bits each time."""
    large = sum(_capi.LINEAR_FORMS[p] << (8 * i) for i, p in enumerate(("forward", "input", "weight")))
    if which == "input":
        rows, n, k, counts = 4700, sums, 8208, [1000, 0, 2000, 257, 1, 1300]  # 142 left over
    else:
        rows, n, k, counts = 6 * sums, 1544, 4104, [sums, 0, 3 * sums, 1, sums // 2, sums // 4]
    t, dout = inputs(rows, n, k, TYPES[dtype], False, False, False, len(counts))
    on_gpu = torch.tensor(counts, dtype=torch.int32, device="cuda")
    runs = [run(t, on_gpu, dout, _flags=large) for _ in range(4)]
    compare(runs[0], ref.grouped(**t, counts=counts, dout=dout))
    name = "dx" if which == "input" else "dw"
    for again in runs[1:]:
        assert torch.equal(again[name], runs[0][name])
