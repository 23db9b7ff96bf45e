"""The products' gradients of operands whose rows lie less than their width apart:
one row broadcast, sliding windows."""

import pytest
import torch

import flaggems_sglang as fgs
import steps_ref as ref
from test_linear_gpu import FORMS, generator, rand

pytestmark = pytest.mark.gpu


def laid_out(gen, kind, rows, cols, scale=1.0, dtype=torch.bfloat16):
    """[rows, cols]: rows of their own, one row broadcast (strides 0, 1), or windows 8
    values apart."""
    if kind == "plain":
        return rand(gen, rows, cols, scale=scale, dtype=dtype)
    if kind == "one row":
        return rand(gen, 1, cols, scale=scale, dtype=dtype).expand(rows, cols)
    return rand(gen, 8 * rows + cols, scale=scale, dtype=dtype).as_strided((rows, cols), (8, 1))


KINDS = ["plain", "one row", "window"]
OVERLAPS = [(a, b, c) for a in KINDS for b in KINDS for c in KINDS if (a, b, c) != ("plain",) * 3]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows", [10, 33, 65, 128])
@pytest.mark.parametrize("x_kind, w_kind, d_kind", OVERLAPS)
def test_dense(gpu, x_kind, w_kind, d_kind, rows, form):
    gen = generator(rows, 51)
    n, k = 72, 136
    x, w, d = (laid_out(gen, x_kind, rows, k), laid_out(gen, w_kind, n, k, k ** -0.5),
               laid_out(gen, d_kind, rows, n))
    leaves = [t.requires_grad_() for t in (x, w)]
    bias = torch.zeros(n, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    out = fgs.fused_linear(*leaves, bias, _flags=form)
    got = dict(zip(("dx", "dw", "dbias"), torch.autograd.grad(out, leaves + [bias], d)), out=out.detach())
    want = ref.product(x.detach(), w.detach(), bias.detach(), dout=d)
    for name in want:
        ref.close(name, got[name], *want[name])


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("gated, kind", [(False, None), (True, "silu")])
@pytest.mark.parametrize("x_kind, w_kind, d_kind", OVERLAPS)
def test_groups(gpu, x_kind, w_kind, d_kind, gated, kind, form):
    gen = generator(52)
    n, k, counts = 72, 136, [10, 0, 33, 65, 1]
    rows, wide = sum(counts) + 7, n * (2 if gated else 1)
    x, d = laid_out(gen, x_kind, rows, k), laid_out(gen, d_kind, rows, n)
    flat = laid_out(gen, w_kind, wide, k, k ** -0.5)
    w = flat[None].expand(len(counts), wide, k)
    leaves = [t.requires_grad_() for t in (x, w)]
    out = fgs.grouped_linear(*leaves, torch.tensor(counts, dtype=torch.int32, device="cuda"),
                             activation=kind, gated=gated, _flags=form)
    got = dict(zip(("dx", "dw"), torch.autograd.grad(out, leaves, d)), out=out.detach())
    want = ref.grouped(x.detach(), w.detach(), counts, kind=kind, gated=gated, dout=d)
    for name in want:
        ref.close(name, got[name], *want[name])


def test_gradient_of_a_sum_over_rows(gpu):
    """Broadcast rows and the gradient that a sum over them hands back, many rows."""
    gen = generator(53)
    for rows in (10, 333, 5000):
        q, w = rand(gen, 1, 264), rand(gen, 520, 264, scale=0.06).requires_grad_()
        g = rand(gen, 520)
        fgs.fused_linear(q.expand(rows, 264), w).sum(0).backward(g)
        want = ref.product(q.expand(rows, 264), w.detach(), dout=g.expand(rows, 520))
        ref.close("dw", w.grad, *want["dw"])


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("which", ["x", "dout", "w"])
def test_infinities_of_one_overlapping_operand(gpu, which, form):
    """What is behind the sums' end is not taken, so infinities stay infinite."""
    gen = generator(54)
    x, w, d = rand(gen, 43, 136).abs(), rand(gen, 72, 136).abs(), rand(gen, 43, 72).abs()
    t = {"x": x, "w": w, "dout": d}
    one = t[which][:1].clone()
    one[0, 5] = float("inf")
    t[which] = one.expand_as(t[which])
    leaves = [t["x"].requires_grad_(), t["w"].requires_grad_()]
    out = fgs.fused_linear(*leaves, _flags=form)
    dx, dw = torch.autograd.grad(out, leaves, t["dout"])
    copies = [v.detach().contiguous().requires_grad_() for v in leaves]
    out2 = fgs.fused_linear(*copies, _flags=form)
    dx2, dw2 = torch.autograd.grad(out2, copies, t["dout"].contiguous())
    for a, b in ((out, out2), (dx, dx2), (dw, dw2)):
        assert torch.equal(a, b)
    assert not bool(dw.isnan().any()) and not bool(dx.isnan().any())
