"""The host side of the routed layer's steps on the CPU: the module's own source
built for CPU tensors (steps_on_cpu.cpp), each test in a process of its own."""

import os
import subprocess
import sys
import sysconfig
import textwrap

import pytest

from test_dense_host import CSRC, PRELUDE, ROOT, TORCH

STEPS = PRELUDE + """
from flaggems_sglang import _capi
host.bind_steps(*(ctypes.cast(getattr(lib, "host_test_" + name), ctypes.c_void_p).value
                  for name in _capi._STEPS))
_capi._host = host  # (the operators' Python side over it)
torch.cuda.is_current_stream_capturing = lambda: False
import flaggems_sglang as fgs
I32, BF16 = torch.int32, torch.bfloat16
ids = torch.zeros(4, 2, dtype=I32)
order = fgs.ops.steps.ExpertOrder(torch.zeros(3, dtype=I32), torch.zeros(4, 2, dtype=I32),
                                  torch.zeros(8, dtype=I32))
rows, weights = torch.ones(8, 256), torch.ones(4, 2)
a, w, bias = torch.ones(4, 64).to(BF16), torch.ones(32, 64).to(BF16), torch.ones(32).to(BF16)
ew, counts = torch.ones(3, 32, 64).to(BF16), torch.ones(3, dtype=I32)
res = torch.ones(4, 32).to(BF16)
permute = lambda x=x, ids=ids, n=3: fgs.moe_permute(x, ids, n)
again = lambda x=x, order=order: fgs.moe_permute(x, order=order)
unpermute = lambda r=rows, o=order, w=weights: fgs.moe_unpermute(r, o, w)
dense = lambda x=a, w=w, b=None, **k: fgs.fused_linear(x, w, b, **k)
grouped = lambda x=a, w=ew, c=counts, b=None, **k: fgs.grouped_linear(x, w, c, b, **k)
ALL = (permute, again, unpermute, dense, grouped)
calls.value = 0
"""


@pytest.fixture(scope="module")
def steps_on_cpu(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("steps") / "_host.so")
    r = subprocess.run(
        ["g++", "-O0", "-std=c++17", "-fPIC", "-Wall", "-shared", "-D__HIP_PLATFORM_AMD__=1",
         "-DUSE_ROCM=1", "-I" + os.path.join(ROOT, "include"), "-I" + CSRC,
         "-isystem", os.path.join(TORCH, "include"),
         "-isystem", os.path.join(TORCH, "include/torch/csrc/api/include"),
         "-isystem", sysconfig.get_paths()["include"], "-isystem", "/opt/rocm/include",
         os.path.join(ROOT, "tests", "steps_on_cpu.cpp"), "-o", so, "-L" + os.path.join(TORCH, "lib"),
         "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_hip", "-ltorch_python"],
        capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-4000:]

    def run(code):
        env = dict(os.environ, PYTHONPATH=os.path.join(ROOT, "flaggems-sglang_amd"))
        r = subprocess.run([sys.executable, "-c", STEPS + textwrap.dedent(code) + "\nprint('ok')", so],
                           capture_output=True, text=True, timeout=300, env=env)
        assert r.returncode == 0 and r.stdout.endswith("ok\n"), (
            r.returncode, r.stdout[-2000:], r.stderr[-4000:])
    return run


def test_calls_and_their_errors(steps_on_cpu):
    steps_on_cpu("""
        for call in ALL:
            call()
        assert (calls.value, locked.value, gpu.value) == (5, 0, 0)
        rc.value = -2
        for call in ALL:
            try:
                call()
            except NotImplementedError as e:
                assert "the entry's text" in str(e)
            else:
                raise AssertionError
        assert (calls.value, locked.value, gpu.value) == (10, 0, 0)
    """)


def test_refusals(steps_on_cpu):
    steps_on_cpu("""
        A = AssertionError
        for kinds, text, call in [
            ((A,), "topk_ids must be int32", lambda: permute(ids=ids.float())),
            ((A,), "topk_ids must be int32", lambda: permute(ids=ids[:3])),
            ((A,), "x must be [tokens", lambda: permute(x=x[0])),
            ((A,), "x must be of", lambda: permute(x=x.double())),
            ((A,), "x must be of", lambda: permute(x=x.to(torch.complex64))),
            ((ValueError,), "num_experts", lambda: permute(n=0)),
            ((ValueError,), "num_experts", lambda: permute(n=1023)),
            ((ValueError,), "or an order", lambda: fgs.moe_permute(x)),
            ((ValueError,), "or an order", lambda: fgs.moe_permute(x, ids)),
            ((ValueError,), "or an order", lambda: fgs.moe_permute(x, ids, 3, order=order)),
            ((A,), "other tokens", lambda: again(x=x[:3])),
            ((A,), "other rows", lambda: unpermute(r=rows[:7])),
            ((A,), "topk_weights", lambda: unpermute(w=weights[:3])),
            ((A,), "rows must be bf", lambda: unpermute(r=rows.to(torch.int32))),
            ((A,), "rows must be [rows", lambda: unpermute(r=rows[:, :0])),
            ((A,), "row_of_slot", lambda: unpermute(o=order._replace(row_of_slot=ids.long()))),
            ((A,), "x must be bfloat16 or", lambda: dense(x=a.float(), w=w.float())),
            ((A,), "weight must be of x's", lambda: dense(w=w.half())),
            ((A,), "[..., k] and weight", lambda: dense(w=w[:, :32])),
            ((A,), "[..., k] and weight", lambda: dense(w=ew)),
            ((A,), "weight must not be empty", lambda: dense(w=w[:0])),
            ((A,), "bias must be", lambda: dense(b=bias[:16])),
            ((A,), "bias must be", lambda: dense(b=bias.float())),
            ((A,), "residual must be", lambda: dense(residual=res[:3])),
            ((A,), "residual must be", lambda: dense(residual=res, gated=True)),
            ((A,), "gate rows and up rows", lambda: dense(w=w[:31], gated=True)),
            ((ValueError,), "Unsupported activation", lambda: dense(activation="tanh")),
            ((A,), "x must be [rows, k]", lambda: grouped(x=a[None])),
            ((A,), "x must be [rows, k]", lambda: grouped(w=w)),
            ((A,), "counts must be", lambda: grouped(c=counts[:2])),
            ((A,), "counts must be", lambda: grouped(c=counts.long())),
            ((A,), "bias must be", lambda: grouped(b=bias)),
            ((TypeError,), "counts must be a tensor", lambda: grouped(c=None)),
            ((TypeError,), "x must be a tensor", lambda: fgs.fused_linear([1.0], w)),
        ]:
            refused(call, *kinds, text=text)
        permute(ids=ids.long()), unpermute(w=weights.half()), unpermute(w=None)
        assert calls.value == 3
    """)


def test_transformed_tensors_raise(steps_on_cpu):
    steps_on_cpu("""
        for f, t in [(lambda t: permute(x=t), x), (lambda t: again(x=t), x),
                     (lambda t: unpermute(r=t), rows), (lambda t: unpermute(w=t), weights),
                     (lambda t: dense(x=t), a), (lambda t: dense(w=t), w),
                     (lambda t: dense(b=t), bias), (lambda t: dense(residual=t), res),
                     (lambda t: grouped(w=t), ew)]:
            refused(lambda: torch.vmap(f)(torch.stack([t, t])))
            refused(lambda: torch.func.jvp(f, (t,), (t,)))
            first = lambda t: f(t)[0] if isinstance(f(t), tuple) else f(t)
            refused(lambda: torch.func.grad(lambda t: first(t).float().sum())(t))
        for call in ALL:
            call()
        assert (calls.value, gpu.value) == (5, 0)
    """)


def test_forward_mode_tangents_are_refused(steps_on_cpu):
    steps_on_cpu("""
        import torch.autograd.forward_ad as fwAD
        with fwAD.dual_level():
            dual = lambda t: fwAD.make_dual(t, torch.ones_like(t))
            leaf = lambda t: fwAD.make_dual(t.clone().requires_grad_(), torch.ones_like(t))
            for make in (dual, leaf):
                for f in (lambda: permute(x=make(x)), lambda: again(x=make(x)),
                          lambda: unpermute(r=make(rows)), lambda: unpermute(w=make(weights)),
                          lambda: dense(x=make(a)), lambda: dense(b=make(bias)),
                          lambda: dense(residual=make(res)), lambda: grouped(w=make(ew))):
                    try:
                        f()
                    except RuntimeError as e:
                        assert "tangent" in str(e) or "jvp" in str(e), str(e)
                    else:
                        raise AssertionError
    """)


def test_tensors_without_memory_are_refused(steps_on_cpu):
    steps_on_cpu("""
        def freed(t):
            t = t.clone()
            t.untyped_storage().resize_(0)
            return t
        for call in (lambda: permute(x=freed(x)), lambda: permute(ids=freed(ids)),
                     lambda: again(order=order._replace(slot_of_row=freed(order.slot_of_row))),
                     lambda: unpermute(r=freed(rows)), lambda: unpermute(w=freed(weights)),
                     lambda: dense(x=freed(a)), lambda: dense(b=freed(bias)),
                     lambda: dense(residual=freed(res)), lambda: grouped(c=freed(counts)),
                     lambda: dense(b=torch._efficientzerotensor((32,), dtype=BF16))):
            refused(call, text="no memory")
        refused(lambda: dense(x=a.to_sparse()), text="no storage")
        refused(lambda: dense(x=torch._neg_view(a)), NotImplementedError, text="negated")
    """)


def test_gradients_reach_their_entries(steps_on_cpu):
    """A backward pass runs on the engine's side, without the lock, asks for what is
    needed alone, and raises what an entry returns; a second one raises."""
    steps_on_cpu("""
        leaf = lambda t: t.clone().requires_grad_()
        grad = torch.autograd.grad
        t = leaf(x)
        out, o = permute(x=t)
        assert out.requires_grad and not any(v.requires_grad for v in o)
        g, = grad(out, t, torch.ones_like(out))
        assert g.shape == t.shape
        t = leaf(rows)
        assert grad(unpermute(r=t), t, torch.ones(4, 256))[0].shape == t.shape
        t = leaf(weights)
        assert grad(unpermute(w=t), t, torch.ones(4, 256))[0].shape == t.shape
        before = calls.value
        ts = [leaf(v) for v in (a, w, bias, res)]
        out = dense(ts[0], ts[1], ts[2], activation="gelu", residual=ts[3])
        for i, entries in ((0, 2), (1, 2), (2, 2), (3, 0)):  # (the activation's and its own)
            before = calls.value
            g, = grad(out, ts[i], torch.ones_like(out), retain_graph=True)
            assert g.shape == ts[i].shape and calls.value == before + entries, (i, calls.value - before)
        before = calls.value
        grad(out, ts, torch.ones_like(out), retain_graph=True)
        assert calls.value == before + 4
        g = grad(out, ts, torch.ones_like(out), create_graph=True)
        for v in g[:3]:
            try:
                v.float().sum().backward(retain_graph=True)
            except RuntimeError as e:
                assert "no second derivative" in str(e), str(e)
            else:
                raise AssertionError
        rc.value = -3
        try:
            grad(out, ts, torch.ones_like(out))
        except RuntimeError as e:
            assert "the entry's text" in str(e)
        else:
            raise AssertionError
        rc.value = 0
        # a saved tensor that was written since
        t = leaf(a)
        out = dense(x=t, w=leaf(w))
        with torch.no_grad():
            t.add_(1)
        try:
            out.float().sum().backward()
        except RuntimeError as e:
            assert "modified by an inplace operation" in str(e)
        else:
            raise AssertionError
        assert locked.value == 0
    """)


def test_only_what_a_gradient_needs_is_kept(steps_on_cpu):
    """A tensor that no gradient asked for reads may be written before the backward pass;
    one that is read may not."""
    steps_on_cpu("""
        leaf = lambda t: t.clone().requires_grad_()

        def passes(out, of, dout, written, raises):
            with torch.no_grad():
                written.add_(1)
            try:
                g, = torch.autograd.grad(out, of, dout)
            except RuntimeError as e:
                assert raises and "modified by an inplace operation" in str(e), str(e)
            else:
                assert not raises and g.shape == of.shape and g.dtype == of.dtype

        for kind in (None, "gelu"):
            for call, w0, more in ((dense, w, {}), (grouped, ew, {"c": counts})):
                b0 = bias if call is dense else torch.ones(3, 32).to(BF16)
                for of in "xwbr":
                    for write in "xwbrc":
                        if write == "c" and call is dense:
                            continue
                        t = dict(x=a.clone(), w=w0.clone(), b=b0.clone(), r=res.clone(), c=counts.clone())
                        t[of].requires_grad_()
                        args = dict(x=t["x"], w=t["w"], b=t["b"], residual=t["r"], activation=kind)
                        if call is grouped:
                            args["c"] = t["c"]
                        read = {"x": "wc", "w": "xc", "b": "c", "r": ""}[of]
                        passes(call(**args), t[of], torch.ones_like(res), t[write], write in read)
        # leading sizes, a vector
        for shape in ((64,), (2, 3, 64), (0, 64)):
            for of in (0, 1):
                t = [torch.ones(shape).to(BF16), w.clone()]
                t[of].requires_grad_()
                out = dense(*t, activation="silu", gated=True)
                passes(out, t[of], torch.ones_like(out), t[of], False)

        for of in "rw":
            for write in "rwo":
                t = dict(r=rows.clone(), w=weights.clone(), o=order.row_of_slot.clone())
                t[of].requires_grad_()
                out = unpermute(t["r"], order._replace(row_of_slot=t["o"]), t["w"])
                passes(out, t[of], torch.ones_like(out), t[write], write == "o" or write != of)

        logits = torch.ones(4, 3)
        for dtype in (torch.float32, BF16):
            for scoring in (0, 1):
                for renormalize in (False, True):
                    t = logits.to(dtype).requires_grad_()
                    out, _ = host.topk_gating(t, 2, scoring, renormalize)
                    passes(out, t, torch.ones_like(out), t, scoring == int(renormalize))
    """)
