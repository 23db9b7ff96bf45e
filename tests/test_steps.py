"""Refusals and schedules of the routed layer's steps: no GPU is touched (the library
checks its arguments before any launch)."""

import os
import subprocess
import sys

import pytest
import torch

from flaggems_sglang import (_capi, fused_linear, fused_topk, get_op, grouped_linear, moe_permute,
                             moe_unpermute)
from test_asan_validation import ROOT, _child_env, asan_setup  # noqa: F401  (the fixture)

P = 0x1000  # an address no call reads


def call(name, defaults, **kw):
    assert set(kw) <= set(defaults)
    rc = getattr(_capi.load(), "fgs_moe_" + name)(*{**defaults, **kw}.values(), None)
    return rc, _capi.last_error()


PERMUTE = dict(x=P, stride=512, m=4, row_bytes=512, ids=P, topk=2, experts=8, rows=P, counts=P,
               row_of_slot=P, slot_of_row=P, ws=P, ws_bytes=1 << 20)
ROWS = dict(x=P, stride=512, m=4, row_bytes=512, row_of_slot=P, topk=2, slot_of_row=P, rows=P)
UNPERMUTE = dict(rows=P, ld=64, n_rows=8, order=P, weights=P, m=4, topk=2, cols=64, dtype=0, out=P)
UNGRAD = dict(dout=P, ldd=64, rows=P, ld=64, n_rows=8, order=P, back=P, weights=P, m=4, topk=2,
              cols=64, dtype=0, drows=P, dweights=P)
TOPK = dict(logits=P, bf16=0, m=4, experts=8, topk=2, scoring=0, renorm=1, weights=P, ids=P,
            dweights=P, dlogits=P)
LINEAR = dict(x=P, ldx=64, w=P, ldw=64, wg=0, bias=None, residual=None, ldr=0, counts=None,
              groups=1, rows=4, n=32, k=64, dtype=0, act=0, gated=0, flags=0, z=None, out=P)
ACT = dict(dout=P, ldd=32, z=P, rows=4, n=32, dtype=0, act=2, gated=0, dz=P)
DX = dict(dz=P, ldz=32, w=P, ldw=64, wg=0, counts=None, groups=1, rows=4, wide=32, k=64, dtype=0,
          flags=0, dx=P)
DW = dict(dz=P, ldz=32, x=P, ldx=64, counts=None, groups=1, rows=4, wide=32, k=64, dtype=0, flags=0,
          dw=P)
DB = dict(dz=P, ldz=32, counts=None, groups=1, rows=4, wide=32, dtype=0, ws=None, ws_bytes=0, db=P)


@pytest.mark.parametrize("name,defaults,kw,rc,text", [
    ("permute", PERMUTE, dict(m=-1), -1, "m >= 0"),
    ("permute", PERMUTE, dict(topk=0), -1, "topk >= 1"),
    ("permute", PERMUTE, dict(m=1 << 30), -2, "2^30 slots"),
    ("permute", PERMUTE, dict(row_bytes=0), -1, "row_bytes"),
    ("permute", PERMUTE, dict(row_bytes=1 << 25), -2, "2^24 bytes"),
    ("permute", PERMUTE, dict(stride=-1), -1, "strides"),
    ("permute", PERMUTE, dict(experts=0), -1, "num_experts"),
    ("permute", PERMUTE, dict(experts=1023), -1, "num_experts"),
    ("permute", PERMUTE, dict(x=None), -1, "null pointer"),
    ("permute", PERMUTE, dict(counts=None), -1, "null pointer"),
    ("permute", PERMUTE, dict(ws=None), -1, "workspace"),
    ("permute", PERMUTE, dict(ws_bytes=1023), -1, "workspace too small"),
    ("permute", PERMUTE, dict(ws=P + 128), -1, "256-byte"),
    ("permute", PERMUTE, dict(ids=P + 2), -1, "aligned to their"),
    ("permute_rows", ROWS, dict(m=-1), -1, "m >= 0"),
    ("permute_rows", ROWS, dict(rows=None), -1, "null pointer"),
    ("permute_rows", ROWS, dict(slot_of_row=P + 1), -1, "aligned to their"),
    ("permute_rows", ROWS, dict(m=0, x=None, rows=None), 0, ""),
    ("unpermute", UNPERMUTE, dict(topk=0), -1, "topk >= 1"),
    ("unpermute", UNPERMUTE, dict(dtype=3), -1, "element type"),
    ("unpermute", UNPERMUTE, dict(cols=0), -1, "cols >= 1"),
    ("unpermute", UNPERMUTE, dict(cols=1 << 23), -2, "2^22 columns"),
    ("unpermute", UNPERMUTE, dict(n_rows=-1), -1, "n_rows >= 0"),
    ("unpermute", UNPERMUTE, dict(n_rows=(1 << 30) + 1), -2, "2^30 rows"),
    ("unpermute", UNPERMUTE, dict(rows=None), -1, "null pointer"),
    ("unpermute", UNPERMUTE, dict(ld=-1), -1, "strides"),
    ("unpermute", UNPERMUTE, dict(rows=P + 1), -1, "aligned to their"),
    ("unpermute", UNPERMUTE, dict(weights=P + 2), -1, "aligned to their"),
    ("unpermute", UNPERMUTE, dict(m=0, out=None), 0, ""),
    ("unpermute_grad", UNGRAD, dict(drows=None, dweights=None), -1, "no output"),
    ("unpermute_grad", UNGRAD, dict(dout=None), -1, "null pointer"),
    ("unpermute_grad", UNGRAD, dict(rows=None), -1, "null pointer"),
    ("unpermute_grad", UNGRAD, dict(back=None), -1, "null pointer"),
    ("unpermute_grad", UNGRAD, dict(ldd=-1), -1, "strides"),
    ("unpermute_grad", UNGRAD, dict(dweights=P + 2), -1, "aligned to their"),
    ("unpermute_grad", UNGRAD, dict(m=0, n_rows=0, drows=None, dweights=None), 0, ""),
    ("topk_gating_grad", TOPK, dict(m=-1), -1, "m must"),
    ("topk_gating_grad", TOPK, dict(experts=1025), -1, "num_experts"),
    ("topk_gating_grad", TOPK, dict(topk=9), -1, "topk must"),
    ("topk_gating_grad", TOPK, dict(scoring=2), -1, "scoring"),
    ("topk_gating_grad", TOPK, dict(dweights=None), -1, "null pointer"),
    ("topk_gating_grad", TOPK, dict(m=0, logits=None), 0, ""),
    ("linear", LINEAR, dict(dtype=2), -2, "bf16 or fp16"),
    ("linear", LINEAR, dict(dtype=3), -1, "bf16 or fp16"),
    ("linear", LINEAR, dict(rows=-1), -1, "rows >= 0"),
    ("linear", LINEAR, dict(n=12), -2, "multiples of 8"),
    ("linear", LINEAR, dict(k=60), -2, "multiples of 8"),
    ("linear", LINEAR, dict(k=1 << 21), -2, "too large"),
    ("linear", LINEAR, dict(rows=1 << 30), -2, "too large"),
    ("linear", LINEAR, dict(n=(1 << 19) + 8, gated=1), -2, "too large"),
    ("linear_act_grad", ACT, dict(n=(1 << 19) + 8, gated=1), -2, "too large"),
    ("linear", LINEAR, dict(groups=4097, counts=P), -2, "too large"),
    ("linear", LINEAR, dict(groups=0, counts=P), -1, "groups >= 1"),
    ("linear", LINEAR, dict(groups=2), -1, "counts are needed"),
    ("linear", LINEAR, dict(act=4), -1, "activation"),
    ("linear", LINEAR, dict(flags=8), -1, "flags"),
    ("linear", LINEAR, dict(x=None), -1, "null pointer"),
    ("linear", LINEAR, dict(x=P + 8), -2, "rows of x must be 16-byte"),
    ("linear", LINEAR, dict(ldx=68), -2, "rows of x must be 16-byte"),
    ("linear", LINEAR, dict(ldw=-8), -2, "row stride of w"),
    ("linear", LINEAR, dict(ldw=(1 << 21) + 8), -2, "row stride of w"),
    ("linear", LINEAR, dict(residual=P + 8, ldr=32), -2, "rows of the residual"),
    ("linear", LINEAR, dict(counts=P, groups=2, wg=12), -2, "matrices of w"),
    ("linear", LINEAR, dict(bias=P + 1), -1, "aligned to their"),
    ("linear", LINEAR, dict(counts=P + 2), -1, "aligned to their"),
    ("linear", LINEAR, dict(rows=0, x=None, w=None, out=None), 0, ""),
    ("linear", LINEAR, dict(rows=(1 << 30) - 1, n=1 << 20), -2, "for a grid"),
    ("linear_act_grad", ACT, dict(z=None), -1, "null pointer"),
    ("linear_act_grad", ACT, dict(act=-1), -1, "activation"),
    ("linear_act_grad", ACT, dict(dout=P + 2), -2, "16-byte"),
    ("linear_act_grad", ACT, dict(rows=(1 << 30) - 1, n=1 << 20), -2, "for a grid"),
    ("linear_input_grad", DX, dict(flags=6), -1, "flags"),
    ("linear_input_grad", DX, dict(wide=4), -2, "multiples of 8"),
    ("linear_input_grad", DX, dict(dx=P + 8), -2, "16-byte"),
    ("linear_input_grad", DX, dict(rows=0, dz=None, w=None, dx=None), 0, ""),
    ("linear_weight_grad", DW, dict(flags=3), -1, "flags"),
    ("linear_weight_grad", DW, dict(x=None), -1, "null pointer"),
    ("linear_weight_grad", DW, dict(dw=None), -1, "null pointer"),
    ("linear_weight_grad", DW, dict(groups=4096, counts=P, wide=1 << 20, k=1 << 20), -2, "for a grid"),
    ("linear_bias_grad", DB, dict(dz=None), -1, "null pointer"),
    ("linear_bias_grad", DB, dict(rows=1 << 20), -1, "workspace"),
    ("linear_bias_grad", DB, dict(db=P + 1), -1, "aligned to their"),
])
def test_entry_refusals(name, defaults, kw, rc, text):
    got, msg = call(name, defaults, **kw)
    assert got == rc, msg
    assert rc == 0 or text in msg, msg


def test_entries_under_asan(asan_setup):  # noqa: F811
    r = subprocess.run(
        [sys.executable, "-m", "pytest", "-q", "-x", "-p", "no:cacheprovider",
         os.path.join(ROOT, "tests", "test_steps.py"), "-k", "refusals or schedule or workspace"],
        cwd=ROOT, env=_child_env(asan_setup), capture_output=True, text=True, timeout=600)
    out = r.stdout + r.stderr
    assert "AddressSanitizer" not in out, out[-4000:]
    assert r.returncode == 0 and "passed" in out, out[-4000:]


def test_workspaces():
    lib = _capi.load()
    assert lib.fgs_moe_permute_workspace_bytes(8, 4) >= 3 * 32
    assert lib.fgs_moe_permute_workspace_bytes(0, 4) >= 0
    assert lib.fgs_moe_permute_workspace_bytes(-1, 4) == -1
    assert lib.fgs_moe_permute_workspace_bytes((1 << 30) + 1, 4) == -1
    assert lib.fgs_moe_permute_workspace_bytes(8, 1023) == -1
    assert lib.fgs_moe_linear_bias_grad_workspace_bytes(1, 64, 64) == 0
    big = lib.fgs_moe_linear_bias_grad_workspace_bytes(1, 1 << 16, 64)
    assert big > 0 and big % (64 * 4) == 0
    assert lib.fgs_moe_linear_bias_grad_workspace_bytes(0, 64, 64) == -1


@pytest.mark.parametrize("which", ["forward", "input", "weight"])
def test_schedules(which):
    """Few rows stream, many take the largest tiles; every form has a name."""
    names = [_capi.linear_schedule(8, 4096, 4096, which=which, flags=f + 1)
             for f in range(_capi.LINEAR_FORMS[which])]
    assert len(set(names)) == len(names)
    assert _capi.linear_schedule(16384, 8192, 8192, which=which) == "tiled 256x256"
    if which != "weight":
        assert "stream" in _capi.linear_schedule(1, 4096, 4096, which=which)
    with pytest.raises(ValueError, match="flags"):
        _capi.linear_schedule(8, 4096, 4096, which=which, flags=len(names) + 1)
    with pytest.raises(NotImplementedError, match="multiples of 8"):
        _capi.linear_schedule(8, 100, 4096, which=which)


def test_operators_need_the_gpu():
    x = torch.ones(4, 64).bfloat16()
    ids = torch.zeros(4, 2, dtype=torch.int32)
    for f in (lambda: moe_permute(x, ids, 4), lambda: fused_linear(x, x),
              lambda: grouped_linear(x, x[None], ids[0, :1])):
        with pytest.raises(RuntimeError, match="GPU tensor"):
            f()
    from flaggems_sglang.ops.steps import ExpertOrder

    order = ExpertOrder(ids[0], ids[:2], ids[:, 0])
    with pytest.raises(RuntimeError, match="GPU tensor"):
        moe_unpermute(x, order)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        fused_topk(x, torch.ones(4, 8, requires_grad=True), 2)


def test_registered():
    import flaggems_sglang

    for name in ("moe_permute", "moe_unpermute", "fused_linear", "grouped_linear"):
        assert get_op(name) is getattr(flaggems_sglang, name)
