"""The dense operators' host module on the CPU: the module's own source built
for CPU tensors (host_on_cpu.cpp), each test in a process of its own, since
what it holds against has ended the process."""

import os
import subprocess
import sys
import sysconfig
import textwrap

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "flaggems-sglang_amd", "csrc")
TORCH = os.path.dirname(torch.__file__)

PRELUDE = """
import ctypes, importlib.machinery, importlib.util, sys
import torch
path = sys.argv[1]
loader = importlib.machinery.ExtensionFileLoader("_host", path)
host = importlib.util.module_from_spec(importlib.util.spec_from_loader("_host", loader))
loader.exec_module(host)
lib = ctypes.CDLL(path)
host.bind(*(ctypes.cast(getattr(lib, "host_test_" + name), ctypes.c_void_p).value
            for name in ("last_error", "rms_norm", "silu_and_mul_quant", "fp8_block_matmul")))
word = lambda name: ctypes.c_int.in_dll(lib, "host_test_" + name)
gpu, calls, locked, rc = (word(name) for name in ("gpu", "calls", "locked", "rc"))
FP8 = torch.float8_e4m3fn

def norm(x, weight=None, residual=None, quant=0, inplace=False):
    weight = torch.ones(x.shape[-1]) if weight is None else weight
    return host.rms_norm(x, weight, 1e-6, residual, 0.0, quant, True, False, inplace)
def act(x):
    return host.silu_and_mul_quant(x, 1, False, False)
def product(a=None, sa=None, w=None, sw=None, bias=None, out=None):
    a = torch.zeros(4, 256).to(FP8) if a is None else a
    sa = torch.ones(4, 2) if sa is None else sa
    w = torch.zeros(48, 256).to(FP8) if w is None else w
    sw = torch.ones(1, 2) if sw is None else sw
    return host.fp8_block_matmul(a, sa, w, sw, bias, 0, out, 0)
def refused(call, *kinds, text=""):
    before = calls.value
    try:
        call()
    except kinds or (RuntimeError,) as e:
        assert text in str(e), str(e)
    else:
        raise AssertionError("not refused")
    assert gpu.value == 0 and calls.value == before
x = torch.ones(4, 256)
"""


@pytest.fixture(scope="module")
def host_on_cpu(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("host") / "_host.so")
    r = subprocess.run(
        ["g++", "-O0", "-std=c++17", "-fPIC", "-Wall", "-shared", "-D__HIP_PLATFORM_AMD__=1",
         "-DUSE_ROCM=1", "-I" + os.path.join(ROOT, "include"), "-I" + CSRC,
         "-isystem", os.path.join(TORCH, "include"),
         "-isystem", os.path.join(TORCH, "include/torch/csrc/api/include"),
         "-isystem", sysconfig.get_paths()["include"], "-isystem", "/opt/rocm/include",
         os.path.join(ROOT, "tests", "host_on_cpu.cpp"), "-o", so, "-L" + os.path.join(TORCH, "lib"),
         "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_hip", "-ltorch_python"],
        capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-4000:]

    def run(code):
        r = subprocess.run([sys.executable, "-c", PRELUDE + textwrap.dedent(code) + "\nprint('ok')",
                            so], capture_output=True, text=True, timeout=300)
        assert r.returncode == 0 and r.stdout.endswith("ok\n"), (
            r.returncode, r.stdout[-2000:], r.stderr[-4000:])
    return run


def test_an_entry_runs_without_the_lock(host_on_cpu):
    host_on_cpu("""
        for call in (lambda: norm(x), lambda: act(x), product):
            call()
        assert (calls.value, locked.value, gpu.value) == (3, 0, 0)
        rc.value = -2
        for call in (lambda: norm(x), lambda: act(x), product):
            try:
                call()
            except NotImplementedError as e:
                assert "the entry's text" in str(e)
            else:
                raise AssertionError
        assert (calls.value, locked.value, gpu.value) == (6, 0, 0)
    """)


def test_transformed_tensors_raise(host_on_cpu):
    """Tensors of torch.vmap and torch.func have no memory to be asked for: an
    error, not the end of the process, and the GPU that was current is so again."""
    host_on_cpu("""
        for f in (norm, act, lambda t: norm(x, t[0]), lambda t: norm(x, residual=t),
                  lambda t: product(sa=t[:, :2]), lambda t: product(sw=t[:1, :2]),
                  lambda t: product(bias=t[0, :48]),
                  lambda t: product(out=t[:, :48].bfloat16())):
            refused(lambda: torch.vmap(f)(torch.ones(3, 4, 256)))
            refused(lambda: torch.func.jvp(f, (x,), (x,)))
        codes = torch.zeros(3, 4, 256).to(FP8)
        refused(lambda: torch.vmap(lambda t: product(a=t))(codes))
        norm(x), act(x), product()
        assert (calls.value, locked.value, gpu.value) == (3, 0, 0)
    """)


def test_forward_mode_tangents_are_refused(host_on_cpu):
    """A dual tensor's tangent would be lost: refused as a leaf that needs a
    gradient is; its primal, and any tensor with tangents off, is taken."""
    host_on_cpu("""
        import torch.autograd.forward_ad as fwAD
        with fwAD.dual_level():
            def dual(t):
                return fwAD.make_dual(t, torch.ones_like(t))
            d = dual(x)
            for call in (lambda: norm(d), lambda: act(d), lambda: norm(x, d[0].clone()),
                         lambda: norm(x, residual=d), lambda: norm(x, residual=d, inplace=True),
                         lambda: product(sa=dual(torch.ones(4, 2))),
                         lambda: product(sw=dual(torch.ones(1, 2))),
                         lambda: product(bias=dual(torch.ones(48))),
                         lambda: product(out=dual(torch.zeros(4, 48).bfloat16()))):
                refused(call, text="tangent")
                with torch.no_grad():  # (which does not turn them off)
                    refused(call, text="tangent")
            norm(fwAD.unpack_dual(d).primal), act(x), product()
            with fwAD._set_fwd_grad_enabled(False):
                norm(d)
        assert calls.value == 4
    """)


def test_tensors_without_memory_are_refused(host_on_cpu):
    """A residual or bias whose memory is gone is not one that was not given, and
    a view's offset into nothing is no address."""
    host_on_cpu("""
        def freed(t, view=lambda t: t):
            v = view(t)
            t.untyped_storage().resize_(0)
            return v
        zeros = torch._efficientzerotensor
        half = lambda t: t[t.shape[0] // 2:]
        for call in (lambda: norm(x, residual=zeros((4, 256))),
                     lambda: norm(x, residual=freed(torch.ones(4, 256))),
                     lambda: norm(x, residual=freed(torch.ones(8, 256), half), inplace=True),
                     lambda: norm(x, freed(torch.ones(512), half)),
                     lambda: norm(freed(torch.ones(8, 256), half)),
                     lambda: act(freed(torch.ones(8, 256), half)),
                     lambda: product(bias=freed(torch.ones(48))),
                     lambda: product(bias=zeros((48,))),
                     lambda: product(sa=freed(torch.ones(8, 2), half)),
                     lambda: product(out=freed(torch.ones(8, 48).bfloat16(), half)),
                     lambda: product(a=freed(torch.zeros(8, 256).to(FP8), half))):
            refused(call, text="no memory")
        short = torch.ones(4, 256)
        short.untyped_storage().resize_(4 * 1023)
        refused(lambda: norm(short), text="no memory")
        for call in (lambda: norm(x.to_sparse()), lambda: act(x.to_sparse_csr()),
                     lambda: product(bias=torch.ones(48).to_sparse())):
            refused(call, text="no storage")
        # no values need none
        norm(x[:0], residual=freed(torch.ones(0, 256)))
        norm(x, residual=torch.ones(1, 256).expand(4, 256))
        assert calls.value == 2
    """)


def test_outputs_that_share_an_inputs_memory_are_refused(host_on_cpu):
    """An in-place residual may be x itself, or columns or rows beside x's; where
    a row of x is another row's sum the result would depend on their order."""
    host_on_cpu("""
        flat = torch.ones(4 * 4096)
        rows = lambda at, stride=256, n=4, cols=256: flat.as_strided((n, cols), (stride, 1), at)
        for at, stride in ((256, 256), (1, 256), (768, 256), (255, 256), (0, 512), (100, 300)):
            refused(lambda: norm(rows(at, stride), residual=rows(0), inplace=True), ValueError,
                    text="share no part")
        refused(lambda: norm(rows(0)[:1].expand(4, 256), residual=rows(0), inplace=True),
                ValueError, text="share no part")
        refused(lambda: norm(rows(255, 512), residual=rows(0, 512), inplace=True), ValueError,
                text="share no part")
        refused(lambda: norm(rows(257, 512), residual=rows(0, 512), inplace=True), ValueError,
                text="share no part")
        refused(lambda: norm(rows(8192), rows(300)[0], residual=rows(0), inplace=True), ValueError,
                text="share no part")
        for at, stride, n in ((0, 256, 4), (1024, 256, 4), (1024, 300, 4)):
            norm(rows(at, stride, n), residual=rows(0), inplace=True)
        for at in (256, 256 + 4 * 512, 511 - 255):  # columns of one wider tensor
            norm(rows(at, 512), residual=rows(0, 512), inplace=True)
        norm(rows(0, 512), residual=rows(256, 512), inplace=True)
        norm(rows(256, 512, 1), residual=rows(0, 512, 1), inplace=True)
        norm(rows(4, 512, 1), residual=rows(4, 256, 1), inplace=True)
        norm(rows(0), rows(1024)[0], residual=rows(0), inplace=True)
        norm(rows(0), rows(0)[0], residual=rows(0))  # (written nowhere)
        assert calls.value == 11

        m, n, k = 4, 48, 256
        room = torch.zeros(1 << 16, dtype=torch.uint8)
        at = lambda b, t, *shape: room[b:b + 2 ** 15].view(t).as_strided(
            shape, [shape[1], 1] if len(shape) == 2 else [1])
        out = at(0, torch.bfloat16, m, n)  # 384 bytes
        for over in (dict(a=at(368, FP8, m, k)), dict(w=at(368, FP8, n, k)),
                     dict(sa=at(380, torch.float32, m, 2)), dict(sw=at(380, torch.float32, 1, 2)),
                     dict(bias=at(380, torch.float32, n)),
                     dict(sa=at(0, torch.float32, 2, m).t())):
            refused(lambda: product(out=out, **over), ValueError, text="shares memory")
        product(out=out, a=at(384, FP8, m, k), w=at(2048, FP8, n, k),
                sa=at(384, torch.float32, 2, m).t(), sw=at(384, torch.float32, 1, 2),
                bias=at(384, torch.float32, n))
        product(a=at(0, FP8, m, k), w=at(0, FP8, n, k))  # inputs may be each other's
        assert calls.value == 13
    """)
