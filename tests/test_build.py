"""The makefile's rules, with a compiler and an interpreter that only note
their calls."""

import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "flaggems-sglang_amd", "csrc")


@pytest.fixture
def make(tmp_path):
    log = tmp_path / "log"
    for name, body in (("cxx", f'echo "$@" >> {log}\nwhile [ "$1" != -o ]; do shift; done\n: > "$2"'),
                       ("python", 'echo "$FAKE_TORCH"')):
        (tmp_path / name).write_text("#!/bin/sh\n" + body + "\n")
        (tmp_path / name).chmod(0o755)

    def run(target, torch, python="python"):
        before = log.read_text() if log.exists() else ""
        r = subprocess.run(
            ["make", "-C", CSRC, f"OUT_DIR={tmp_path}", f"OBJ_DIR={tmp_path}/obj",
             f"CXX={tmp_path}/cxx", f"HIPCC={tmp_path}/cxx", f"PYTHON={tmp_path}/{python}",
             target], env={**os.environ, "FAKE_TORCH": torch}, capture_output=True, text=True,
            timeout=120)
        return r.returncode, (log.read_text() if log.exists() else "")[len(before):]
    run.path = str(tmp_path)
    return run


def test_host_module_follows_its_torch(make):
    """Built once for a torch, not again for the same one, and again for
    another, in whose headers it is then built."""
    target = make.path + "/_host.so"
    for torch, built in (("/a/torch", True), ("/a/torch", False), ("/b/torch", True),
                         ("/b/torch", False), ("/a/torch", True)):
        rc, log = make(target, torch)
        assert rc == 0
        assert ("host_ext.cpp" in log) == built, (torch, log)
        assert not built or torch + "/include" in log


def test_library_alone_needs_no_torch(make):
    rc, log = make("lib", "", python="none")
    assert rc == 0 and "libfgs_moe.so" in log and "host_ext" not in log
    assert "capi.hip" in log and "block_gemm.hip" in log
