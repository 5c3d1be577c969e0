"""The C++ operators' library: one that does not load leaves the rest of the
package usable, and another torch makes it be built again."""
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

import h3_engine_b200
from h3_engine_b200.csrc import build

PKG = Path(h3_engine_b200.__file__).resolve().parent

CALLS = """
from h3_engine_b200 import blocks, dit, mxfp4, nvfp4, ops, torch_ops
from h3_engine_b200.kernels import ffn_qkvo_gemms
import torch
assert hasattr(torch.ops.h3b, "nvfp4_gemm")
for call in (torch_ops.ext_op("mxfp4_quantize"), mxfp4._LINEAR, ops._WINDOW):
    try:
        call(torch.zeros(1))
    except RuntimeError as e:
        assert "h3_engine_b200.csrc.build" in str(e), e
    else:
        raise SystemExit("an operator without its library ran")
"""


@pytest.mark.parametrize("content", [None, b"", b"\x7fELF" + bytes(60), b"not a library"])
def test_a_library_that_does_not_load(tmp_path, content):
    shutil.copytree(PKG, tmp_path / PKG.name, ignore=shutil.ignore_patterns("*.so*", "__pycache__"))
    if content is not None:
        (tmp_path / PKG.name / "_h3b_torch.so").write_bytes(content)
    r = subprocess.run([sys.executable, "-c", CALLS], cwd=tmp_path, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def test_another_torch_needs_another_build(tmp_path, monkeypatch):
    import torch
    ran = []

    def compiler(cmd, **_):
        ran.append(cmd)
        Path(cmd[cmd.index("-o") + 1]).write_bytes(b"built")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build, "EXT", tmp_path / "_h3b_torch.so")
    monkeypatch.setattr(build.subprocess, "run", compiler)
    build.build_ext()
    build.build_ext()
    assert len(ran) == 1
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    build.build_ext()
    build.build_ext()
    assert len(ran) == 2
    build.build_ext(force=True)
    assert len(ran) == 3
    (tmp_path / "_h3b_torch.so.torch").unlink()        # built by an older build: not known
    build.build_ext()
    assert len(ran) == 4
