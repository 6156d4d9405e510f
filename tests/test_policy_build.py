"""What of ``navi_amd.policy`` works without the extension that makes calls of a block's operators, and how the build
finds PyTorch (no GPU)."""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]

PROGRAM = """
import torch
from navi_amd import policy, _policy_native
print(_policy_native.lib().navi_policy_last_error() == b"")
x = torch.zeros(2, 3, 4, 8)
for call in (lambda: policy.gated_delta_rule(x, x, x, x[..., 0], x[..., 0]), lambda: policy.clip_grad_norm([x], 1.0),
             lambda: policy.orthogonalize([x[0, 0]]),
             lambda: policy.selective_scan(x, x[..., 0], x[0, 0, :, 0], x, x), lambda: policy.causal_conv(x[0], x[0, 0]),
             lambda: policy.selective_scan_step(x[0], x[0, ..., 0], x[0, 0, :, 0], x[0], x[0], x),
             lambda: policy.causal_conv_step(x[0, 0], x[0, 0], x[0]), lambda: policy.block_norm(x[0], x[0])):
    try:
        call()
        print("done")
    except RuntimeError as e:
        print(str(e).splitlines()[0])
"""


def package(tmp_path, extension):
    """A copy of the package with the library alone, or with an `extension` beside it."""
    shutil.copytree(ROOT / "navi_amd", tmp_path / "navi_amd", ignore=shutil.ignore_patterns("_lib", "csrc", "__pycache__"))
    lib = tmp_path / "navi_amd" / "_lib"
    lib.mkdir()
    for name in ("libnavi_policy.so", "libnavi_trace.so", "libnavi_scene.so"):
        (lib / name).symlink_to(ROOT / "navi_amd" / "_lib" / name)
    if extension is not None:
        (lib / "_policy_calls.so").write_bytes(extension)
    return tmp_path


def run(root, **more):
    env = {k: v for k, v in os.environ.items() if k not in ("NAVI_POLICY_LIB", "PYTHONPATH")}
    return subprocess.run([sys.executable, "-c", PROGRAM], cwd=root, env={**env, **more}, capture_output=True, text=True)


@pytest.mark.parametrize("extension", [None, b"not a library"], ids=["none", "another"])
def test_without_the_extension(tmp_path, extension):
    """The older operators and orthogonalize look their arguments over as ever; the others say what is not there."""
    done = run(package(tmp_path, extension))
    assert done.returncode == 0, done.stderr
    lines = done.stdout.splitlines()
    assert lines[0] == "True"
    for said in lines[1:4]:
        assert "CUDA" in said
    assert len(lines) == 9
    for said in lines[4:]:
        assert "_policy_calls.so" in said and "make -C" in said


def test_with_a_library_of_the_users_own(tmp_path):
    done = run(package(tmp_path, None), NAVI_POLICY_LIB=str(ROOT / "navi_amd" / "_lib" / "libnavi_policy.so"))
    assert done.returncode == 0 and done.stdout.startswith("True"), done.stderr


def test_without_the_library(tmp_path):
    root = package(tmp_path, None)
    (root / "navi_amd" / "_lib" / "libnavi_policy.so").unlink()
    done = run(root)
    assert done.returncode != 0 and "ImportError" in done.stderr and "libnavi_policy.so not found" in done.stderr


def test_the_build_takes_the_running_python(monkeypatch):
    """The extension is compiled against the PyTorch of the interpreter that builds, not of `python3` on the path."""
    import __graft_entry__ as entry

    made = []
    monkeypatch.setattr(entry.subprocess, "run", lambda command, check: made.append(command))
    entry._make(ROOT / "navi_amd" / "csrc" / "policy")
    assert f"PYTHON={sys.executable}" in made[0]
    makefile = (ROOT / "navi_amd" / "csrc" / "policy" / "Makefile").read_text()
    assert "$(PYTHON) -c" in makefile
