"""Building and loading the direct calls (csrc/calls.cpp -> _calls.so), which are optional: no compute, no GPU."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT


def _fast(before):
    """What _capi.lib() took as the direct calls in a new interpreter that runs `before` first."""
    code = f"import torch; {before}; from imagecaption_amd import _capi; _capi.lib(); print(_capi.fast is not None)"
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    return r.stdout.strip() == "True"


def test_direct_calls_built_for_another_torch_are_not_loaded():
    """They read torch's objects by their layout, which an import does not check."""
    if not _fast("pass"):
        pytest.skip("the direct calls are not built")
    assert not _fast("torch.__version__ = '1.0.0'")
    assert not _fast("torch.version.git_version = 'another'")


def test_direct_calls_built_for_another_torch_are_built_again(monkeypatch, tmp_path):
    import torch
    from imagecaption_amd import build
    runs = []

    def run(cmd, **kw):
        runs.append(cmd)
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build, "CALLS", str(tmp_path / "_calls.so"))
    if not os.path.exists(os.path.join(ROOT, "imagecaption_amd", "_calls.so")):
        pytest.skip("the direct calls are not built")
    with open(os.path.join(ROOT, "imagecaption_amd", "_calls.so"), "rb") as f:
        (tmp_path / "_calls.so").write_bytes(f.read())  # newer than its sources
    monkeypatch.setattr(build.subprocess, "run", run)
    build.build_calls(verbose=False)
    assert not runs
    monkeypatch.setattr(torch, "__version__", "1.0.0")
    build.build_calls(verbose=False)
    assert len(runs) == 1
