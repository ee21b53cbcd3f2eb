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


@pytest.mark.parametrize("missing", ["g++", "torch", "Python.h", "torch's headers"])
def test_the_library_builds_without_what_the_direct_calls_need(missing, monkeypatch, tmp_path, capsys):
    """hipcc is enough for libcapdec.so; direct calls of older sources, which cannot be made anew then, go."""
    import shutil
    import sysconfig
    import torch
    from imagecaption_amd import build
    run = subprocess.run

    def only_gxx(cmd, **kw):
        assert cmd[0] == "g++", cmd  # the library itself is up to date
        return run(cmd, **kw)

    shutil.copy(os.path.join(build.CSRC, "calls.cpp"), tmp_path)
    for name in ("a.hip", "a.o", "libcapdec.so", "_calls.so"):
        (tmp_path / name).write_bytes(b"")
    os.utime(tmp_path / "_calls.so", (1, 1))
    for name, at in (("CSRC", ""), ("OBJ", ""), ("LIB", "libcapdec.so"), ("CALLS", "_calls.so")):
        monkeypatch.setattr(build, name, str(tmp_path / at))
    monkeypatch.setattr(build, "_hipcc", lambda: "hipcc")
    monkeypatch.setattr(build.subprocess, "run", only_gxx)
    if missing == "g++":
        monkeypatch.setenv("PATH", str(tmp_path))
    elif missing == "torch":
        monkeypatch.setitem(sys.modules, "torch", None)
    elif missing == "Python.h":
        monkeypatch.setattr(sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    else:
        monkeypatch.setattr(torch, "__file__", str(tmp_path / "__init__.py"))
    assert build.build() == str(tmp_path / "libcapdec.so")
    assert not (tmp_path / "_calls.so").exists() and missing in capsys.readouterr().out


def test_direct_calls_that_fit_stay_without_a_compiler(monkeypatch, tmp_path):
    from imagecaption_amd import build
    if not build.calls_fit():
        pytest.skip("the direct calls are not built")
    with open(build.CALLS, "rb") as f:
        (tmp_path / "_calls.so").write_bytes(f.read())
    monkeypatch.setattr(build, "CALLS", str(tmp_path / "_calls.so"))
    monkeypatch.setenv("PATH", str(tmp_path))
    build.build_calls()
    assert (tmp_path / "_calls.so").exists() and build.calls_fit()


def test_direct_calls_that_do_not_compile_are_an_error(monkeypatch, tmp_path):
    from imagecaption_amd import build
    monkeypatch.setattr(build, "CALLS", str(tmp_path / "_calls.so"))
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **kw: subprocess.CompletedProcess(cmd, 1, "", "no such thing"))
    with pytest.raises(RuntimeError, match="no such thing"):
        build.build_calls(verbose=False)
