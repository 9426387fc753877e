"""CPU: what depends on the compiled torch binding of the node features, and when it is built again."""
import importlib.util
import json
import os
import subprocess
import sys
from pathlib import Path

import pytest

PKG = Path(__file__).resolve().parents[1] / "lanczos-gpu_b200"


def python(code):
    return subprocess.run([sys.executable, "-c", f"import sys; sys.path.insert(0, {str(PKG)!r})\n{code}"],
                          capture_output=True, text=True)


def test_other_modules_import_without_the_binding():
    """Where it is missing or does not load, what does not call it works."""
    res = python("sys.modules['gpu_eigsh.features'] = None   # an import of it raises\n"
                 "import gpu_eigsh, gpu_eigsh.graph, gpu_eigsh.imgp, gpu_eigsh.imgp_train, gpu_eigsh.differentiable\n"
                 "import gpu_eigsh.ordering, gpu_eigsh.funm_torch, gpu_eigsh.distributed\n"
                 "from gpu_eigsh import differentiable_eigsh\n")
    assert res.returncode == 0, res.stderr


@pytest.fixture()
def build(tmp_path, monkeypatch):
    """build.py with a binding in tmp_path whose compilation adds a byte to it."""
    spec = importlib.util.spec_from_file_location("_build_under_test", PKG / "build.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    lib = tmp_path / "_torch_features.so"
    mod.TORCH_LIB, mod.TORCH_STAMP = lib, tmp_path / "_torch_features.json"
    mod.torch_binding_command = lambda: [sys.executable, "-c", f"open({str(lib)!r}, 'a').write('x')"]
    mod.runs = lambda: lib.stat().st_size
    return mod


def test_binding_is_built_again_when_torch_changes(build):
    build.build_torch_binding()
    build.build_torch_binding()
    assert build.runs() == 1
    stamp = build.TORCH_STAMP.read_text()
    for k, change in enumerate(("torch", "python", "compiler", "command")):
        build.TORCH_STAMP.write_text(json.dumps({**json.loads(stamp), change: "another"}, indent=1))
        build.build_torch_binding()
        assert build.runs() == 2 + k and build.TORCH_STAMP.read_text() == stamp, change
        build.build_torch_binding()
        assert build.runs() == 2 + k
    build.TORCH_STAMP.unlink()
    build.build_torch_binding()
    assert build.runs() == 6
    os.utime(build.TORCH_LIB, (1, 1))   # older than the sources
    build.build_torch_binding()
    assert build.runs() == 7
    build.build_torch_binding(force=True)
    assert build.runs() == 8


def test_a_failed_build_is_tried_again(build):
    good = build.torch_binding_command
    build.build_torch_binding()
    build.torch_binding_command = lambda: [sys.executable, "-c", "raise SystemExit(3)"]
    for _ in range(2):
        with pytest.raises(RuntimeError, match="features.cpp"):
            build.build_torch_binding()
    build.torch_binding_command = good
    assert build.runs() == 1 and not build.TORCH_STAMP.exists()
    build.build_torch_binding()   # the same command as the last good one, whose library may be overwritten in part
    assert build.runs() == 2


def test_a_binding_for_another_torch_is_refused(tmp_path):
    from gpu_eigsh import features

    lib = tmp_path / "_torch_features.so"
    with pytest.raises(ImportError, match="missing; build it"):
        features._load(lib)
    lib.write_text("not a library")
    with pytest.raises(ImportError, match="does not load"):
        features._load(lib)
    lib.with_suffix(".json").write_text(json.dumps({"torch": "1.0"}))
    with pytest.raises(ImportError, match="built for torch 1.0, this is"):
        features._load(lib)
