"""CPU: what depends on the compiled torch binding of the node features, and when it is built again."""
import subprocess
import sys
from pathlib import Path

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
