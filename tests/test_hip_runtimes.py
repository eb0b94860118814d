"""torch's tensors are taken only where torch and the library run on one HIP runtime,
whichever of the two was loaded first.  CPU only, each order in a process of its own."""
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]

CALL = """
import sys
sys.path[:0] = [{root!r}, {tests!r}]
{imports}
import torch
from tatara_amd import _lib, ops
from test_learned_ops_devices import Elsewhere

class Here(Elsewhere):
    def get_device(self):
        return 0

torch.cuda.is_initialized = lambda: True
torch._C._cuda_getDevice = lambda: 0
torch._C._cuda_getCurrentRawStream = lambda device: 0
_lib._LIB.tatara_get_device = lambda p: 0  # device 0 of a machine that may have none
calls = []
norm = ops.LayerNorm(8)
norm._lib = type("Lib", (), dict(tatara_op_layer_norm_forward=lambda self, *a: calls.append(a) or 0))()
x = Here(3, 8)
try:
    norm.forward(x, None, None, x)
    print("taken", len(calls))
except RuntimeError as e:
    print("refused", len(calls), e)
"""


def run(imports):
    code = CALL.format(root=str(ROOT), tests=str(ROOT / "tests"), imports=imports)
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr
    return res.stdout


def two_runtimes_exist():
    torch = pytest.importorskip("torch")
    return (Path(torch.__file__).parent / "lib" / "libamdhip64.so").exists()


def test_torch_first():
    assert run("import torch; from tatara_amd import _lib; _lib.load()").startswith("taken 1")


def test_library_first():
    if not two_runtimes_exist():
        pytest.skip("torch brings no HIP runtime of its own")
    out = run("from tatara_amd import _lib; _lib.load()")
    assert out.startswith("refused 0") and "import torch before" in out
