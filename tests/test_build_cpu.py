"""The CUDA library builds and its C ABI is there without torch; only the binding needs it."""

import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_library_builds_without_torch():
    code = """
import sys
class NoTorch:
    def find_spec(self, name, path=None, target=None):
        if name == "torch" or name.startswith("torch."):
            raise ModuleNotFoundError("No module named 'torch'", name="torch")
sys.meta_path.insert(0, NoTorch())
from moat_b200 import _lib, build
assert build.build() == build.LIB
assert _lib.lib().mb_abi_version() > 0
assert build.build_bind() is None
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
