"""The library is built with nvcc alone: without torch, whom the C ABI does not
need, the build leaves out the torch binding and says so."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CODE = """
import os, sys, importlib.abc
class Gone(importlib.abc.MetaPathFinder):
    def find_spec(self, name, path, target=None):
        if name.split('.')[0] == 'torch':
            raise ModuleNotFoundError("No module named 'torch'", name='torch')
sys.meta_path.insert(0, Gone())
from inferc_b200 import build
build._compile = lambda src, force, verbose: src      # nothing is compiled or linked here
build.subprocess.run = lambda cmd, **kw: print('ran', os.path.basename(cmd[0]))
build._stale = lambda target, sources: True
print('built', os.path.basename(build.build()))
"""


def test_build_without_torch():
    r = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert r.stdout.split() == ["ran", "nvcc", "built", "libinferc_b200.so"]
    assert "torch" in r.stderr and "_paged" in r.stderr
