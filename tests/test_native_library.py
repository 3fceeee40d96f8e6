"""Both bindings call one library: the one that load_library was given (no launch)."""
import shutil
import subprocess
import sys

from conftest import PKG

_CHILD = r"""
import os, sys
sys.path.insert(0, sys.argv[1])
from epure import _native
os.chdir(os.path.dirname(sys.argv[2]))
_native.load_library(os.path.basename(sys.argv[2]))
_native.load_tensor_calls()
with open("/proc/self/maps") as f:
    print("MAPPED", sorted({line.split()[-1] for line in f if "libepq" in line and line.split()[-1].endswith(".so")}))
"""


def test_tensor_calls_use_the_library_that_was_loaded(tmp_path):
    from epure import _native
    other = tmp_path / "libepq_other.so"
    shutil.copy(_native.LIB_PATH, other)
    r = subprocess.run([sys.executable, "-c", _CHILD, PKG, str(other)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and f"MAPPED ['{other}']" in r.stdout, r.stdout + r.stderr[-2000:]
