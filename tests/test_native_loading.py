"""What loading liblfm_hip.so does to the process (no device needed)."""
import ast
import importlib.util
import os
import subprocess
import sys

import pytest

from lightfm_amd import _native

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SCRIPT = """
import sys
from lightfm_amd import _native
_native.lib()
%s
print(sorted(set(line.split()[-1] for line in open("/proc/self/maps") if "hsa-runtime" in line)))
"""


def runtimes(more="", **env):
    out = subprocess.run([sys.executable, "-c", SCRIPT % more], cwd=ROOT, env=dict(os.environ, **env), capture_output=True,
                         text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    return ast.literal_eval(out.stdout.strip().splitlines()[-1])


@pytest.fixture(scope="module", autouse=True)
def built():
    if not os.path.exists(_native.LIB_PATH):
        from lightfm_amd import build
        build.build()


def test_no_other_runtime_is_loaded(tmp_path):
    """A libhsa-runtime64.so of another installation that the loader would find first stays out of the process."""
    (tmp_path / "other.c").write_text("int other_runtime(void) { return 1; }\n")
    other = str(tmp_path / "libhsa-runtime64.so")
    subprocess.check_call(["gcc", "-shared", "-fPIC", "-o", other, str(tmp_path / "other.c")])
    path = os.pathsep.join([str(tmp_path)] + [p for p in [os.environ.get("LD_LIBRARY_PATH")] if p])
    loaded = runtimes(LD_LIBRARY_PATH=path)
    assert loaded == runtimes() and os.path.realpath(other) not in loaded
    if importlib.util.find_spec("torch"):
        assert other not in runtimes("import torch", LD_LIBRARY_PATH=path)


def test_a_torch_imported_later_shares_the_runtime():
    pytest.importorskip("torch")
    if "libhsa-runtime64.so" not in os.listdir(os.path.dirname(os.path.realpath(runtimes()[0]))):
        pytest.skip("the runtime in use is not known under its plain name")
    assert len(runtimes("import torch")) == 1
