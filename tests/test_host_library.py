"""The library that is built with one PyTorch: what does not go through it needs none of it."""
import os
import shutil
import subprocess
import sys

import pytest

from conftest import PKG, ROOT

CALLS = """
import torch
g, x, w = torch.zeros(8), torch.zeros(2, 64, dtype=torch.bfloat16), torch.ones(8, 64, dtype=torch.bfloat16)
calls = [lambda: m.gradient_norm([g]), lambda: m.clip_gradients([g], 1.0), lambda: m.rms_norm(x, w[0]),
         lambda: m.rms_norm_quantized(x, w[0]), lambda: m.grouped_linear(x, w)]
for call in calls:
    try:
        call()
    except ImportError as e:
        assert "build.py" in str(e) and SAID in str(e), e
    else:
        raise SystemExit("no refusal")
"""


def run(at, code):
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([str(at), ROOT]))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, env=env, cwd=ROOT)
    assert r.returncode == 0, r.stderr


@pytest.fixture()
def package_without(tmp_path, built_library):
    shutil.copytree(os.path.join(PKG, "sonicmoe"), tmp_path / "sonicmoe", ignore=shutil.ignore_patterns("*.so", "__pycache__"))
    os.symlink(built_library, tmp_path / "sonicmoe" / "libsmoe_b200.so")
    return tmp_path


def test_the_package_is_imported_without_it(package_without):
    """Routing on the host, the C ABI and refusals of the other operators are there; the calls that need it say what to do."""
    run(package_without, "import sonicmoe as m\nfrom sonicmoe._lib import lib\nassert m.__file__.startswith(%r)\n" % str(package_without)
        + "assert lib.smoe_gradient_workspace(-1) == -1 and callable(m.run_sonic_moe)\nSAID = '_host.so'\n" + CALLS)


def test_that_of_another_pytorch_is_refused():
    run(PKG, "import torch\ntorch.__version__ = '1.0'\nimport sonicmoe as m\nSAID = 'PyTorch'\n" + CALLS)


def test_it_is_loaded_once(built_library):
    from sonicmoe._lib import host
    assert host.torch_version and "grouped_call" in vars(host)
    with pytest.raises(AttributeError):
        host.no_such_function
