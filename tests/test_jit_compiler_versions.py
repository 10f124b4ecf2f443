"""Which options kernels for unlisted shapes are compiled with follows from the compiler in use: those of the build's version get all, older and newer
ones, and ones that do not say, only what every compiler knows. (The installed compiler, as a copy in an installation of another version; what it was
asked for is in its own log.)"""
import os
import shutil
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
COMGR, VERSION = "/opt/rocm/lib/libamd_comgr.so.3", "/opt/rocm/.info/version"
CODE = """
import ctypes, sys
ctypes.CDLL(sys.argv[1], ctypes.RTLD_GLOBAL)
from neural_block_textures_amd.trainer import Layout, Trainer
sec, why = Trainer.jit_compile_check(Trainer.model_desc(Layout(32, 32, [(8, 8, 4, False)], [20, 12])))
assert sec is not None, why
assert {x.split()[-1] for x in open("/proc/self/maps") if "libamd_comgr" in x} == {sys.argv[1]}
"""


@pytest.fixture(scope="module")
def installation(tmp_path_factory):
    if not os.path.exists(COMGR) or not os.path.exists(VERSION):
        pytest.skip("no installation of the compiler here")
    root = tmp_path_factory.mktemp("rocm")
    (root / "lib").mkdir()
    (root / ".info").mkdir()
    shutil.copy(os.path.realpath(COMGR), root / "lib" / "libamd_comgr.so.3")
    yield root
    shutil.rmtree(root)


@pytest.mark.parametrize("version", ["same", "older", "newer", None])
def test_options(installation, version, tmp_path):
    major, minor = (int(x) for x in open(VERSION).read().split(".")[:2])
    text = {"same": f"{major}.{minor}.9", "older": f"{major - 1}.{minor + 1}.0", "newer": f"{major}.{minor + 1}.0", None: None}[version]
    at = installation / ".info" / "version"
    at.write_text(text) if text else at.unlink(missing_ok=True)
    env = {**os.environ, "AMD_COMGR_EMIT_VERBOSE_LOGS": "1", "AMD_COMGR_REDIRECT_LOGS": "stderr", "NTC_HIP_JIT_CACHE": str(tmp_path)}
    run = subprocess.run([sys.executable, "-c", CODE, str(installation / "lib" / "libamd_comgr.so.3")], capture_output=True, text=True, timeout=300, env=env, cwd=HERE)
    assert run.returncode == 0, run.stderr[-1500:]
    assert "-packed-fp32-ops" in run.stderr                  # the log is there
    assert ("amdgpu-mfma-vgpr-form" in run.stderr) == (version == "same")
