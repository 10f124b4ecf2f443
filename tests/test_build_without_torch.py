"""The library is built without torch too: its binding alone is left out. (The compilers are stood in for; what they are asked for is looked at.)"""
import subprocess
import sys

import pytest

CODE = """
import importlib.abc, sys
class NoTorch(importlib.abc.MetaPathFinder):
    def find_spec(self, name, path=None, target=None):
        if name == "torch" or name.startswith("torch."):
            raise ModuleNotFoundError(f"No module named {{name!r}}", name=name)
if {hidden}:
    sys.meta_path.insert(0, NoTorch())
    import importlib.util
    found = importlib.util.find_spec
    importlib.util.find_spec = lambda name, *a: None if name == "torch" else found(name, *a)
from neural_block_textures_amd import build as b
import types
b.subprocess = types.SimpleNamespace(run=lambda cmd, **k: print("ran", cmd[-1] if "-shared" not in cmd else "shared " + cmd[cmd.index("-o") + 1]) or types.SimpleNamespace(returncode=0, stdout="", stderr=""))
b.os.replace = lambda a, c: print("made", c)
print("built", b.build())
"""


@pytest.mark.parametrize("hidden", [True, False])
def test_build(hidden):
    run = subprocess.run([sys.executable, "-c", CODE.format(hidden=hidden)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-1500:]
    made = [x for x in run.stdout.splitlines() if x.startswith("made")]
    assert len(made) == (1 if hidden else 2) and made[0].endswith("libntc_hip.so") and "built" in run.stdout
    assert ("binding" in run.stderr) == hidden and (hidden or made[1].endswith("_ops.so"))
