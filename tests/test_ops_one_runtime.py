"""torch and the kernels' library share one HIP runtime, or the operators refuse to run: each order of loading in a process of its own."""
import subprocess
import sys

import pytest

CODE = """
{first}
from neural_block_textures_amd import ops, trainer
{second}
try:
    ops._binding()
except RuntimeError as e:
    print("refused:", e)
else:
    print("bound")
print(len({{x.split()[-1] for x in open("/proc/self/maps") if "libamdhip64" in x}}), "runtimes")
try:
    ops._binding()
except RuntimeError:
    print("refused again")
"""


@pytest.mark.parametrize("first,second", [("import torch", ""), ("import torch", "trainer.library()"), ("from neural_block_textures_amd import ops", "trainer.library()"),
                                          ("", "trainer.library()")])
def test_torch_first(first, second):
    run = subprocess.run([sys.executable, "-c", CODE.format(first=first, second=second)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.splitlines() == ["bound", "1 runtimes"], (run.stdout, run.stderr[-1500:])


def test_the_library_first():
    first = "from neural_block_textures_amd import trainer\ntrainer.library()"
    run = subprocess.run([sys.executable, "-c", CODE.format(first=first, second="")], capture_output=True, text=True, timeout=300)
    lines = run.stdout.splitlines()
    if lines[1:2] == ["1 runtimes"]:
        pytest.skip("torch's libraries and the system's have the same runtime here")
    assert run.returncode == 0 and lines[0].startswith("refused: two HIP runtimes") and lines[1:] == ["2 runtimes", "refused again"], (run.stdout, run.stderr[-1500:])
