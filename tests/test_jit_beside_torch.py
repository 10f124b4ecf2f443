"""A program that imports torch first has torch's own HIP libraries, whose compiler may not know every option of this build: kernels for
unlisted shapes compile there all the same, and before torch's libraries are loaded as well. Each order in a process of its own."""
import subprocess
import sys

import pytest

CODE = """
{first}
from neural_block_textures_amd.trainer import PK_LV1LOCAL, Layout, Trainer
{second}
for layout in (Layout(32, 32, [(8, 8, 4, False)], [20, 12]),
               Layout(48, 40, [(48, 40, 2, True), (12, 10, 4, False)], [28, 28], T=4, pos=[PK_LV1LOCAL], leak=0.0)):
    sec, why = Trainer.jit_compile_check(Trainer.model_desc(layout))
    assert sec is not None, why
print("both compiled")
"""


@pytest.mark.parametrize("first,second", [("import torch", ""), ("", "from neural_block_textures_amd import ops"), ("", "")], ids=["torch_first", "torch_second", "no_torch"])
def test_shapes_compile(first, second):
    run = subprocess.run([sys.executable, "-c", CODE.format(first=first, second=second)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "both compiled" in run.stdout, (run.returncode, run.stderr[-1500:])
