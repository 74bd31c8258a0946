"""The modules that import torch where they use it go on doing so."""
import subprocess
import sys
from pathlib import Path

import pytest


@pytest.mark.parametrize("module", ["lmhead", "moe", "quant"])
def test_import_leaves_torch_alone(module):
    code = f"import sys; import powerinfer_x64_b200.{module}; sys.exit('torch' in sys.modules)"
    assert subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parents[1]).returncode == 0
