"""The training example as it is run."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_loss_falls():
    r = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "train_block.py"), "--steps", "40"], capture_output=True, text=True, timeout=300, cwd="/")
    assert r.returncode == 0, r.stderr
    first, last = (float(v) for v in r.stdout.strip().splitlines()[-1].removeprefix("loss ").split(" -> "))
    assert last < 0.5 * first
