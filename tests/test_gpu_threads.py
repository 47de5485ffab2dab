"""First calls from several host threads."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.parametrize("what", ["scored", "fused"])
def test_first_calls_of_several_threads(what):
    """Threads with batches of different sizes set the same kernel up at the same time: no launch is refused then or later."""
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    run = subprocess.run([sys.executable, os.path.join(HERE, "threads_driver.py"), what], capture_output=True, text=True, timeout=300,
                         env=dict(os.environ, PYTHONPATH=HERE))
    assert run.returncode == 0, run.stdout[-500:] + run.stderr[-1500:]
