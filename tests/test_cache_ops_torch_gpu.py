"""The torch binding of the cache operators on the GPU (streamtx.cache): a prompt and steps through two layers,
torch's current stream, a captured step, refusals. One child process, since torch brings its own HIP
runtime (tests/torch_cache_ops.py)."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


def test_torch_binding():
    script = Path(__file__).resolve().parent / 'torch_cache_ops.py'
    out = subprocess.run([sys.executable, '-u', str(script)], capture_output=True, text=True, timeout=110)
    print(out.stdout[-2000:], flush=True)
    assert out.returncode == 0 and out.stdout.strip().endswith('ok'), out.stderr[-3000:]
