"""More of the packed-sequence operators on the IEEE-half flavour of the library, in a child process (one 16-bit format a
process): what tests/test_packed_fp16_gpu.py runs at one head size or with one set of heads only, the norms of output and
gradients, and the edges."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


def test_half_flavour_at_other_sizes():
    env = dict(os.environ, MELGPT_HALF="fp16")
    env.pop("MELGPT_LAB_LIB", None)
    r = subprocess.run([sys.executable, os.path.join(HERE, "packed_fp16_more_worker.py")], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "all ok" in r.stdout, (r.returncode, r.stdout[-800:], r.stderr[-3000:])
