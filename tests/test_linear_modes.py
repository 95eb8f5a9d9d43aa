"""Every kernel of moe_linear on every shape.

The library picks a kernel by the sizes: few tokens, tiles of 128 or 256 columns, CTA pairs,
k split over clusters.  MOE_LINEAR_TILE forces one, once per process, so the tests of
test_linear.py run again in a child process with each: whole-number inputs give the exact
bits in all of them, tails, odd sizes, strides and empty halves of a pair included.
"""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.parametrize("mode", ["few", "narrow", "wide", "pair", "pairn", "split2", "split4", "split8", "split2n", "split4n"])
def test_each_kernel(mode):
    env = dict(os.environ, MOE_LINEAR_TILE=mode)
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", "-m", "gpu", "-p", "no:cacheprovider",
                        os.path.join(HERE, "test_linear.py"), "-k", "exact or activations or strides or repeatable or rounded"],
                       cwd=os.path.dirname(HERE), env=env, capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stdout[-4000:] + r.stderr[-2000:]
