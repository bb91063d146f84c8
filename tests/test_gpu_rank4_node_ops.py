"""The node-wise operators with the library for ranks up to 4, which carries their kernels too. The library is chosen at
import, so the checks run in a process of their own; skipped when it has not been built
(``FLASHCART_KERNEL_L_MAX=4 python -m flashcart_amd.build``)."""

import os
import subprocess
import sys

import pytest

from flashcart_amd import _lib

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CHECKS = """
from flashcart_amd import _lib
from tests import test_gpu_embedding_paths as P, test_gpu_feed_forward as T, test_gpu_node_ops as N

for dtype in T.DTYPES:
    T.test_feed_forward(257, 519, 103, dtype)
    N.test_embedding(2049, 257, 19, "uniform", dtype)
    N.test_dropout(4101, 0.3, dtype)
    P.test_gradient_is_exact("few rows", dtype)
with open("/proc/self/maps") as fh:
    maps = fh.read()
assert _lib.library_path(4) in maps and _lib.library_path(3) not in maps
print("all node-wise checks passed")
"""


@pytest.mark.skipif(not os.path.exists(_lib.library_path(4)),
                    reason="libflashcart_hip_l4.so not built (FLASHCART_KERNEL_L_MAX=4 python -m flashcart_amd.build)")
def test_node_operators_of_the_rank4_library():
    res = subprocess.run([sys.executable, "-u", "-c", CHECKS], env=dict(os.environ, FLASHCART_KERNEL_L_MAX="4"),
                         capture_output=True, text=True, timeout=100, cwd=ROOT)
    print(res.stdout[-4000:])
    assert res.returncode == 0, res.stdout[-3000:] + res.stderr[-3000:]
    assert "all node-wise checks passed" in res.stdout
