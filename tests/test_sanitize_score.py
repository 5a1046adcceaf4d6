"""The host half of the calls on scores (score_api.cpp) under AddressSanitizer and UndefinedBehaviorSanitizer, on the CPU:
argument checks on scalars of every size, planning over many shapes and workspaces, checks of host tables of exactly their
documented sizes, whole and broken.  See test_sanitize.py."""
import os
import subprocess

import pytest

from test_sanitize import KERNEL_OBJS, LIB_BUILD, SAN, _run

SCORE_OBJS = ["score_attention.o", "score_tiles.o", "score_weights.o", "score_evict.o"]


@pytest.mark.skipif(not os.path.exists("/opt/rocm/bin/hipcc"), reason="no hipcc")
def test_scores_host_half_under_sanitizers():
    if not all(os.path.exists(os.path.join(LIB_BUILD, o)) for o in KERNEL_OBJS + SCORE_OBJS):
        pytest.skip("build the library first (python -c 'import __graft_entry__ as g; g.build()')")
    if not os.path.isdir(SAN):
        pytest.skip("tests/sanitize is not present")
    r = subprocess.run(["make", "-C", SAN, "-f", "score.mk", "-j4", "_build/score_san"], capture_output=True, text=True,
                       timeout=600)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-3000:]
    _run(os.path.join(SAN, "_build/score_san"), leaks=False)
