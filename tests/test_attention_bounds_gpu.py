"""The bounds-checking build checks what the attention training operators write beside their results (row
statistics, scratch, pieces, partial weight gradients), as its header promises: an access beyond the extent is
skipped and reported.  The extents are capped below the buffers' sizes; nothing is ever out of bounds."""
import json
import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def report(cuda_device):
    from kernelcodegen_b200 import build

    build.build_bounds()
    res = subprocess.run([sys.executable, str(ROOT / "tests" / "_bounds_train_child.py")], env=dict(os.environ, KCG_DEBUG_BOUNDS="1"),
                         capture_output=True, text=True, timeout=600)
    assert res.returncode == 0, res.stdout[-2000:] + res.stderr[-3000:]
    return json.loads(res.stdout.strip().splitlines()[-1])


@pytest.mark.parametrize("what", ["lse", "stat", "dw", "dw_pairs"])
def test_accesses_beyond_the_extent_are_skipped_and_reported(report, what):
    r = report[what]
    assert report["enabled"] == 1
    assert r["plain"] == [0, 0] and r["capped"] == [0, 10], r      # status of the call, of the device (DEV_BOUNDS)
    assert r["kept"] and r["untouched"], r


@pytest.mark.parametrize("what", ["pieces", "pieces_q"])
def test_pieces_beyond_the_extent_are_skipped_and_reported(report, what):
    r = report[what]
    assert r["bytes"] > 2 * r["cap"], r                            # the scratch is what the cap cuts
    assert r["plain"] == [0, 0] and r["capped"] == [0, 10] and r["extent"] == r["cap"], r
    assert r["after"] == [0, 0] and r["same"], r
