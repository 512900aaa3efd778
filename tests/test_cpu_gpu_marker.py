"""Without a HIP device every test that needs one is skipped, also in a plain run that selects no marker."""

from __future__ import annotations

import os
import re
import subprocess
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent


def test_marked_tests_are_skipped_without_a_device() -> None:
    bare = sorted(p.name for p in HERE.glob("test_gpu_*.py") if re.search(r"^pytestmark = pytest\.mark\.gpu$", p.read_text(), re.M))
    assert "test_gpu_many_rows.py" in bare
    run = subprocess.run([sys.executable, "-m", "pytest", "-q", "-p", "no:cacheprovider", *bare], cwd=HERE, capture_output=True, text=True,
                         env={**os.environ, "HIP_VISIBLE_DEVICES": "-1", "CUDA_VISIBLE_DEVICES": "-1"})
    assert run.returncode == 0, run.stdout[-2000:]
    assert re.search(r"^\d+ skipped", run.stdout.splitlines()[-1]), run.stdout[-500:]
