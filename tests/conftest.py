"""pytest configuration: import paths and the ``gpu`` marker.

``gpu`` marks tests that need a HIP device (the reference's convention, pyproject.toml:38-41); without one they are
skipped, whatever else their file says.
"""

from __future__ import annotations

import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
for path in (ROOT / "moss-image_amd", ROOT):
    if str(path) not in sys.path:
        sys.path.insert(0, str(path))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: requires a HIP device (MI355X)")


def pytest_collection_modifyitems(items):
    marked = [item for item in items if item.get_closest_marker("gpu")]
    if not marked:
        return
    import torch

    if not torch.cuda.is_available():
        for item in marked:
            item.add_marker(pytest.mark.skip(reason="requires a HIP device"))
