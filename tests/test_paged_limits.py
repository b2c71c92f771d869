"""What the paged cache's C entries refuse, on the CPU."""
from __future__ import annotations

import pytest

from diffusorrt_amd import _lib

pytestmark = pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="library not built")


def test_no_event_is_refused():
    assert _lib.load().drt_event_wait(None) == _lib.INVALID_ARGUMENT
