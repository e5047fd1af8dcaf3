"""What the sources of the serving kernels must not say."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "l4-parakeet-rs_b200" / "csrc"
FILES = sorted(p.name for pattern in ("gemv_w4*", "paged_*", "rms_norm*", "element16*") for p in CSRC.glob(pattern))


@pytest.mark.parametrize("name", FILES)
def test_kernels_that_start_early_read_by_plain_loads(name):
    """Every one of these kernels may start while the one in front still writes what it reads.  The read-only path (`__ldg`, or a
    `const` pointer that is `__restrict__`) is for data that nobody writes while a kernel lives, and its loads may be moved."""
    text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    assert not re.search(r"__ldg\b|ld\.global\.nc|const[^;,()]*\*\s*__restrict__", text)
