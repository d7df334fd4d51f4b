"""Which attention kernels of the 8-bit cache with block scales are built."""
import re

import pytest

from test_kernel_resources import metadata  # noqa: F401  (a fixture)

pytest.importorskip("msgpack")


def test_no_kernel_is_built_that_no_call_reaches(metadata):  # noqa: F811
    """Blocks of whole groups of 8 tokens divide their pages, which are whole
    groups then; of other blocks both kinds of pages are there."""
    found = {}
    for name in metadata:
        m = re.search(r"block_attend_kernelINS_11BlockEngineI.*ELb([01])EEELb([01])ELb[01]EEE", name)
        if m:
            found.setdefault(m.groups(), []).append(name)
    assert sorted(found) == [("0", "1"), ("1", "0"), ("1", "1")]  # (a scale a token, pages of whole groups)
    assert len({len(names) for names in found.values()}) == 1
