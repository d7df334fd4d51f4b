"""The attention kernels for pages that are no whole groups of tokens, as the
compiler allocated them."""
import pytest

from test_kernel_resources import metadata  # noqa: F401  (a fixture)

pytest.importorskip("msgpack")


def test_only_the_widest_binary32_heads_spill(metadata):  # noqa: F811
    """More than 192 values of binary32: 512 registers and 6 words beside them."""
    found = {n: k[".vgpr_spill_count"] for n, k in metadata.items() if "attend_kernel" in n and "ELb0ELb" in n}
    assert len(found) >= 5 * 8
    spilled = {n: v for n, v in found.items() if v}
    assert all("Engine32ILi256" in n and v <= 6 for n, v in spilled.items()), spilled
