"""The key-value cache's kernels as the compiler allocated them."""
import pytest

from test_kernel_resources import metadata  # noqa: F401  (a fixture)

pytest.importorskip("msgpack")


def _attend(metadata):  # noqa: F811
    return {n: k for n, k in metadata.items() if "attend_kernel" in n}


def test_attention_over_whole_groups_of_tokens_spills_nothing(metadata):  # noqa: F811
    """Pages that are whole groups of tokens: the ordinary ones."""
    found = {n: k for n, k in _attend(metadata).items() if "ELb1ELb1EEEvNS" in n or "ELb1ELb0EEEvNS" in n}
    assert len(found) >= 5 * 10
    assert {n: k[".vgpr_spill_count"] for n, k in found.items() if k[".vgpr_spill_count"]} == {}


def test_attention_kernels_fit_the_waves_that_are_launched(metadata):  # noqa: F811
    """8 waves of a workgroup are two on each SIMD: 256 registers each."""
    for name, k in _attend(metadata).items():
        waves = k[".max_flat_workgroup_size"] // 64
        assert waves in (4, 8)
        total = (k[".vgpr_count"] + 7) // 8 * 8
        assert total <= (512 if waves == 4 else 256), name


def test_the_other_kernels_spill_no_vector_register(metadata):  # noqa: F811
    found = {n: k for n, k in metadata.items() if any(x in n for x in ("append_kernel", "plan_kernel", "join_kernel"))}
    assert len(found) >= 20
    assert all(k[".vgpr_spill_count"] == 0 for k in found.values())
