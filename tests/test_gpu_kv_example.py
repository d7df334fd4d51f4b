"""GPU: the decode loop of examples/paged_decode.py at other lengths and pool
sizes than its first ones."""
import sys
from pathlib import Path

import pytest

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))

pytestmark = pytest.mark.gpu

PROMPTS = [[1, 2, 3], [10, 11, 12, 13, 14], [7], [5, 6]]


@pytest.mark.parametrize("steps", [17, 100, 130])
def test_any_number_of_steps_has_room(sampler, steps):
    """Every step's tokens reach the cache: lengths and pages say so."""
    import paged_decode

    lens = []
    out, m = paged_decode.generate(sampler, PROMPTS, steps, on_step=lambda t, h: lens.append(m_lens(t)), make=Kept)
    assert [len(o) for o in out] == [steps] * 4
    assert lens == [[t + 1] * 4 for t in range(steps)]


class Kept:
    """Builds the example's decoder and remembers it."""

    last = None

    def __new__(cls, *args, **kwargs):
        import paged_decode

        cls.last = paged_decode.Decoder(*args, **kwargs)
        return cls.last


def m_lens(t):
    return Kept.last.lens.tolist()


def test_a_pool_without_room_is_an_error(sampler):
    import paged_decode

    with pytest.raises(RuntimeError, match="room"):
        paged_decode.generate(sampler, PROMPTS, 40, pages=5)
    with pytest.raises(RuntimeError, match="room"):
        paged_decode.generate(sampler, PROMPTS, 40, context=32)
    # Four requests of 40 tokens are three pages each.
    paged_decode.generate(sampler, PROMPTS, 40, pages=12, context=48)
