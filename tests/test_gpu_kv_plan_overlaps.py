"""GPU: llmhip_kv_plan refuses outputs that overlap what its workgroups still
read, whichever two arguments they are. Nothing is launched then."""
import pytest

pytestmark = pytest.mark.gpu

R = T = 4
PAGES = 8
# int32 words of each argument's memory, and where it starts in the buffer.
WORDS = dict(lens=R, new_tokens=R, release=R, free_state=2, free_ring=PAGES, table=2 * R, out_lens=R, out_free_state=2, granted=R,
             start=R + 1, slots=2 * T, positions=T)
INPUTS = ("lens", "new_tokens", "release", "free_state", "free_ring", "table")
PLACES = {n: 16 * i for i, n in enumerate(WORDS)}


def _plan(sampler, places):
    import torch

    from scriptonait_amd.kv import PagePool

    x = torch.zeros(256, dtype=torch.int32, device="cuda")
    a = {n: x[at:at + WORDS[n]] for n, at in places.items()}
    a["table"], a["slots"] = a["table"].view(R, 2), a["slots"].view(torch.int64)
    pool = PagePool(sampler, PAGES, 16, a.pop("free_ring"), a.pop("free_state"))
    pool.free_state.copy_(torch.tensor([0, PAGES], dtype=torch.int32))
    pool.plan(**a)


# A read and a write that meet: ring and table are both.
PAIRS = [(a, b) for a in INPUTS for b in WORDS
         if a != b and (b not in INPUTS or {a, b} & {"free_ring", "table"})]


@pytest.mark.parametrize("first,second", PAIRS)
@pytest.mark.parametrize("shift", ["same", "end"])
def test_overlaps(sampler, first, second, shift):
    """`second` starts where `first` does, or in its last word."""
    from scriptonait_amd.sampler import SamplerError

    places = dict(PLACES)
    places[first] = 200
    places[second] = 200 if shift == "same" else 200 + WORDS[first] - 1
    if second == "slots" and places[second] % 2:
        places[second] -= 1
    if shift == "same" and (first, second) in (("lens", "out_lens"), ("free_state", "out_free_state")):
        _plan(sampler, places)
        return
    with pytest.raises(SamplerError, match="overlap"):
        _plan(sampler, places)


def test_neighbours_in_memory_are_served(sampler):
    at, places = 0, {}
    for n, words in sorted(WORDS.items(), key=lambda w: w[0] != "slots"):
        places[n] = at
        at += words
    _plan(sampler, places)
    sampler.status()
