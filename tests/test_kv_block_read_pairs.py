"""llmhip_kv_block_read's two outputs in one memory, without a GPU: refused where
their rows lie over one another, taken where they lie beside one another."""
import numpy as np
import pytest
import torch

from scriptonait_amd import kv, kv_blocks
from test_kv_block_refusals import _cache, _make, _ref, _state
from test_kv_refusals import BAD, SOME, _refused

E = 2  # bytes of a bf16 value


def _read(c, k, v, k_st=(512, 64), v_st=(512, 64), T=2):
    return kv.load_kv().llmhip_kv_block_read(None, _ref(c), kv.BF16, T, SOME, k, *k_st, v, *v_st, None)


@pytest.mark.parametrize("k,v,k_st,v_st,T", [
    (SOME, SOME, (512, 64), (512, 64), 2), (SOME, SOME, (512, 64), (512, 64), 1),
    (SOME, SOME + E, (512, 64), (512, 64), 2), (SOME, SOME + 64 * E, (512, 64), (512, 64), 2),  # a value, a head on
    (SOME + 512 * E, SOME, (512, 64), (512, 64), 2),  # a token on
    (SOME, SOME + 63 * E, (2048, 128), (2048, 128), 3), (SOME, SOME + 65 * E, (2048, 128), (2048, 128), 3),
    (SOME, SOME + 512 * E, (1023, 64), (1023, 64), 3), (SOME, SOME + 512 * E - 1, (1024, 64), (1024, 64), 3),
    (SOME, SOME + 511 * E, (512, 64), (512, 64), 1), (SOME, SOME + 64, (1024, 64), (2048, 64), 2)])
def test_rows_over_one_another_are_refused(k, v, k_st, v_st, T):
    c = _cache()
    _refused(_read(c, k, v, k_st, v_st, T), BAD, "out_k and out_v overlap")
    _refused(_read(c, v, k, v_st, k_st, T), BAD, "out_k and out_v overlap")


@pytest.mark.parametrize("k,v,k_st,v_st,T", [
    (SOME, SOME + 1024 * E, (512, 64), (512, 64), 2), (SOME, SOME + 512 * E, (512, 64), (2048, 128), 1),
    (SOME, SOME + 512 * E, (1024, 64), (1024, 64), 1000),  # values behind a token's keys
    (SOME, SOME + 64 * E, (1024, 128), (1024, 128), 1000),  # or behind each head's
    (SOME, SOME + 512 * E, (1088, 64), (1088, 64), 5),  # in wider rows
    (SOME, SOME + (1024 + 512) * E, (1024, 64), (1024, 64), 5),  # the next token's
    (SOME, SOME + 64 * E, (128, 256), (128, 256), 2),  # heads before tokens, keys beside values
    (SOME, SOME + 512 * 1000 * E, (512, 64), (64, 64000), 1000)])
def test_rows_beside_one_another_are_taken(k, v, k_st, v_st, T):
    c = _cache()
    _refused(_read(c, k, v, k_st, v_st, T), BAD, "ctx")
    _refused(_read(c, v, k, v_st, k_st, T), BAD, "ctx")


def test_all_small_layouts():
    """Of every two places in a small array with these strides, the refused ones
    are those whose rows meet."""
    c = _cache(heads=2, head_dim=8, k_stride=(kv.ctypes.c_int64 * 3)(8192, 512, 64))
    T, seen = 3, set()
    for st in [(16, 8), (32, 8), (32, 16), (40, 8), (8, 24), (16, 56), (48, 16), (24, 96)]:
        at = (np.arange(T)[:, None, None] * st[0] + np.arange(2)[None, :, None] * st[1] + np.arange(8)).ravel()
        assert len(set(at)) == len(at)
        for apart in range(0, 220):
            meet = bool(set(at) & set(at + apart))
            status = _read(c, SOME, SOME + apart * E, st, st, T)
            refused = "overlap" in kv.load_kv().llmhip_last_error().decode()
            assert status == BAD and refused == meet, (st, apart)
            seen.add(meet)
    assert seen == {True, False}


def test_mirror():
    c = _make(*_state())
    c._read = lambda *a: kv.load_kv().llmhip_kv_block_read(None, *a[1:])
    kv_blocks_current, kv_blocks._current = kv_blocks._current, lambda device: 0
    try:
        slots, x = torch.zeros(3, dtype=torch.int64), torch.zeros(3, 5, 64)
        for k, v in ((x[:, :2], x[:, :2]), (x[:, :2], x[:, 1:3])):
            with pytest.raises(ValueError, match="overlap"):
                c.read(slots, k, v)
    finally:
        kv_blocks._current = kv_blocks_current
