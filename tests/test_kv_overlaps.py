"""Rows that lie over one another (expanded tensors, strides shorter than a
row) are no outputs: refused by the C entries and by the Python mirror, without
a GPU. As inputs they are ordinary."""
import ctypes

import pytest
import torch

from scriptonait_amd import kv

BAD = -1
SOME = 4096  # an address that no refused call follows


def _cache(k=(8192, 512, 64), v=(8192, 512, 64), pages=10, page=16, heads=8):
    return kv.LlmhipKvCache(SOME, SOME, None, None, (ctypes.c_int64 * 3)(*k), (ctypes.c_int64 * 3)(*v), kv.BF16, pages, page,
                            heads, 64)


def _append(cache, out=(512, 64), T=2, heads=8):
    st = (512, 64)
    return kv.load_kv().llmhip_kv_append(None, ctypes.byref(cache), kv.BF16, T, SOME, *st, SOME, *st, SOME, heads, SOME, *st, SOME,
                                         *out, None, None, None)


def _attend(cache, out=(512, 64), B=2):
    return kv.load_kv().llmhip_kv_attend(None, ctypes.byref(cache), kv.BF16, B, 8, SOME, 0, 0, SOME, 4, 4, SOME, 0, 0.1, SOME, *out,
                                         None, SOME, 1 << 40, None)


def _says(status, text):
    assert status == BAD
    assert text in kv.load_kv().llmhip_last_error().decode()


@pytest.mark.parametrize("stride", [0, 8, 63, -63])
def test_outputs_over_themselves(stride):
    c = _cache()
    for out in [(stride, 64), (512, stride)]:
        _says(_append(c, out), "out_q")
        _says(_attend(c, out), "out")
    # One row in a direction has no neighbour there; a row may end where the next one starts.
    _says(_append(c, (stride, 64), T=1), "ctx")
    _says(_attend(c, (stride, 64), B=1), "ctx")
    _says(_append(c, (64, 128)), "ctx")
    _says(_attend(c, (-512, -64)), "ctx")


@pytest.mark.parametrize("stride", [0, 8, 56])
@pytest.mark.parametrize("at", [0, 1, 2])
def test_pools_over_themselves(stride, at):
    strides = [8192, 512, 64]
    strides[at] = stride
    one = {("pages", "page", "heads")[at]: 1}
    for side in "kv":
        c = _cache(**{side: strides})
        _says(_append(c), "pool")
        _says(_attend(c), "ctx")  # reading them is no matter
        _says(_append(_cache(**{side: strides}, **one)), "ctx")


class _NoSampler:
    ctx = None


def test_mirror():
    pools = [torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16) for _ in range(2)]
    c = kv.KVCache(_NoSampler, *pools)
    x, q = torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    slots, lens = torch.zeros(3, dtype=torch.int64), torch.zeros(3, dtype=torch.int32)
    table, ws = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(256, dtype=torch.uint8)
    for wrong in [q[:1].expand(3, 4, 64), q[:, :1].expand(3, 4, 64),
                  torch.zeros(800, dtype=q.dtype).as_strided((3, 4, 64), (60, 180, 1))]:
        with pytest.raises(ValueError, match="out_q.*overlap"):
            c.append(x, x, slots, q=q, out_q=wrong)
        with pytest.raises(ValueError, match="out.*overlap"):
            c.attend(q, table, lens, wrong, ws)
        with pytest.raises(ValueError, match="not on a GPU"):
            c.attend(wrong, table, lens, q, ws)
    for i in range(2):
        for wrong in [p.expand(4, 16, 2, 64) for p in (pools[i][:1], pools[i][:, :1], pools[i][:, :, :1])]:
            p = list(pools)
            p[i] = wrong
            c = kv.KVCache(_NoSampler, *p)
            with pytest.raises(ValueError, match="pool.*overlap"):
                c.append(x, x, slots)
            with pytest.raises(ValueError, match="not on a GPU"):
                c.attend(q, table, lens, q.clone(), ws)
