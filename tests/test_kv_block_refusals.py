"""What the entries of the 8-bit cache refuse, without a GPU: the C entries
check their arguments before the context, the Python mirror before the call."""
import ctypes
import subprocess

import pytest
import torch

from scriptonait_amd import kv, kv_blocks
from test_kv_devices import _gpu1, _Sampler, _Stream
from test_kv_refusals import BAD, HEADER, SOME, UNSUPPORTED, _NoSampler, _refused

I8 = 4


def test_the_struct_is_the_headers(tmp_path):
    src = tmp_path / "a.c"
    src.write_text('#include "llmhip_kv.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(void) { printf("%zu %zu %zu %d\\n", '
                   "sizeof(llmhip_kv_blocks), offsetof(llmhip_kv_blocks, v_scale_stride), offsetof(llmhip_kv_blocks, block), "
                   "LLMHIP_I8); return 0; }\n")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", f"-I{HEADER.parent}", str(src), "-o", str(tmp_path / "a")], check=True)
    out = subprocess.run([str(tmp_path / "a")], check=True, capture_output=True, text=True).stdout.split()
    c = kv.LlmhipKvBlocks
    assert [int(x) for x in out] == [ctypes.sizeof(c), c.v_scale_stride.offset, c.block.offset, I8]
    assert kv_blocks.CODES[torch.int8] == I8


def _three(*x):
    return (ctypes.c_int64 * 3)(*x)


def _cache(**change):
    c = kv.LlmhipKvBlocks(SOME, SOME, SOME, SOME, _three(8192, 512, 64), _three(8192, 512, 64), _three(16, 8, 1), _three(16, 8, 1),
                          I8, 10, 16, 8, 8, 64)
    for k, v in change.items():
        setattr(c, k, v)
    return c


def _ref(c):
    return ctypes.byref(c) if c else None


def _append(cache, dtype=kv.BF16, T=2, k=SOME, slots=SOME, heads=8, q=SOME, out_q=SOME, out=(512, 64), positions=SOME, rope=None):
    st = (512, 64)
    return kv.load_kv().llmhip_kv_block_append(None, _ref(cache), dtype, T, k, *st, SOME, *st, slots, heads, q, *st, out_q, *out,
                                               positions, None if rope is None else ctypes.byref(rope), None)


def _read(cache, dtype=kv.BF16, T=2, slots=SOME, out_k=SOME, out_v=SOME, st=(512, 64)):
    return kv.load_kv().llmhip_kv_block_read(None, _ref(cache), dtype, T, slots, out_k, *st, out_v, *st, None)


def _attend(cache, dtype=kv.BF16, B=2, new=2, heads=8, q=SOME, out=(1024, 512, 64), table=SOME, P=4, ld=4, ws=SOME, window=0):
    return kv.load_kv().llmhip_kv_block_attend(None, _ref(cache), dtype, B, new, heads, q, 1024, 512, 64, table, P, ld, SOME, window,
                                               0.1, SOME, *out, None, ws, 1 << 40, None)


def _size(cache, new=1, heads=8):
    n = ctypes.c_size_t()
    return kv.load_kv().llmhip_kv_block_attend_workspace(None, _ref(cache), new, heads, ctypes.byref(n))


@pytest.mark.parametrize("change,code,text", [
    (dict(k_pool=None), BAD, "k_pool"), (dict(v_scale=None), BAD, "v_scale"), (dict(dtype=kv.BF16), BAD, "dtype"),
    (dict(dtype=5), BAD, "dtype"), (dict(pages=0), BAD, "pages"), (dict(heads=0), BAD, "heads"), (dict(page=0), BAD, "page"),
    (dict(block=0), BAD, "block"), (dict(block=5), BAD, "block"), (dict(block=32), BAD, "block"),
    (dict(page=512, block=512), UNSUPPORTED, "block"), (dict(pages=1 << 31), UNSUPPORTED, "pages"),
    (dict(head_dim=0), UNSUPPORTED, "head_dim"), (dict(head_dim=12), UNSUPPORTED, "head_dim"),
    (dict(head_dim=264), UNSUPPORTED, "head_dim"), (dict(v_pool=SOME + 4), UNSUPPORTED, "aligned"),
    (dict(k_stride=_three(8192, 512, 68)), UNSUPPORTED, "aligned"), (dict(k_scale=SOME + 2), BAD, "aligned"),
    (dict(v_stride=_three(-8192, 512, 64)), BAD, "negative"), (dict(k_scale_stride=_three(16, -8, 1)), BAD, "negative")])
def test_caches_that_are_refused(change, code, text):
    c = _cache(**change)
    for call in (_append, _read, _attend, _size):
        _refused(call(c), code, text)


def test_append_refusals():
    c = _cache()
    freqs = (ctypes.c_double * 32)()
    rope = lambda dims, style=0, f=ctypes.addressof(freqs): kv.LlmhipRope(f, dims, style)  # noqa: E731
    _refused(_append(None), BAD, "cache")
    _refused(_append(c, dtype=kv.E4M3), BAD, "dtype")
    _refused(_append(c, dtype=I8), BAD, "dtype")
    _refused(_append(c, out_q=None), BAD, "out_q")
    _refused(_append(c, q=None, out_q=None), BAD, "q_heads")
    _refused(_append(c, rope=rope(33)), BAD, "dims")
    _refused(_append(c, rope=rope(66)), BAD, "dims")
    _refused(_append(c, rope=rope(64, style=2)), BAD, "style")
    _refused(_append(c, rope=rope(64, f=None)), BAD, "freqs")
    _refused(_append(c, rope=rope(64), positions=None), BAD, "positions")
    _refused(_append(c, k=None), BAD, "required")
    _refused(_append(c, slots=None), BAD, "required")
    _refused(_append(c, out=(63, 64)), BAD, "out_q overlap")
    _refused(_append(c, out=(64, 64)), BAD, "out_q overlap")
    _refused(_append(c, T=(1 << 23) + 1), UNSUPPORTED, "T")
    _refused(_append(_cache(k_stride=_three(0, 512, 64))), BAD, "pool overlap")
    _refused(_append(_cache(v_stride=_three(4096, 512, 64))), BAD, "pool overlap")  # pages over one another
    _refused(_append(_cache(k_scale_stride=_three(8, 8, 1))), BAD, "scales overlap")
    _refused(_append(_cache(v_scale_stride=_three(16, 8, 0))), BAD, "scales overlap")
    _refused(_append(c, rope=rope(64)), BAD, "ctx")
    # Heads before tokens, and keys beside values, are no overlap.
    _refused(_append(_cache(k_stride=_three(8192, 64, 1024), v_stride=_three(16384, 1024, 128))), BAD, "ctx")
    assert _append(c, T=0) == 0


def test_read_refusals():
    c = _cache()
    _refused(_read(None), BAD, "cache")
    _refused(_read(c, dtype=kv.E4M3), BAD, "dtype")
    _refused(_read(c, out_k=None, out_v=None), BAD, "out_k")
    _refused(_read(c, slots=None), BAD, "slots")
    _refused(_read(c, st=(512, 63)), BAD, "overlap")
    _refused(_read(c, st=(256, 64)), BAD, "overlap")
    _refused(_read(c, st=(-512, 64)), BAD, "negative")
    _refused(_read(c, T=(1 << 23) + 1), UNSUPPORTED, "T")
    _refused(_read(c, out_k=None), BAD, "ctx")
    assert _read(c, T=0, out_k=None, out_v=None, slots=None) == 0


def test_attend_refusals():
    c = _cache()
    _refused(_attend(None), BAD, "cache")
    for dtype in (kv.F32, kv.E4M3, I8):
        _refused(_attend(c, dtype=dtype), BAD, "dtype")
    _refused(_attend(c, new=0), BAD, "new_tokens")
    _refused(_attend(c, new=17), UNSUPPORTED, "new_tokens")
    _refused(_size(c, new=0), BAD, "new_tokens")
    _refused(_size(c, new=17), UNSUPPORTED, "new_tokens")
    _refused(_size(c, heads=9), BAD, "multiple")
    _refused(_attend(c, heads=12), BAD, "multiple")
    _refused(_attend(c, heads=0), BAD, "multiple")
    _refused(_attend(c, B=65536), UNSUPPORTED, "B")
    _refused(_attend(c, ld=3), BAD, "table_ld")
    _refused(_attend(c, P=1 << 27, ld=1 << 27), UNSUPPORTED, "table_pages")
    _refused(_attend(c, q=None), BAD, "required")
    _refused(_attend(c, table=None), BAD, "table")
    _refused(_attend(c, ws=None), BAD, "workspace")
    _refused(_attend(c, ws=SOME + 4), BAD, "workspace")
    _refused(_attend(c, out=(1024, 256, 64)), BAD, "overlap")
    _refused(_attend(c, out=(512, 512, 64)), BAD, "overlap")
    _refused(_attend(c, out=(1024, 512, 32)), BAD, "overlap")
    _refused(_attend(c, out=(1024, -512, 64)), BAD, "negative")
    _refused(_attend(c), BAD, "ctx")
    assert _attend(c, B=0) == 0


def _state(dtype=torch.int8, shape=(4, 16, 2, 64), blocks=2):
    return [torch.zeros(shape).to(dtype) for _ in range(2)] + [torch.ones(shape[0], blocks, shape[2]) for _ in range(2)]


def _make(*state):
    return kv_blocks.BlockKVCache(_NoSampler, *state)


def test_mirror_refuses_wrong_pools_and_scales():
    k, v, ks, vs = _state()
    for bad in [(k, v[:2], ks, vs), (k[0], v[0], ks, vs), (k.float(), v.float(), ks, vs), (k, v.to(torch.float8_e4m3fn), ks, vs),
                (k.transpose(2, 3), v.transpose(2, 3), ks, vs), (k[..., :12], v[..., :12], ks, vs), (k[:0], v[:0], ks[:0], vs[:0]),
                (k, v, ks.double(), vs.double()), (k, v, ks[:3], vs[:3]), (k, v, ks, vs[:, :1]), (k, v, ks[..., :1], vs[..., :1]),
                (k, v, ks[:, :0], vs[:, :0]), (k, v, *_state(blocks=3)[2:]), (k, v, ks[0], vs[0]), (k, v, ks.half(), vs.half()),
                _state(shape=(1, 512, 1, 8), blocks=1)]:
        with pytest.raises(ValueError):
            _make(*bad)
    assert _make(k, v, ks, vs).block_size == 8


def test_mirror_refuses_wrong_calls():
    c = _make(*_state())
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    q4 = torch.zeros(3, 2, 4, 64, dtype=torch.bfloat16)
    one = torch.zeros((), dtype=torch.int32)
    slots, pos = torch.zeros(3, dtype=torch.int64), torch.zeros(3, dtype=torch.int32)
    table, lens, ws = torch.zeros(3, 2, dtype=torch.int32), pos, torch.zeros(256, dtype=torch.uint8)
    rope = kv.Rope(64)
    for bad in [lambda: c.append(x.double(), x.double(), slots), lambda: c.append(x.char(), x.char(), slots),
                lambda: c.append(x, x.float(), slots), lambda: c.append(x, x[:2], slots), lambda: c.append(x, q, slots),
                lambda: c.append(x, x, slots.int()), lambda: c.append(x, x, slots[:2]), lambda: c.append(x, x, slots, q=q),
                lambda: c.append(x, x, slots, q=q, out_q=q[:, :2]), lambda: c.append(x, x, slots, rope=rope),
                lambda: c.append(x, x, slots, positions=pos.long(), rope=rope),
                lambda: c.append(x, x, slots, positions=pos, rope=kv.Rope(66)), lambda: c.append(x, x, one.long()),
                lambda: c.append(x, x, slots, q=q, out_q=q[:, :1].expand(-1, 4, -1)),
                lambda: c.read(slots), lambda: c.read(slots.int(), x), lambda: c.read(slots, x[:2]), lambda: c.read(slots, x, x.float()),
                lambda: c.read(slots, x.double()), lambda: c.read(slots, x[:, :1].expand(-1, 2, -1)), lambda: c.read(slots, q),
                lambda: c.attend(q.float(), table, lens, q, ws), lambda: c.attend(q[:, :3], table, lens, q[:, :3], ws),
                lambda: c.attend(q, table.long(), lens, q, ws), lambda: c.attend(q, table[:2], lens, q, ws),
                lambda: c.attend(q, table, lens.long(), q, ws), lambda: c.attend(q, table, lens, q[:, :2], ws),
                lambda: c.attend(q, table, lens, q4, ws), lambda: c.attend(q4, table, lens, q4[:, :1].expand(-1, 2, -1, -1), ws),
                lambda: c.attend(q4[:, :0], table, lens, q4[:, :0], ws), lambda: c.attend(one.bfloat16(), table, lens, x, ws),
                lambda: c.attend(torch.zeros(3, 17, 4, 64).half(), table, lens, torch.zeros(3, 17, 4, 64).half(), ws),
                lambda: c.attend(q, table, lens, q, ws.int()), lambda: c.attend(q, table, lens, q, ws, window=-1),
                lambda: c.attend(q, table, lens, q, ws, out_lse=torch.zeros(3, 5)),
                lambda: c.attend(q4, table, lens, q4.clone(), ws, out_lse=torch.zeros(3, 4)),
                lambda: c.workspace(0), lambda: c.workspace(4, 0)]:
        with pytest.raises(ValueError):
            bad()
    k, v, ks, vs = _state()
    for state in [(k[:1].expand(4, -1, -1, -1), v, ks, vs), (k, v, ks, vs[:, :1].expand(-1, 2, -1))]:
        with pytest.raises(ValueError, match="overlap"):
            _make(*state).append(x, x, slots)


def test_mirror_refuses_the_hosts_memory_and_other_devices():
    c = _make(*_state())
    x, slots = torch.zeros(1, 2, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int64)
    table, lens, ws = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(256, dtype=torch.uint8)
    for bad in [lambda s: c.append(x, x, slots, stream=s), lambda s: c.read(slots, x.clone(), stream=s),
                lambda s: c.attend(x, table, lens, x.clone(), ws, stream=s)]:
        for stream in (None, object()):
            with pytest.raises(ValueError, match="not on a GPU"):
                bad(stream)
    state = [_gpu1(4, 16, 2, 64, dtype=torch.int8) for _ in range(2)] + [_gpu1(4, 2, 2, dtype=torch.float32) for _ in range(2)]
    with pytest.raises(ValueError, match="cuda:1.*cuda:0"):
        kv_blocks.BlockKVCache(_Sampler(0), *state)
    with pytest.raises(ValueError, match="k_scale is on cpu"):
        kv_blocks.BlockKVCache(_Sampler(1), *state[:2], *_state()[2:])
    c = kv_blocks.BlockKVCache(_Sampler(1), *state)
    on = lambda t: t.as_subclass(type(state[0]))  # noqa: E731
    with pytest.raises(ValueError, match="k is on cpu"):
        c.append(x, x, on(slots))
    with pytest.raises(ValueError, match="stream.*cuda:0"):
        c.read(on(slots), on(x.clone()), stream=_Stream("cuda:0"))
