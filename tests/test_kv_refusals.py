"""What the key-value cache's entries refuse, without a GPU: the C entries
check their arguments before the context, the Python mirror before the call."""
import ctypes
import re
import subprocess
from pathlib import Path

import pytest
import torch

from scriptonait_amd import kv
from scriptonait_amd import sampler as smp

ROOT = Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "llmhip_kv.h"
BAD, UNSUPPORTED = -1, -5
SOME = 4096  # an address that no refused call follows


def test_header_library_and_mirror_name_the_same_entries():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(llmhip_kv_\w+)\s*\(", text)))
    assert declared == sorted(kv.EXPORTED_SYMBOLS)
    lib = kv.load_kv()
    out = subprocess.run(["nm", "-D", "--defined-only", str(smp.LIB_PATH)], check=True, capture_output=True, text=True).stdout
    exported = {line.split()[-1] for line in out.splitlines() if line.strip()}
    notes = (ROOT / "INTEGRATION.md").read_text()
    for name in declared:
        assert name in exported and hasattr(lib, name) and name in notes
    assert re.search(rf"#define LLMHIP_KSTATUS_BAD_INDEX {kv.KSTATUS_BAD_INDEX}u", HEADER.read_text())


def test_header_is_plain_c(tmp_path):
    src = tmp_path / "a.c"
    src.write_text('#include "llmhip_kv.h"\n#include <stdio.h>\nint main(void) { printf("%zu %zu\\n", '
                   "sizeof(llmhip_kv_cache), sizeof(llmhip_rope)); return LLMHIP_F32; }\n")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", f"-I{HEADER.parent}", str(src), "-o", str(tmp_path / "a")], check=True)
    out = subprocess.run([str(tmp_path / "a")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in out] == [ctypes.sizeof(kv.LlmhipKvCache), ctypes.sizeof(kv.LlmhipRope)]


def _cache(**change):
    c = kv.LlmhipKvCache(SOME, SOME, None, None, (ctypes.c_int64 * 3)(8192, 512, 64), (ctypes.c_int64 * 3)(8192, 512, 64),
                         kv.BF16, 10, 16, 8, 64)
    for k, v in change.items():
        setattr(c, k, v)
    return c


def _refused(status, code, text):
    assert status == code
    assert text in kv.load_kv().llmhip_last_error().decode()


CACHES = [
    (dict(k_pool=None), BAD, "k_pool"),
    (dict(dtype=9), BAD, "dtype"),
    (dict(k_scale=SOME), BAD, "k_scale"),
    (dict(dtype=kv.E4M3), BAD, "k_scale"),
    (dict(pages=0), BAD, "pages"),
    (dict(page=0), BAD, "pages"),
    (dict(heads=0), BAD, "heads"),
    (dict(head_dim=0), UNSUPPORTED, "head_dim"),
    (dict(head_dim=12), UNSUPPORTED, "head_dim"),
    (dict(head_dim=264), UNSUPPORTED, "head_dim"),
    (dict(v_pool=SOME + 8), UNSUPPORTED, "aligned"),
    (dict(k_stride=(ctypes.c_int64 * 3)(8192, 512, 68)), UNSUPPORTED, "aligned"),
    (dict(k_stride=(ctypes.c_int64 * 3)(-8192, 512, 64)), BAD, "negative"),
]


def _attend(cache, dtype=kv.BF16, B=2, heads=8, q=SOME, table=SOME, P=4, ld=4, ws=SOME, window=0, ctx=None):
    st = (512, 64)
    return kv.load_kv().llmhip_kv_attend(ctx, ctypes.byref(cache) if cache else None, dtype, B, heads, q, *st, table, P, ld, SOME,
                                         window, 0.1, SOME, *st, None, ws, 1 << 40, None)


def _append(cache, dtype=kv.BF16, T=2, k=SOME, slots=SOME, heads=8, q=SOME, out_q=SOME, positions=SOME, rope=None, ctx=None):
    st = (512, 64)
    return kv.load_kv().llmhip_kv_append(ctx, ctypes.byref(cache) if cache else None, dtype, T, k, *st, SOME, *st, slots, heads,
                                         q, *st, out_q, *st, positions, None if rope is None else ctypes.byref(rope), None)


@pytest.mark.parametrize("change,code,text", CACHES)
def test_caches_that_are_refused(change, code, text):
    c = _cache(**change)
    _refused(_attend(c), code, text)
    _refused(_append(c), code, text)
    n = ctypes.c_size_t()
    _refused(kv.load_kv().llmhip_kv_attend_workspace(None, ctypes.byref(c), 8, ctypes.byref(n)), code, text)


def test_attend_refusals():
    c = _cache()
    e4m3 = _cache(dtype=kv.E4M3, k_scale=SOME, v_scale=SOME)
    _refused(_attend(None), BAD, "cache")
    _refused(_attend(c, dtype=kv.F16), BAD, "dtype")
    _refused(_attend(c, dtype=kv.E4M3), BAD, "dtype")
    _refused(_attend(e4m3, dtype=kv.F32), BAD, "dtype")
    _refused(_attend(c, heads=12), BAD, "multiple")
    _refused(_attend(c, heads=0), BAD, "multiple")
    _refused(_attend(c, B=65536), UNSUPPORTED, "B")
    _refused(_attend(c, ld=3), BAD, "table_ld")
    _refused(_attend(c, P=1 << 27, ld=1 << 27), UNSUPPORTED, "table_pages")
    _refused(_attend(c, q=None), BAD, "required")
    _refused(_attend(c, table=None), BAD, "table")
    _refused(_attend(c, ws=None), BAD, "workspace")
    _refused(_attend(c, ws=SOME + 4), BAD, "workspace")
    _refused(_attend(c), BAD, "ctx")
    assert _attend(c, B=0) == 0


def test_append_refusals():
    c = _cache()
    freqs = (ctypes.c_double * 32)()
    rope = lambda dims, style=0, f=ctypes.addressof(freqs): kv.LlmhipRope(f, dims, style)  # noqa: E731
    _refused(_append(None), BAD, "cache")
    _refused(_append(c, dtype=kv.F32), BAD, "dtype")
    _refused(_append(c, dtype=7), BAD, "dtype")
    _refused(_append(c, out_q=None), BAD, "out_q")
    _refused(_append(c, q=None, out_q=None), BAD, "q_heads")
    _refused(_append(c, rope=rope(33)), BAD, "dims")
    _refused(_append(c, rope=rope(66)), BAD, "dims")
    _refused(_append(c, rope=rope(64, style=2)), BAD, "style")
    _refused(_append(c, rope=rope(64, f=None)), BAD, "freqs")
    _refused(_append(c, rope=rope(64), positions=None), BAD, "positions")
    _refused(_append(c, k=None), BAD, "required")
    _refused(_append(c, slots=None), BAD, "required")
    _refused(_append(c, T=1 << 31), UNSUPPORTED, "T")
    _refused(_append(c, rope=rope(64)), BAD, "ctx")
    assert _append(c, T=0) == 0


@pytest.mark.parametrize("change,code,text", [
    (dict(pages=0), BAD, "pages"), (dict(page=0), BAD, "pages"), (dict(pages=1 << 31), UNSUPPORTED, "pages"),
    (dict(ring=None), BAD, "ring"), (dict(state=None), BAD, "free_state"), (dict(lens=None), BAD, "lens"),
    (dict(table=None), BAD, "table"), (dict(start=None), BAD, "start"), (dict(slots=None), BAD, "slots"),
    (dict(R=1 << 31), UNSUPPORTED, "R"), (dict(ld=3), BAD, "table_ld"), (dict(P=1 << 27, ld=1 << 27), UNSUPPORTED, "table_pages"),
    (dict(), BAD, "ctx")])
def test_plan_refusals(change, code, text):
    a = dict(pages=10, page=16, ring=SOME, state=SOME, R=2, lens=SOME, table=SOME, P=4, ld=4, start=SOME, T=3, slots=SOME)
    a.update(change)
    _refused(kv.load_kv().llmhip_kv_plan(None, a["pages"], a["page"], a["ring"], a["state"], a["R"], a["lens"], None, None,
                                         a["table"], a["P"], a["ld"], SOME, SOME, a["start"], a["T"], a["slots"], SOME, SOME,
                                         None), code, text)


class _NoSampler:
    ctx = None


def _pools(dtype=torch.bfloat16, shape=(4, 16, 2, 64)):
    return [torch.zeros(shape).to(dtype) for _ in range(2)]


def test_mirror_refuses_wrong_pools():
    k, v = _pools()
    for bad in [lambda: kv.KVCache(_NoSampler, k, v[:2]), lambda: kv.KVCache(_NoSampler, k[0], v[0]),
                lambda: kv.KVCache(_NoSampler, k.double(), v.double()), lambda: kv.KVCache(_NoSampler, k, v.half()),
                lambda: kv.KVCache(_NoSampler, k.transpose(2, 3), v.transpose(2, 3)),
                lambda: kv.KVCache(_NoSampler, k[..., :12], v[..., :12]), lambda: kv.KVCache(_NoSampler, k[:0], v[:0]),
                lambda: kv.KVCache(_NoSampler, k, v, torch.ones(2), torch.ones(2)),
                lambda: kv.KVCache(_NoSampler, *_pools(torch.float8_e4m3fn)),
                lambda: kv.KVCache(_NoSampler, *_pools(torch.float8_e4m3fn), torch.ones(2), None),
                lambda: kv.KVCache(_NoSampler, *_pools(torch.float8_e4m3fn), torch.ones(3), torch.ones(3))]:
        with pytest.raises(ValueError):
            bad()


def test_mirror_refuses_wrong_calls():
    c = kv.KVCache(_NoSampler, *_pools())
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    slots, pos = torch.zeros(3, dtype=torch.int64), torch.zeros(3, dtype=torch.int32)
    table, lens, ws = torch.zeros(3, 2, dtype=torch.int32), pos, torch.zeros(256, dtype=torch.uint8)
    rope = kv.Rope(64)
    for bad in [lambda: c.append(x.float(), x.float(), slots), lambda: c.append(x, x.float(), slots),
                lambda: c.append(x, x[:2], slots), lambda: c.append(x, q, slots), lambda: c.append(x, x, slots.int()),
                lambda: c.append(x, x, slots[:2]), lambda: c.append(x, x, slots, q=q),
                lambda: c.append(x, x, slots, q=q, out_q=q[:, :2]), lambda: c.append(x, x, slots, rope=rope),
                lambda: c.append(x, x, slots, positions=pos.long(), rope=rope),
                lambda: c.append(x, x, slots, positions=pos, rope=kv.Rope(66)),
                lambda: c.append(x[..., ::2].repeat(1, 1, 2)[..., :64].transpose(1, 2).contiguous().transpose(1, 2), x, slots),
                lambda: c.attend(q.float(), table, lens, q, ws), lambda: c.attend(q[:, :3], table, lens, q[:, :3], ws),
                lambda: c.attend(q, table.long(), lens, q, ws), lambda: c.attend(q, table[:2], lens, q, ws),
                lambda: c.attend(q, table, lens.long(), q, ws), lambda: c.attend(q, table, lens, q[:, :2], ws),
                lambda: c.attend(q, table, lens, q, ws.int()), lambda: c.attend(q, table, lens, q, ws, window=-1),
                lambda: c.attend(q, table, lens, q, ws, out_lse=torch.zeros(3, 5))]:
        with pytest.raises(ValueError):
            bad()


def test_mirror_refuses_wrong_pages_and_ropes():
    ring, state = torch.arange(8, dtype=torch.int32), torch.tensor([0, 8], dtype=torch.int32)
    for bad in [lambda: kv.PagePool(_NoSampler, 0, 16), lambda: kv.PagePool(_NoSampler, 8, 0),
                lambda: kv.PagePool(_NoSampler, 8, 16, free_ring=ring), lambda: kv.PagePool(_NoSampler, 9, 16, ring, state),
                lambda: kv.PagePool(_NoSampler, 8, 16, ring.long(), state), lambda: kv.PagePool(_NoSampler, 8, 16, ring, ring),
                lambda: kv.Rope(0), lambda: kv.Rope(7), lambda: kv.Rope(8, style="pairs"), lambda: kv.Rope(8, theta=0.0),
                lambda: kv.Rope(8, freqs=[1.0] * 3), lambda: kv.Rope(8, freqs=[1.0, 1.0, 1.0, float("nan")])]:
        with pytest.raises(ValueError):
            bad()
    pool = kv.PagePool(_NoSampler, 8, 16, ring, state)
    i = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    args = dict(lens=i(2), table=torch.zeros(2, 3, dtype=torch.int32), out_lens=i(2), granted=i(2), start=i(3),
                slots=torch.zeros(5, dtype=torch.int64), positions=i(5))
    for name, wrong in [("lens", i(2).long()), ("lens", i(3)), ("table", i(2)), ("table", torch.zeros(3, 3, dtype=torch.int32)),
                        ("out_lens", i(1)), ("granted", i(4)[::2]), ("start", i(2)), ("slots", i(5)), ("positions", i(4)),
                        ("new_tokens", i(1)), ("release", i(2).bool()), ("out_free_state", i(1))]:
        with pytest.raises(ValueError):
            pool.plan(**{**args, name: wrong})


def test_mirror_refuses_numbers_for_vectors_and_host_memory():
    """Tensors of no dimension and tensors of the host reach no kernel."""
    one = torch.zeros((), dtype=torch.int32)
    c = kv.KVCache(_NoSampler, *_pools())
    x, slots = torch.zeros(1, 2, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int64)
    table, lens, ws = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(256, dtype=torch.uint8)
    ring, state = torch.arange(8, dtype=torch.int32), torch.tensor([0, 8], dtype=torch.int32)
    pool = kv.PagePool(_NoSampler, 8, 16, ring, state)
    rest = (lens.clone(), lens.clone(), torch.zeros(2, dtype=torch.int32))
    for bad in [lambda: c.append(one.bfloat16(), x, slots), lambda: c.append(x, x, one.long()),
                lambda: c.append(x, x, slots, q=one.bfloat16(), out_q=one.bfloat16()),
                lambda: c.attend(one.bfloat16(), table, lens, x, ws), lambda: c.attend(x, one, lens, x, ws),
                lambda: c.attend(x, table, one, x, ws), lambda: pool.plan(one, table, *rest, slots, lens),
                lambda: pool.plan(lens, table, *rest, one.long(), lens)]:
        with pytest.raises(ValueError):
            bad()
    for bad in [lambda: c.append(x, x, slots), lambda: c.attend(x, table, lens, x.clone(), ws),
                lambda: pool.plan(lens, table, *rest, slots, lens.clone()),
                lambda: c.append(x, x, slots, stream=object()), lambda: c.attend(x, table, lens, x.clone(), ws, stream=object()),
                lambda: pool.plan(lens, table, *rest, slots, lens.clone(), stream=object())]:
        with pytest.raises(ValueError, match="not on a GPU"):
            bad()
