"""Paged key-value cache of a decode loop, over the gfx950 C ABI (include/llmhip_kv.h).

  PagePool   hands out a pool's pages: block tables, slots and positions for
             the tokens that each request adds (llmhip_kv_plan)
  Rope       rotary positions
  KVCache    one layer's cache: append (llmhip_kv_append) stores new keys and
             values and rotates queries, attend (llmhip_kv_attend) is the
             attention of one new token for each request

kv_blocks.BlockKVCache is such a cache in 8 bits whose scales follow from what
is written into it.

All of them work on torch tensors on the device, are enqueued on `stream`
(default: torch's current stream), allocate nothing and do not synchronize,
so a whole step can be captured into a graph. With a `stream` of the caller's
choice, ordering against the tensors' own streams is the caller's as well.
Wrong types, shapes, devices and layouts raise ValueError; what only the
device knows (lengths, page ids, slots) is checked by the kernels and shows
in Sampler.status() as KSTATUS_BAD_INDEX.

The reference keeps one ring cache for each generation
(crates/llm-core/src/model.rs:329-402); there is no CPU fallback here.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from .sampler import Sampler, SamplerError, load_library

KSTATUS_BAD_INDEX = 2
F32, BF16, F16, E4M3 = 0, 1, 2, 3
DTYPES = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16, torch.float8_e4m3fn: E4M3}
EXPORTED_SYMBOLS = ("llmhip_kv_plan", "llmhip_kv_append", "llmhip_kv_attend_workspace", "llmhip_kv_attend",
                    "llmhip_kv_block_append", "llmhip_kv_block_read", "llmhip_kv_block_attend_workspace",
                    "llmhip_kv_block_attend")
STYLES = {"halves": 0, "neighbours": 1}
_NO_ROWS = (None, 0, 0)

_vp, _sz, _u32, _i64 = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_uint32, ctypes.c_int64


class LlmhipKvCache(ctypes.Structure):
    _fields_ = [("k_pool", _vp), ("v_pool", _vp), ("k_scale", _vp), ("v_scale", _vp), ("k_stride", _i64 * 3),
                ("v_stride", _i64 * 3), ("dtype", _u32), ("pages", _u32), ("page", _u32), ("heads", _u32),
                ("head_dim", _u32)]


class LlmhipRope(ctypes.Structure):
    _fields_ = [("freqs", _vp), ("dims", _u32), ("style", _u32)]


class LlmhipKvBlocks(ctypes.Structure):
    _fields_ = [("k_pool", _vp), ("v_pool", _vp), ("k_scale", _vp), ("v_scale", _vp), ("k_stride", _i64 * 3),
                ("v_stride", _i64 * 3), ("k_scale_stride", _i64 * 3), ("v_scale_stride", _i64 * 3), ("dtype", _u32),
                ("pages", _u32), ("page", _u32), ("block", _u32), ("heads", _u32), ("head_dim", _u32)]


_lib: Optional[ctypes.CDLL] = None


def load_kv() -> ctypes.CDLL:
    """The library with the argument types of this module's entries."""
    global _lib
    if _lib is None:
        lib = load_library()
        lib.llmhip_kv_plan.restype = ctypes.c_int
        lib.llmhip_kv_plan.argtypes = [_vp, _sz, _sz, _vp, _vp, _sz, _vp, _vp, _vp, _vp, _sz, _sz, _vp, _vp, _vp, _sz,
                                       _vp, _vp, _vp, _vp]
        lib.llmhip_kv_append.restype = ctypes.c_int
        rows = [_vp, _i64, _i64]
        lib.llmhip_kv_append.argtypes = [_vp, _vp, _u32, _sz, *rows, *rows, _vp, _sz, *rows, *rows, _vp, _vp, _vp]
        lib.llmhip_kv_attend_workspace.restype = ctypes.c_int
        lib.llmhip_kv_attend_workspace.argtypes = [_vp, _vp, _sz, ctypes.POINTER(_sz)]
        lib.llmhip_kv_attend.restype = ctypes.c_int
        lib.llmhip_kv_attend.argtypes = [_vp, _vp, _u32, _sz, _sz, *rows, _vp, _sz, _sz, _vp, _sz, ctypes.c_float, *rows,
                                         _vp, _vp, _sz, _vp]
        lib.llmhip_kv_block_append.restype = ctypes.c_int
        lib.llmhip_kv_block_append.argtypes = lib.llmhip_kv_append.argtypes
        lib.llmhip_kv_block_read.restype = ctypes.c_int
        lib.llmhip_kv_block_read.argtypes = [_vp, _vp, _u32, _sz, _vp, *rows, *rows, _vp]
        lib.llmhip_kv_block_attend_workspace.restype = ctypes.c_int
        lib.llmhip_kv_block_attend_workspace.argtypes = [_vp, _vp, _sz, _sz, ctypes.POINTER(_sz)]
        lib.llmhip_kv_block_attend.restype = ctypes.c_int
        lib.llmhip_kv_block_attend.argtypes = [_vp, _vp, _u32, _sz, _sz, _sz, *rows, _i64, _vp, _sz, _sz, _vp, _sz,
                                               ctypes.c_float, *rows, _i64, _vp, _vp, _sz, _vp]
        _lib = lib
    return _lib


def _check(lib, status: int) -> None:
    if status != 0:
        raise SamplerError(status, lib.llmhip_last_error().decode(errors="replace"))


# A small call's time is the host's, so the checks below ask a tensor for each
# thing once and format nothing before they fail.
def _vector(t, n: int, dtype, name: str, device) -> int:
    """A dense device vector of n values; its address."""
    if t.dtype is not dtype or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} vector of {n} values")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    return t.data_ptr()


def _rows(t, shape, dtype, name: str, device):
    """A tensor of `shape` whose last dimension is dense; its address and its
    other strides."""
    a, b, c = t.stride() if t.dim() == 3 else (0, 0, 0)
    if t.shape != shape or t.dtype is not dtype or (c != 1 and shape[0]):
        raise ValueError(f"{name} must be {dtype} {list(shape)} with dense rows")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    return t.data_ptr(), a, b


def _out_rows(t, shape, dtype, name: str, device):
    """_rows of a tensor that is written."""
    r = _rows(t, shape, dtype, name, device)
    if (r[1] < shape[2] and shape[0] > 1) or (r[2] < shape[2] and shape[1] > 1):
        raise ValueError(f"rows of {name} overlap")
    return r


def _table(t, n: int, device):
    """A block table of n requests; its address, pages and row stride."""
    if t.dtype is not torch.int32 or t.dim() != 2 or t.shape[0] != n or (t.stride(1) != 1 and t.shape[1] > 1 and n):
        raise ValueError(f"table must be an int32 [{n}, pages] tensor with dense rows")
    if t.device != device:
        raise ValueError(f"table is on {t.device}, not on {device}")
    pages = t.shape[1]
    return t.data_ptr(), pages, t.stride(0) if n > 1 else pages


def _on(stream, device, tensors) -> int:
    """A stream of the caller's choice; the tensors' memory is not handed out
    again before it has used them."""
    if device.type != "cuda":
        raise ValueError(f"the tensors are on {device}, not on a GPU")
    if getattr(stream, "device", device) != device:
        raise ValueError(f"the stream is on {stream.device}, the tensors on {device}")
    for t in tensors:
        if t is not None:
            t.record_stream(stream)
    return stream.cuda_stream


# torch.cuda.current_stream builds a Stream object for each call (about a
# microsecond); this is the query beneath it.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _current(device) -> int:
    try:
        return _raw_stream(device.index)
    except (TypeError, RuntimeError):  # no such query, or the host's device, which has no index
        if device.type != "cuda":
            raise ValueError(f"the tensors are on {device}, not on a GPU") from None
        return torch.cuda.current_stream(device).cuda_stream


def _same_gpu(sampler: Sampler, device) -> None:
    """Kernels and flags are the sampler's device's. (The host's tensors are
    refused where a call would use them.)"""
    index = getattr(sampler, "device", device.index)
    if device.type == "cuda" and device.index != index:
        raise ValueError(f"the tensors are on {device}, the sampler on cuda:{index}")


class Rope:
    """Rotary positions of the first `dims` values of each head row: pair i
    turns by position * theta ** (-2 i / dims), or by position * freqs[i]
    where freqs (dims / 2 numbers) are given. style "halves" pairs values i
    and i + dims / 2, "neighbours" values 2 i and 2 i + 1."""

    def __init__(self, dims: int, theta: float = 10000.0, style: str = "halves", freqs=None):
        if dims < 2 or dims % 2:
            raise ValueError("dims must be even and at least 2")
        if style not in STYLES:
            raise ValueError(f"style must be one of {sorted(STYLES)}")
        if freqs is None:
            if not theta > 0:
                raise ValueError("theta must be positive")
            freqs = [theta ** (-2.0 * i / dims) for i in range(dims // 2)]
        freqs = [float(f) for f in freqs]
        if len(freqs) != dims // 2 or not all(math.isfinite(f) for f in freqs):
            raise ValueError("freqs must be dims / 2 finite numbers")
        self.dims, self.style, self.freqs = dims, style, tuple(freqs)
        self._array = (ctypes.c_double * len(freqs))(*freqs)
        self._c = LlmhipRope(ctypes.addressof(self._array), dims, STYLES[style])
        self._ref = ctypes.addressof(self._c)


class PagePool:
    """The free pages of a pool of `pages` pages of `page_size` tokens.
    free_ring ([pages] int32) and free_state ([2] int32: the first free id's
    place in the ring, and how many are free) live on the device; without
    them every page starts out free, on the sampler's device. One pool's plan
    serves the caches of all layers, whose page ids are the same."""

    def __init__(self, sampler: Sampler, pages: int, page_size: int, free_ring=None, free_state=None, device=None):
        if pages < 1 or page_size < 1:
            raise ValueError("pages and page_size must be at least 1")
        if (free_ring is None) != (free_state is None):
            raise ValueError("free_ring and free_state go together")
        if free_ring is None:
            device = torch.device("cuda", sampler.device) if device is None else torch.device(device)
            free_ring = torch.arange(pages, dtype=torch.int32, device=device)
            free_state = torch.tensor([0, pages], dtype=torch.int32, device=device)
        self.sampler, self.lib, self.pages, self.page_size = sampler, load_kv(), pages, page_size
        self.device = free_ring.device
        _same_gpu(sampler, self.device)
        self._ring = _vector(free_ring, pages, torch.int32, "free_ring", self.device)
        self._state = _vector(free_state, 2, torch.int32, "free_state", self.device)
        self.free_ring, self.free_state = free_ring, free_state
        self._plan = self.lib.llmhip_kv_plan

    def plan(self, lens, table, out_lens, granted, start, slots, positions, new_tokens=None, release=None,
             out_free_state=None, stream=None) -> None:
        """llmhip_kv_plan. lens, out_lens, granted ([R] int32; out_lens may be
        lens), start ([R + 1] int32), table ([R, pages] int32, changed in
        place), slots ([T] int64) and positions ([T] int32), new_tokens and
        release ([R] int32, optional). Without out_free_state the pool's
        state moves on; with it ([2] int32) the pool's stays and the new one
        goes there."""
        dev, i32 = self.device, torch.int32
        R, T = lens.numel(), slots.numel()
        state = self.free_state if out_free_state is None else out_free_state
        status = self._plan(
            self.sampler.ctx, self.pages, self.page_size, self._ring, self._state, R, _vector(lens, R, i32, "lens", dev),
            None if new_tokens is None else _vector(new_tokens, R, i32, "new_tokens", dev),
            None if release is None else _vector(release, R, i32, "release", dev), *_table(table, R, dev),
            _vector(out_lens, R, i32, "out_lens", dev), _vector(granted, R, i32, "granted", dev),
            _vector(start, R + 1, i32, "start", dev), T, _vector(slots, T, torch.int64, "slots", dev),
            _vector(positions, T, i32, "positions", dev),
            self._state if out_free_state is None else _vector(out_free_state, 2, i32, "out_free_state", dev),
            _current(dev) if stream is None else _on(stream, dev, (lens, new_tokens, release, table, out_lens, granted,
                                                                   start, slots, positions, state, self.free_ring, self.free_state)))
        if status:
            _check(self.lib, status)


class KVCache:
    """One layer's cache: pools of keys and values [pages, page_size, heads,
    head_dim], dense in their last dimension, of float32, bfloat16, float16
    or float8_e4m3fn; with the last one k_scale and v_scale ([heads] float32)
    are what a stored value is multiplied with. head_dim is a multiple of 8
    up to 256. Pools whose rows overlap (expanded ones) can be attended over,
    not appended to."""

    def __init__(self, sampler: Sampler, k_pool, v_pool, k_scale=None, v_scale=None):
        if k_pool.dim() != 4 or k_pool.shape != v_pool.shape:
            raise ValueError("k_pool and v_pool must be [pages, page_size, heads, head_dim], of one shape")
        if k_pool.dtype not in DTYPES or k_pool.dtype != v_pool.dtype:
            raise ValueError("the pools must be float32, bfloat16, float16 or float8_e4m3fn, both the same")
        if k_pool.device != v_pool.device:
            raise ValueError("k_pool and v_pool are on different devices")
        if k_pool.stride(3) != 1 or v_pool.stride(3) != 1:
            raise ValueError("the pools' rows must be dense")
        pages, page, heads, dim = k_pool.shape
        if not (pages and page and heads):
            raise ValueError("the pools must not be empty")
        if dim % 8 or not 8 <= dim <= 256:
            raise ValueError("head_dim must be a multiple of 8 up to 256")
        self.dtype, self.device = k_pool.dtype, k_pool.device
        _same_gpu(sampler, self.device)
        if (self.dtype == torch.float8_e4m3fn) != (k_scale is not None) or (k_scale is None) != (v_scale is None):
            raise ValueError("k_scale and v_scale go with float8_e4m3fn pools, and only with those")
        self.sampler, self.lib = sampler, load_kv()
        self.k_pool, self.v_pool, self.k_scale, self.v_scale = k_pool, v_pool, k_scale, v_scale
        self.pages, self.page_size, self.heads, self.head_dim = pages, page, heads, dim
        scales = [None if s is None else _vector(s, heads, torch.float32, n, self.device)
                  for s, n in ((k_scale, "k_scale"), (v_scale, "v_scale"))]
        self._c = LlmhipKvCache(k_pool.data_ptr(), v_pool.data_ptr(), *scales, (_i64 * 3)(*k_pool.stride()[:3]),
                                (_i64 * 3)(*v_pool.stride()[:3]), DTYPES[self.dtype], pages, page, heads, dim)
        self._ref = ctypes.addressof(self._c)
        # Rows that lie over one another can be read, not appended to.
        self._apart = all(s >= dim or n < 2 for p in (k_pool, v_pool) for s, n in zip(p.stride()[:3], p.shape))
        self._scale = 1.0 / math.sqrt(dim)
        self._append, self._attend = self.lib.llmhip_kv_append, self.lib.llmhip_kv_attend
        # What may come beside this cache, as the C entries name it.
        self._codes = {t: c for t, c in DTYPES.items()
                       if c != E4M3 and (t is self.dtype or self.dtype is torch.float8_e4m3fn)}

    def append(self, k, v, slots, q=None, out_q=None, positions=None, rope: Optional[Rope] = None, stream=None) -> None:
        """llmhip_kv_append: k and v [T, heads, head_dim] into the slots ([T]
        int64; negative: nowhere), keys rotated by rope at positions ([T]
        int32); with q [T, q_heads, head_dim] its rotated rows go to out_q
        (which may be q). k, v and q may be views of one packed tensor; their
        type is the cache's, or any of the wider ones beside a float8 cache."""
        dt, dev = k.dtype, self.device
        code = self._codes.get(dt)
        if code is None:
            raise ValueError(f"k is {dt}, which does not go into a {self.dtype} cache")
        if not self._apart:
            raise ValueError("rows of a pool overlap")
        if (q is None) != (out_q is None):
            raise ValueError("q and out_q go together")
        T = slots.numel()
        shape = (T, self.heads, self.head_dim)
        if rope is None:
            turn = None
        elif positions is None or rope.dims > self.head_dim:
            raise ValueError("rope needs positions, and dims of at most head_dim")
        else:
            turn = rope._ref
        if q is None:
            heads, q_rows, out_rows = 0, _NO_ROWS, _NO_ROWS
        else:
            if q.dim() != 3:
                raise ValueError("q must be [T, q_heads, head_dim]")
            heads = q.shape[1]
            q_shape = (T, heads, self.head_dim)
            q_rows, out_rows = _rows(q, q_shape, dt, "q", dev), _out_rows(out_q, q_shape, dt, "out_q", dev)
        status = self._append(
            self.sampler.ctx, self._ref, code, T, *_rows(k, shape, dt, "k", dev), *_rows(v, shape, dt, "v", dev),
            _vector(slots, T, torch.int64, "slots", dev), heads, *q_rows, *out_rows,
            None if positions is None else _vector(positions, T, torch.int32, "positions", dev), turn,
            _current(dev) if stream is None else _on(stream, dev, (k, v, slots, q, out_q, positions, self.k_pool,
                                                                   self.v_pool, self.k_scale, self.v_scale)))
        if status:
            _check(self.lib, status)

    def workspace(self, q_heads: int):
        """A workspace for attend with q_heads query heads, whatever the
        batch. Calls that may overlap need one each."""
        n = _sz()
        _check(self.lib, self.lib.llmhip_kv_attend_workspace(self.sampler.ctx, self._ref, q_heads, ctypes.byref(n)))
        return torch.empty(n.value, dtype=torch.uint8, device=self.device)

    def attend(self, q, table, lens, out, workspace, window: int = 0, scale: Optional[float] = None, out_lse=None,
               stream=None) -> None:
        """llmhip_kv_attend: q [B, q_heads, head_dim] over each request's last
        min(lens[b], window) tokens (window 0: all), whose pages are table
        ([B, pages] int32); lens ([B] int32) counts the newest token. out is
        like q, out_lse [B, q_heads] float32; scale defaults to
        head_dim ** -0.5. q_heads is a multiple of the cache's heads, and q
        of the cache's type (bfloat16 or float16 beside a float8 cache)."""
        dt, dev = q.dtype, self.device
        code = self._codes.get(dt)
        if code is None or (dt is torch.float32 and self.dtype is not dt):
            raise ValueError(f"q is {dt}, which does not go with a {self.dtype} cache")
        if q.dim() != 3:
            raise ValueError("q must be [B, q_heads, head_dim]")
        B, heads = q.shape[0], q.shape[1]
        if not heads or heads % self.heads:
            raise ValueError(f"q must have a multiple of {self.heads} heads")
        if window < 0:
            raise ValueError("window must not be negative")
        if out_lse is None:
            lse = None
        elif out_lse.dtype is not torch.float32 or out_lse.shape != (B, heads) or not out_lse.is_contiguous() \
                or out_lse.device != dev:
            raise ValueError(f"out_lse must be a contiguous float32 [{B}, {heads}] tensor on {dev}")
        else:
            lse = out_lse.data_ptr()
        shape = (B, heads, self.head_dim)
        size = workspace.numel()
        status = self._attend(
            self.sampler.ctx, self._ref, code, B, heads, *_rows(q, shape, dt, "q", dev), *_table(table, B, dev),
            _vector(lens, B, torch.int32, "lens", dev), window, self._scale if scale is None else scale,
            *_out_rows(out, shape, dt, "out", dev), lse, _vector(workspace, size, torch.uint8, "workspace", dev), size,
            _current(dev) if stream is None else _on(stream, dev, (q, table, lens, out, out_lse, workspace, self.k_pool,
                                                                   self.v_pool, self.k_scale, self.v_scale)))
        if status:
            _check(self.lib, status)
