"""Paged key-value cache of a decode loop, over the gfx950 C ABI (include/llmhip_kv.h).

  PagePool   hands out a pool's pages: block tables, slots and positions for
             the tokens that each request adds (llmhip_kv_plan)
  Rope       rotary positions
  KVCache    one layer's cache: append (llmhip_kv_append) stores new keys and
             values and rotates queries, attend (llmhip_kv_attend) is the
             attention of one new token for each request

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
EXPORTED_SYMBOLS = ("llmhip_kv_plan", "llmhip_kv_append", "llmhip_kv_attend_workspace", "llmhip_kv_attend")
STYLES = {"halves": 0, "neighbours": 1}

_vp, _sz, _u32, _i64 = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_uint32, ctypes.c_int64
_Stride = _i64 * 2


class LlmhipKvCache(ctypes.Structure):
    _fields_ = [("k_pool", _vp), ("v_pool", _vp), ("k_scale", _vp), ("v_scale", _vp), ("k_stride", _i64 * 3),
                ("v_stride", _i64 * 3), ("dtype", _u32), ("pages", _u32), ("page", _u32), ("heads", _u32),
                ("head_dim", _u32)]


class LlmhipRope(ctypes.Structure):
    _fields_ = [("freqs", _vp), ("dims", _u32), ("style", _u32)]


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
        lib.llmhip_kv_append.argtypes = [_vp, _vp, _u32, _sz, _vp, _vp, _vp, _vp, _vp, _sz, _vp, _vp, _vp, _vp, _vp,
                                         _vp, _vp]
        lib.llmhip_kv_attend_workspace.restype = ctypes.c_int
        lib.llmhip_kv_attend_workspace.argtypes = [_vp, _vp, _sz, ctypes.POINTER(_sz)]
        lib.llmhip_kv_attend.restype = ctypes.c_int
        lib.llmhip_kv_attend.argtypes = [_vp, _vp, _u32, _sz, _sz, _vp, _vp, _vp, _sz, _sz, _vp, _sz, ctypes.c_float,
                                         _vp, _vp, _vp, _vp, _sz, _vp]
        _lib = lib
    return _lib


def _check(lib, status: int) -> None:
    if status != 0:
        raise SamplerError(status, lib.llmhip_last_error().decode(errors="replace"))


def _vector(t, n: Optional[int], dtype, name: str, device):
    """A dense device vector of n values; its address."""
    if t.dtype != dtype or t.dim() != 1 or not t.is_contiguous() or (n is not None and t.shape[0] != n):
        raise ValueError(f"{name} must be a contiguous {dtype} vector" + ("" if n is None else f" of {n} values"))
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    return t.data_ptr()


def _table(t, n: int, device) -> int:
    """A block table of n requests; its row stride."""
    if t.dtype != torch.int32 or t.dim() != 2 or t.shape[0] != n or (t.stride(1) != 1 and t.shape[1] > 1 and n):
        raise ValueError(f"table must be an int32 [{n}, pages] tensor with dense rows")
    if t.device != device:
        raise ValueError(f"table is on {t.device}, not on {device}")
    return t.stride(0) if n > 1 else t.shape[1]


def _stream(stream, device, *tensors) -> int:
    if stream is None:
        return torch.cuda.current_stream(device).cuda_stream
    for t in tensors:  # their memory is not to be handed out again before this stream has used it
        if t is not None:
            t.record_stream(stream)
    return stream.cuda_stream


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
    them every page starts out free. One pool's plan serves the caches of all
    layers, whose page ids are the same."""

    def __init__(self, sampler: Sampler, pages: int, page_size: int, free_ring=None, free_state=None, device=None):
        if pages < 1 or page_size < 1:
            raise ValueError("pages and page_size must be at least 1")
        if (free_ring is None) != (free_state is None):
            raise ValueError("free_ring and free_state go together")
        if free_ring is None:
            device = torch.device("cuda:0") if device is None else torch.device(device)
            free_ring = torch.arange(pages, dtype=torch.int32, device=device)
            free_state = torch.tensor([0, pages], dtype=torch.int32, device=device)
        self.sampler, self.lib, self.pages, self.page_size = sampler, load_kv(), pages, page_size
        self.device = free_ring.device
        self._ring = _vector(free_ring, pages, torch.int32, "free_ring", self.device)
        self._state = _vector(free_state, 2, torch.int32, "free_state", self.device)
        self.free_ring, self.free_state = free_ring, free_state

    def plan(self, lens, table, out_lens, granted, start, slots, positions, new_tokens=None, release=None,
             out_free_state=None, stream=None) -> None:
        """llmhip_kv_plan. lens, out_lens, granted ([R] int32; out_lens may be
        lens), start ([R + 1] int32), table ([R, pages] int32, changed in
        place), slots ([T] int64) and positions ([T] int32), new_tokens and
        release ([R] int32, optional). Without out_free_state the pool's
        state moves on; with it ([2] int32) the pool's stays and the new one
        goes there."""
        dev, i32 = self.device, torch.int32
        R, T = lens.shape[0], slots.shape[0]
        ld = _table(table, R, dev)
        state = self.free_state if out_free_state is None else out_free_state
        status = self.lib.llmhip_kv_plan(
            self.sampler.ctx, self.pages, self.page_size, self._ring, self._state, R,
            _vector(lens, R, i32, "lens", dev),
            None if new_tokens is None else _vector(new_tokens, R, i32, "new_tokens", dev),
            None if release is None else _vector(release, R, i32, "release", dev), table.data_ptr(), table.shape[1],
            ld, _vector(out_lens, R, i32, "out_lens", dev),
            _vector(granted, R, i32, "granted", dev), _vector(start, R + 1, i32, "start", dev), T,
            _vector(slots, T, torch.int64, "slots", dev), _vector(positions, T, i32, "positions", dev),
            _vector(state, 2, i32, "out_free_state", dev),
            _stream(stream, dev, lens, new_tokens, release, table, out_lens, granted, start, slots, positions, state,
                    self.free_ring, self.free_state))
        _check(self.lib, status)


class KVCache:
    """One layer's cache: pools of keys and values [pages, page_size, heads,
    head_dim], dense in their last dimension, of float32, bfloat16, float16
    or float8_e4m3fn; with the last one k_scale and v_scale ([heads] float32)
    are what a stored value is multiplied with. head_dim is a multiple of 8
    up to 256."""

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

    def _rows(self, t, n: int, heads: Optional[int], dtype, name: str):
        """A [n, heads, head_dim] tensor with dense rows; its strides."""
        shape, stride = t.shape, t.stride()
        if (len(shape) != 3 or shape[0] != n or (heads is not None and shape[1] != heads) or shape[2] != self.head_dim
                or (stride[2] != 1 and n) or t.dtype != dtype):
            raise ValueError(f"{name} must be {dtype} [{n}, {'heads' if heads is None else heads}, {self.head_dim}] "
                             "with dense rows")
        if t.device != self.device:
            raise ValueError(f"{name} is on {t.device}, not on {self.device}")
        return _Stride(stride[0], stride[1])

    def append(self, k, v, slots, q=None, out_q=None, positions=None, rope: Optional[Rope] = None, stream=None) -> None:
        """llmhip_kv_append: k and v [T, heads, head_dim] into the slots ([T]
        int64; negative: nowhere), keys rotated by rope at positions ([T]
        int32); with q [T, q_heads, head_dim] its rotated rows go to out_q
        (which may be q). k, v and q may be views of one packed tensor; their
        type is the cache's, or any of the wider ones beside a float8 cache."""
        dt = k.dtype
        T = k.shape[0]
        if dt not in DTYPES or dt == torch.float8_e4m3fn or (dt != self.dtype and self.dtype != torch.float8_e4m3fn):
            raise ValueError(f"k is {dt}, which does not go into a {self.dtype} cache")
        if (q is None) != (out_q is None):
            raise ValueError("q and out_q go together")
        if rope is not None and (positions is None or rope.dims > self.head_dim):
            raise ValueError("rope needs positions, and dims of at most head_dim")
        q_heads = 0 if q is None else q.shape[1]
        status = self.lib.llmhip_kv_append(
            self.sampler.ctx, self._ref, DTYPES[dt], T, k.data_ptr(), self._rows(k, T, self.heads, dt, "k"),
            v.data_ptr(), self._rows(v, T, self.heads, dt, "v"), _vector(slots, T, torch.int64, "slots", self.device),
            q_heads, None if q is None else q.data_ptr(), None if q is None else self._rows(q, T, None, dt, "q"),
            None if q is None else out_q.data_ptr(),
            None if q is None else self._rows(out_q, T, q_heads, dt, "out_q"),
            None if positions is None else _vector(positions, T, torch.int32, "positions", self.device),
            None if rope is None else rope._ref, _stream(stream, self.device, k, v, slots, q, out_q, positions,
                                                         self.k_pool, self.v_pool, self.k_scale, self.v_scale))
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
        dt = q.dtype
        if dt not in DTYPES or dt == torch.float8_e4m3fn or (dt != self.dtype and (
                self.dtype != torch.float8_e4m3fn or dt == torch.float32)):
            raise ValueError(f"q is {dt}, which does not go with a {self.dtype} cache")
        B, heads, dev = q.shape[0], q.shape[1], self.device
        if not heads or heads % self.heads:
            raise ValueError(f"q must have a multiple of {self.heads} heads")
        ld = _table(table, B, dev)
        if window < 0:
            raise ValueError("window must not be negative")
        if out_lse is not None and (out_lse.dtype != torch.float32 or out_lse.shape != q.shape[:2]
                                    or not out_lse.is_contiguous() or out_lse.device != dev):
            raise ValueError(f"out_lse must be a contiguous float32 [{B}, {heads}] tensor on {dev}")
        status = self.lib.llmhip_kv_attend(
            self.sampler.ctx, self._ref, DTYPES[dt], B, heads, q.data_ptr(), self._rows(q, B, heads, dt, "q"),
            table.data_ptr(), table.shape[1], ld,
            _vector(lens, B, torch.int32, "lens", dev), window,
            1.0 / math.sqrt(self.head_dim) if scale is None else scale, out.data_ptr(),
            self._rows(out, B, heads, dt, "out"), None if out_lse is None else out_lse.data_ptr(),
            _vector(workspace, None, torch.uint8, "workspace", dev), workspace.numel(),
            _stream(stream, dev, q, table, lens, out, out_lse, workspace, self.k_pool, self.v_pool, self.k_scale,
                    self.v_scale))
        _check(self.lib, status)
