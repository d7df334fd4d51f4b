"""Paged key-value cache in 8 bits with a scale for each block of tokens and
head, over the gfx950 C ABI (include/llmhip_kv.h).

  BlockKVCache  one layer's cache: append (llmhip_kv_block_append) quantises
                new keys and values as it writes them and rotates queries,
                read (llmhip_kv_block_read) gives tokens back, attend
                (llmhip_kv_block_attend) is the attention of the newest
                token, or the newest few, of each request

Its pages are handed out by kv.PagePool and its rotary positions are kv.Rope's,
as those of kv.KVCache are; all that is said there of streams, captured
graphs, errors and status holds here too.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from .kv import _NO_ROWS, _check, _current, _on, _out_rows, _rows, _same_gpu, _table, _vector, DTYPES, LlmhipKvBlocks, Rope, load_kv
from .sampler import Sampler

CODES = {torch.int8: 4, torch.float8_e4m3fn: 3}
_ROWS = {t: c for t, c in DTYPES.items() if t is not torch.float8_e4m3fn}
_i64 = ctypes.c_int64
MAX_BLOCK, MAX_NEW_TOKENS = 256, 16
_ERR_ARGUMENT = -1  # LLMHIP_ERR_INVALID_ARGUMENT


def _apart(t, inner: int, dims: int) -> bool:
    """Whether no two rows of `inner` values lie over one another: each of the
    first dims directions steps past all that the smaller steps span."""
    span = inner
    for step, n in sorted(zip(t.stride()[:dims], t.shape)):
        if n > 1:
            if step < span:
                return False
            span += step * (n - 1)
    return True


def _queries(t, shape, dtype, name: str, device):
    """A tensor of `shape` ([B, heads, dim] or [B, tokens, heads, dim]) whose
    last dimension is dense; its address and its other strides."""
    if t.shape != shape or t.dtype is not dtype or (t.stride(-1) != 1 and shape[0]):
        raise ValueError(f"{name} must be {dtype} {list(shape)} with dense rows")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    s = t.stride()
    return (t.data_ptr(), s[0], 0, s[1]) if len(shape) == 3 else (t.data_ptr(), s[0], s[1], s[2])


class BlockKVCache:
    """One layer's cache: pools of keys and values [pages, page_size, heads,
    head_dim] of int8 or float8_e4m3fn, dense in their last dimension, and
    their scales, float32 [pages, blocks, heads], where blocks divides
    page_size: block b of a page is its tokens b * block_size and on, with
    block_size (page_size // blocks) at most 256. A stored value is its code
    times its block's scale. append writes the scales; they need no values
    before. head_dim is a multiple of 8 up to 256. Pools and scales whose rows
    overlap (expanded ones) can be read and attended over, not appended to."""

    def __init__(self, sampler: Sampler, k_pool, v_pool, k_scale, v_scale):
        if k_pool.dim() != 4 or k_pool.shape != v_pool.shape:
            raise ValueError("k_pool and v_pool must be [pages, page_size, heads, head_dim], of one shape")
        if k_pool.dtype not in CODES or k_pool.dtype != v_pool.dtype:
            raise ValueError("the pools must be int8 or float8_e4m3fn, both the same")
        if k_pool.stride(3) != 1 or v_pool.stride(3) != 1:
            raise ValueError("the pools' rows must be dense")
        pages, page, heads, dim = k_pool.shape
        if not (pages and page and heads):
            raise ValueError("the pools must not be empty")
        if dim % 8 or not 8 <= dim <= 256:
            raise ValueError("head_dim must be a multiple of 8 up to 256")
        if k_scale.dim() != 3 or k_scale.shape != v_scale.shape or k_scale.shape[0] != pages or k_scale.shape[2] != heads \
                or k_scale.dtype is not torch.float32 or v_scale.dtype is not torch.float32:
            raise ValueError(f"k_scale and v_scale must be float32 [{pages}, blocks, {heads}], of one shape")
        blocks = k_scale.shape[1]
        if not blocks or page % blocks or page // blocks > MAX_BLOCK:
            raise ValueError(f"a page of {page} tokens is no whole number of {blocks} blocks of at most {MAX_BLOCK} tokens")
        self.dtype, self.device = k_pool.dtype, k_pool.device
        for t, name in ((v_pool, "v_pool"), (k_scale, "k_scale"), (v_scale, "v_scale")):
            if t.device != self.device:
                raise ValueError(f"{name} is on {t.device}, not on {self.device}")
        _same_gpu(sampler, self.device)
        self.sampler, self.lib = sampler, load_kv()
        self.k_pool, self.v_pool, self.k_scale, self.v_scale = k_pool, v_pool, k_scale, v_scale
        self.pages, self.page_size, self.heads, self.head_dim, self.block_size = pages, page, heads, dim, page // blocks
        self._c = LlmhipKvBlocks(k_pool.data_ptr(), v_pool.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                                 (_i64 * 3)(*k_pool.stride()[:3]), (_i64 * 3)(*v_pool.stride()[:3]), (_i64 * 3)(*k_scale.stride()),
                                 (_i64 * 3)(*v_scale.stride()), CODES[self.dtype], pages, page, page // blocks, heads, dim)
        self._ref = ctypes.addressof(self._c)
        self._apart = all(_apart(p, dim, 3) for p in (k_pool, v_pool)) and all(_apart(s, 1, 3) for s in (k_scale, v_scale))
        self._scale = 1.0 / math.sqrt(dim)
        self._append, self._read = self.lib.llmhip_kv_block_append, self.lib.llmhip_kv_block_read
        self._attend = self.lib.llmhip_kv_block_attend
        self._state = (k_pool, v_pool, k_scale, v_scale)

    def append(self, k, v, slots, q=None, out_q=None, positions=None, rope: Optional[Rope] = None, stream=None) -> None:
        """llmhip_kv_block_append: k and v [T, heads, head_dim], float32,
        bfloat16 or float16, into the slots ([T] int64; negative: nowhere),
        keys rotated by rope at positions ([T] int32); with q [T, q_heads,
        head_dim] its rotated rows go to out_q (which may be q). k, v and q
        may be views of one packed tensor. The tokens of one block stand next
        to each other in the batch, in order, as PagePool.plan gives them.
        Where a block's scale grows, its older tokens are restated."""
        dt, dev = k.dtype, self.device
        code = _ROWS.get(dt)
        if code is None:
            raise ValueError(f"k is {dt}, not float32, bfloat16 or float16")
        if not self._apart:
            raise ValueError("rows of a pool or scales overlap")
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
            _current(dev) if stream is None else _on(stream, dev, (k, v, slots, q, out_q, positions, *self._state)))
        if status:
            _check(self.lib, status)

    def read(self, slots, out_k=None, out_v=None, stream=None) -> None:
        """llmhip_kv_block_read: the keys and values of the slots ([T] int64;
        negative: a row of zeros) into out_k and out_v [T, heads, head_dim]
        of float32, bfloat16 or float16; either may be left out. They may be
        views of one tensor whose rows do not overlap."""
        out = out_k if out_k is not None else out_v
        if out is None:
            raise ValueError("out_k or out_v is required")
        dt, dev = out.dtype, self.device
        code = _ROWS.get(dt)
        if code is None:
            raise ValueError(f"the rows are {dt}, not float32, bfloat16 or float16")
        T = slots.numel()
        shape = (T, self.heads, self.head_dim)
        status = self._read(
            self.sampler.ctx, self._ref, code, T, _vector(slots, T, torch.int64, "slots", dev),
            *(_NO_ROWS if out_k is None else _out_rows(out_k, shape, dt, "out_k", dev)),
            *(_NO_ROWS if out_v is None else _out_rows(out_v, shape, dt, "out_v", dev)),
            _current(dev) if stream is None else _on(stream, dev, (slots, out_k, out_v, *self._state)))
        if status == _ERR_ARGUMENT and out_k is not None and out_v is not None:
            raise ValueError(self.lib.llmhip_last_error().decode(errors="replace"))  # rows of the one over the other's
        if status:
            _check(self.lib, status)

    def workspace(self, q_heads: int, new_tokens: int = 1):
        """A workspace for attend with q_heads query heads and so many new
        tokens of each request, whatever the batch. Calls that may overlap
        need one each."""
        if q_heads < 1 or new_tokens < 1:
            raise ValueError("q_heads and new_tokens must be at least 1")
        n = ctypes.c_size_t()
        _check(self.lib, self.lib.llmhip_kv_block_attend_workspace(self.sampler.ctx, self._ref, new_tokens, q_heads, ctypes.byref(n)))
        return torch.empty(n.value, dtype=torch.uint8, device=self.device)

    def attend(self, q, table, lens, out, workspace, window: int = 0, scale: Optional[float] = None, out_lse=None,
               stream=None) -> None:
        """llmhip_kv_block_attend: q [B, q_heads, head_dim], or [B, n, q_heads,
        head_dim] for the newest n (at most 16) tokens of each request, bfloat16
        or float16, over the request's pages in table ([B, pages] int32). lens
        ([B] int32) counts all of them: token j is attended over the first
        lens[b] - n + 1 + j tokens, of those the last `window` (0: all). out is
        like q, out_lse float32 like q without its last dimension; scale
        defaults to head_dim ** -0.5. q_heads is a multiple of the cache's
        heads."""
        dt, dev = q.dtype, self.device
        if dt is not torch.bfloat16 and dt is not torch.float16:
            raise ValueError(f"q is {dt}, not bfloat16 or float16")
        if q.dim() not in (3, 4):
            raise ValueError("q must be [B, q_heads, head_dim] or [B, tokens, q_heads, head_dim]")
        B, heads, new = q.shape[0], q.shape[-2], q.shape[1] if q.dim() == 4 else 1
        if not heads or heads % self.heads:
            raise ValueError(f"q must have a multiple of {self.heads} heads")
        if not 1 <= new <= MAX_NEW_TOKENS:
            raise ValueError(f"q must have 1 to {MAX_NEW_TOKENS} tokens of each request")
        if window < 0:
            raise ValueError("window must not be negative")
        if out_lse is None:
            lse = None
        elif out_lse.dtype is not torch.float32 or out_lse.shape != q.shape[:-1] or not out_lse.is_contiguous() \
                or out_lse.device != dev:
            raise ValueError(f"out_lse must be a contiguous float32 {list(q.shape[:-1])} tensor on {dev}")
        else:
            lse = out_lse.data_ptr()
        shape = (*q.shape[:-1], self.head_dim)
        rows, out_rows = _queries(q, shape, dt, "q", dev), _queries(out, shape, dt, "out", dev)
        if not out.is_contiguous() and not _apart(out, self.head_dim, out.dim() - 1):
            raise ValueError("rows of out overlap")
        size = workspace.numel()
        status = self._attend(
            self.sampler.ctx, self._ref, _ROWS[dt], B, new, heads, *rows, *_table(table, B, dev),
            _vector(lens, B, torch.int32, "lens", dev), window, self._scale if scale is None else scale, *out_rows, lse,
            _vector(workspace, size, torch.uint8, "workspace", dev), size,
            _current(dev) if stream is None else _on(stream, dev, (q, table, lens, out, out_lse, workspace, *self._state)))
        if status:
            _check(self.lib, status)
