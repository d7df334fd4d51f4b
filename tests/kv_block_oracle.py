"""The 8-bit cache with a scale for each block of tokens and head on the host:
what a call writes, bit for bit where the definition fixes the bits, and error
bounds that follow from the types elsewhere."""
import numpy as np
import torch

import kv_oracle

MOST = {torch.int8: np.float32(127), torch.float8_e4m3fn: np.float32(448)}
TINY = np.float32(2.0**-126)


def codes(x, kind):
    """Scaled binary32 values (numpy) to codes, as a torch tensor."""
    most = MOST[kind]
    if kind is torch.int8:
        y = np.clip(np.rint(x), -most, most)
        return torch.from_numpy(np.where(np.isnan(y), np.float32(0), y).astype(np.int8))
    y = np.where(np.isnan(x), x, np.clip(x, -most, most)).astype(np.float32)
    return torch.from_numpy(y).to(kind)


def raw(t):
    return t.view(torch.uint8) if t.dtype is torch.float8_e4m3fn else t


def runs(slots, block):
    """(first token, tokens) of each block's neighbouring new tokens."""
    t = 0
    while t < len(slots):
        n = 1
        if slots[t] >= 0:
            while t + n < len(slots) and slots[t + n] == slots[t] + n and slots[t + n] % block:
                n += 1
            yield t, n
        t += n


def write(pool, scale, x, slots):
    """New rows x [T, H, D] (binary32, as they are quantised) into a copy of the
    pool and its scales: (pool, scale), each bit of them fixed."""
    pool, scale = pool.clone(), scale.clone()
    pages, page, H, D = pool.shape
    block = page // scale.shape[1]
    kind, most = pool.dtype, MOST[pool.dtype]
    x = x.numpy()
    with np.errstate(all="ignore"):
        for t, n in runs(slots, block):
            if slots[t] >= pages * page:
                continue
            p, at = slots[t] // page, slots[t] % page
            b, place = at // block, at % block
            size = np.abs(x[t:t + n])
            top = np.where(np.isfinite(size), size, np.float32(0)).max((0, 2))
            s = top / most
            s = np.where(s < TINY, np.float32(0), s)
            old = scale[p, b].numpy().copy() if place else np.zeros(H, np.float32)
            s = np.where(old > s, old, s)
            r = np.where(s > 0, np.float32(1) / s, np.float32(1)).astype(np.float32)
            if place:
                f = (old / s).astype(np.float32)[:, None]
                kept = pool[p, b * block:at].float().numpy()
                again = codes(kept * f, kind)
                grown = torch.from_numpy(s > old)[:, None]
                raw(pool)[p, b * block:at] = torch.where(grown, raw(again), raw(pool)[p, b * block:at])
            raw(pool)[p, at:at + n] = raw(codes(x[t:t + n] * r[:, None], kind))
            scale[p, b] = torch.from_numpy(s.astype(np.float32))
    return pool, scale


def values(pool, scale):
    """What a pool stands for, [pages, page, H, D] in binary64."""
    block = pool.shape[1] // scale.shape[1]
    return pool.double() * scale.double().repeat_interleave(block, 1)[..., None]


def half_step(value, s, kind):
    """How far a code times s may be from what it was rounded from, in
    binary64; s broadcasts against value. Half a step of the codes, and the
    roundings of 1 / s, of the product and of the code times s (each 2^-24 of
    the value)."""
    u = kv_oracle.F32
    if kind is torch.int8:
        return s * (0.5 + 1e-12) + 4 * u * value.abs()
    return value.abs() * 2.0**-4 * 1.001 + s * 2.0**-10


def attend(q, pool, scale, table, lens, window, factor):
    """q [B, n, Hq, D] over the newest n tokens' own lengths; pool and scale are
    pairs. out, lse and their bounds, [B, n, Hq, D] and [B, n, Hq], by
    kv_oracle.attend on what the codes stand for. Of its bounds' 8 u the scale
    of a key's block and that of a value's take one rounding each.

    Those bounds are relative to the numerators. A numerator has no less than
    binary32's and bfloat16's smallest normal number to be off by: where it is
    below 2^-126 it counts as 0, and where its first part is below 2^-117 its
    second part (2^-9 of it) is: 2^-126 each. The sum of the numerators is at
    least 2^-8 (the reference is passed by 8 in the exponent at most, and the
    largest is at least 1 when it moves), so n tokens' outputs are off by
    n 2^-117 max |v| besides."""
    k, v = (values(p, s) for p, s in zip(pool, scale))
    n = q.shape[1]
    cap = table.shape[1] * pool[0].shape[1]
    lens = lens.clamp(0, cap)
    found = [kv_oracle.attend(q[:, j], k, v, table, lens - n + 1 + j, window, factor) for j in range(n)]
    out, lse, out_tol, lse_tol = (torch.stack(x, 1) for x in zip(*found))
    most = torch.nan_to_num(v).abs().amax()  # (what no request may see can be NaN)
    return out, lse, out_tol + lens[:, None, None, None] * 2.0**-117 * most, lse_tol
