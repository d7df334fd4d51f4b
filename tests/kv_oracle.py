"""The paged key-value cache's operators in 64 bits on the host, from their
definitions, and the error bounds that follow from the types."""
import math

import torch

HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
HALF_STEP[torch.float8_e4m3fn] = 2.0**-4
F32 = 2.0**-24


def plan(page, ring, state, lens, table, T, new=None, release=None):
    """The requests one after the other. Lists in, a dict of lists out."""
    ring, table = list(ring), [list(r) for r in table]
    before, N = list(ring), len(ring)
    head, free = state
    tail, left, taken, asked, stop = head + free, free, 0, 0, False
    slots, positions = [-1] * T, [0] * T
    out_lens, granted, start = list(lens), [0] * len(lens), [0]
    for r in range(len(lens)):
        gone = release is not None and release[r] != 0
        if gone:
            for p in range(-(-lens[r] // page)):
                ring[tail % N] = table[r][p]
                tail += 1
            out_lens[r] = 0
        n = new[r] if new is not None else int(not gone)
        first = asked
        asked += n
        start.append(asked)
        base = out_lens[r]
        if base + n > len(table[r]) * page or asked > T:
            continue
        have, want = -(-base // page), -(-(base + n) // page)
        if want > have and (stop or want - have > left):
            stop = True
            continue
        for p in range(have, want):
            table[r][p] = before[(head + taken) % N]
            taken += 1
            left -= 1
        granted[r], out_lens[r] = n, base + n
        for i in range(n):
            pos = base + i
            positions[first + i] = pos
            slots[first + i] = table[r][pos // page] * page + pos % page
    return dict(lens=out_lens, granted=granted, start=start, slots=slots, positions=positions, table=table, ring=ring,
                state=[(head + taken) % N, tail - head - taken])


def rotate(x, positions, freqs, style):
    """x [T, H, D] in binary64, its first 2 len(freqs) values turned."""
    x = x.clone()
    half = len(freqs)
    if not half:
        return x
    first = torch.arange(half) if style == "halves" else 2 * torch.arange(half)
    second = first + (half if style == "halves" else 1)
    angle = positions.double()[:, None, None] * torch.tensor(freqs, dtype=torch.float64)
    z = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.ones_like(angle), angle)
    x[..., first], x[..., second] = z.real, z.imag
    return x


def rotate_bound(x, freqs, style):
    """How far a pair's binary32 values may be from rotate's: cosine and sine
    are off by half a step (and 2^-40 of their own), each product, the sum of
    the two and no more are rounded, all relative to |a| + |b|."""
    size = x.abs()
    half = len(freqs)
    first = torch.arange(half) if style == "halves" else 2 * torch.arange(half)
    second = first + (half if style == "halves" else 1)
    out = torch.zeros_like(x)
    pair = size[..., first] + size[..., second]
    out[..., first], out[..., second] = 4 * F32 * pair, 4 * F32 * pair
    return out


def attend(q, k_pool, v_pool, table, lens, window, scale, k_scale=None, v_scale=None):
    """out, lse and their error bounds, [B, Hq, D] and [B, Hq], in binary64.
    Tokens on pages outside the pool are left out.

    With u = 2^-24 a score is off by at most ds = (D + 8) u max(scale |q| |k|)
    (D products summed in any order, the scale, its base-2 form, the
    subtraction of the maximum); a probability's numerator by 2 ds + 8 u of
    itself; sums of n terms by n u of the terms' absolute sum. Both sums are
    off, so the quotient by twice that. 16-bit types hold a numerator as two
    values of their type: 2^-16 of it, and float16 2^-24 of the largest
    value, as it has no smaller steps."""
    B, Hq, D = q.shape
    pages, page, Hkv = k_pool.shape[:3]
    G = Hq // Hkv
    out, lse = torch.zeros(B, Hq, D, dtype=torch.float64), torch.full((B, Hq), -math.inf, dtype=torch.float64)
    out_tol, lse_tol = torch.zeros_like(out), torch.zeros_like(lse)
    cap = table.shape[1] * page
    for b in range(B):
        n = max(0, min(int(lens[b]), cap))
        t = torch.arange(max(0, n - window) if window else 0, n)
        ids = table[b].long()[t // page]
        good = (ids >= 0) & (ids < pages)
        t, ids = t[good], ids[good]
        if not len(t):
            continue
        raw = [p.view(torch.uint8) if p.element_size() == 1 else p for p in (k_pool, v_pool)]
        k, v = (p[ids, t % page].view(k_pool.dtype).double() for p in raw)
        if k_scale is not None:
            k, v = k * k_scale.double()[:, None], v * v_scale.double()[:, None]
        for h in range(Hkv):
            hs = slice(h * G, (h + 1) * G)
            x = q[b, hs].double()
            s = x @ k[:, h].T * scale
            ds = (D + 8) * F32 * (abs(scale) * (x.abs() @ k[:, h].abs().T)).amax(-1)
            p = torch.softmax(s, -1)
            lse[b, hs] = torch.logsumexp(s, -1)
            out[b, hs] = p @ v[:, h]
            rel = 2 * ds + (8 + len(t)) * F32
            lse_tol[b, hs] = ds + rel + 8 * F32 * (lse[b, hs].abs() + 1)
            rel = rel * 2
            if q.dtype != torch.float32:
                rel = rel + 2.0**-16
            tol = rel[:, None] * (p @ v[:, h].abs())
            if q.dtype == torch.float16:
                tol = tol + F32 * v[:, h].abs().amax(0)
            out_tol[b, hs] = tol
    out_tol = out_tol * (1 + HALF_STEP[q.dtype]) + HALF_STEP[q.dtype] * out.abs()
    if q.dtype == torch.float16:
        out_tol = out_tol + 2.0**-25  # subnormals
    return out, lse, out_tol, lse_tol
