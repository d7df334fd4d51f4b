"""The work around a key-value cache held in 8 bits, as measurable cases.

The cache's pages hold whole numbers of 8 bits or E4M3 values, and a scale
for each block of tokens and head that follows from the values as they are
written. A case's "op" names its operator:

  append  BlockKVCache.append   rotary positions on the new queries and keys;
                                each block's scale from the largest of its
                                values; the block's older values restated
                                where it grew; keys and values quantised into
                                their pages. What the cache then stands for
                                is read back (BlockKVCache.read), as a
                                program does that goes on with it in 16 bits
  read    BlockKVCache.read     tokens' keys and values out of their pages
  attend  BlockKVCache.attend   attention of the newest token, or the newest
                                few, of each request over its pages

A block's rule, with MAX 127 or 448: its tokens before the first new one are
kept and the others' places are new. a is the largest |value| of its new
tokens. The scale s is a / MAX, or the old scale where tokens are kept and it
is no smaller. A value x is stored as round(x * (1 / s)), a kept code c as
round(c * (old / s)).

`run` computes them in plain torch operations where `own` is false and
through the library where it is true, on the same state.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "i8": torch.int8, "e4m3": torch.float8_e4m3fn}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
MOST = {"i8": 127.0, "e4m3": 448.0}

# A serving process keeps one context for all of its calls.
_sampler = None


def _handle():
    global _sampler
    if _sampler is None:
        from scriptonait_amd.sampler import Sampler

        _sampler = Sampler(0)
    return _sampler


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------
def _append(name, T, Hq, Hkv, D, page, block, q, kv, style, dims, far, mode):
    return dict(name=name, op="append", T=T, Hq=Hq, Hkv=Hkv, D=D, page=page, block=block, q=q, kv=kv, style=style, dims=dims,
                far=far, mode=mode)


def _read(name, T, Hkv, D, page, block, q, kv):
    return dict(name=name, op="read", T=T, Hkv=Hkv, D=D, page=page, block=block, q=q, kv=kv)


def _attend(name, B, new, Hq, Hkv, D, page, block, longest, lens, window, q, kv):
    return dict(name=name, op="attend", B=B, new=new, Hq=Hq, Hkv=Hkv, D=D, page=page, block=block, longest=longest, lens=lens,
                window=window, q=q, kv=kv)


def listed():
    return [
        # One generation of a small binary32 model: latency.
        _append("append_one_f32", 1, 8, 2, 64, 16, 16, "f32", "i8", "neighbours", 64, 1024, "decode"),
        # A decode step's new tokens, each in the middle of its block.
        _append("append_decode_256", 256, 32, 8, 128, 16, 16, "bf16", "i8", "halves", 128, 131072, "decode"),
        # Prompts into an E4M3 cache, an odd number of tokens, blocks of a whole page.
        _append("append_e4m3_2047", 2047, 12, 12, 80, 64, 64, "f16", "e4m3", "halves", 80, 8192, "prompts"),
        # A full batch of prompt tokens.
        _append("append_prompt", 16384, 32, 8, 128, 64, 16, "bf16", "i8", "halves", 128, 32768, "prompts"),
        # One generation's cache of a small binary32 model, read back.
        _read("read_700_f32", 700, 2, 64, 16, 16, "f32", "i8"),
        # A prompt's tokens out of an E4M3 cache with a scale for every 4 tokens.
        _read("read_e4m3_6001", 6001, 12, 80, 24, 4, "f16", "e4m3"),
        # The requests of a batch, moved out of the cache.
        _read("read_65536", 65536, 8, 128, 64, 16, "bf16", "i8"),
        # One generation of a small model with a sliding window: latency.
        _attend("attend_one", 1, 1, 8, 2, 64, 16, 16, 700, "equal", 512, "bf16", "i8"),
        # One head for each cache head, head size 80, pages of 24, a window.
        _attend("attend_heads_f16", 37, 1, 12, 12, 80, 24, 8, 2000, "ragged", 1000, "f16", "e4m3"),
        # Four draft tokens of each request of a server batch, a scale for each token.
        _attend("attend_drafts_64", 64, 4, 32, 8, 128, 16, 1, 4096, "ragged", 0, "bf16", "i8"),
        # One generation over a very long context.
        _attend("attend_long", 1, 1, 32, 8, 128, 64, 64, 131072, "equal", 0, "bf16", "i8"),
        # A large batch of ragged lengths.
        _attend("attend_256", 256, 1, 32, 8, 128, 16, 16, 8192, "ragged", 0, "bf16", "i8"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "read", "attend", "attend"])
    Hkv = rng.choice([1, 2, 3, 4, 8, 12])
    G = rng.choice([1, 2, 4, 5, 7, 8, 12, 16])
    if Hkv * G > 48:
        G = rng.choice([1, 2, 4])
    D = rng.choice([16, 32, 64, 80, 96, 112, 128, 192, 256])
    page = rng.choice([1, 8, 16, 20, 24, 32, 64, 128, 256])
    block = rng.choice([b for b in (1, 2, 4, 8, 12, 16, 24, 32, 64, 128, 256) if page % b == 0])
    kv = rng.choice(["i8", "i8", "e4m3"])
    q = rng.choice(["bf16", "f16"] if op == "attend" else ["f32", "bf16", "f16"])
    if op == "append":
        mode = rng.choice(["decode", "prompts"])
        # Decoding requests have a block of tokens each in the state.
        most = min(16384, 200_000_000 // ((G + 2) * Hkv * D * BYTES[q]))
        most = min(most, max(64, 32_000_000 // (Hkv * D * page))) if mode == "decode" else most
        dims = rng.choice([D, D, D // 2, 0])
        return dict(op=op, T=_log(rng, 1, most), Hq=Hkv * G, Hkv=Hkv, D=D, page=page, block=block, q=q, kv=kv,
                    style=rng.choice(["halves", "neighbours"]), dims=dims, far=rng.choice([512, 8192, 131072, 1048576]), mode=mode)
    if op == "read":
        return dict(op=op, T=_log(rng, 1, min(65536, 400_000_000 // (2 * Hkv * D * (1 + BYTES[q])))), Hkv=Hkv, D=D, page=page,
                    block=block, q=q, kv=kv)
    new = rng.choice([1, 1, 1, 2, 3, 4, 8])
    most = 1_000_000_000 // (2 * Hkv * D * 2)
    B = _log(rng, 1, 300)
    longest = _log(rng, new, max(new, min(131072, most // B)))
    return dict(op=op, B=B, new=new, Hq=Hkv * G, Hkv=Hkv, D=D, page=page, block=block, longest=longest,
                lens=rng.choice(["equal", "ragged", "ragged", "skewed"]), window=rng.choice([0, 0, 128, 1000]), q=q, kv=kv)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _lens(case, seed):
    """The requests' cache lengths: on the host, from the seed."""
    rs = np.random.RandomState((seed * 7919 + 17) % (1 << 31))
    B, longest, new = case["B"], case["longest"], case["new"]
    if case["lens"] == "equal":
        lens = np.full(B, longest)
    elif case["lens"] == "ragged":
        lens = rs.randint(new, longest + 1, B)
        lens[rs.rand(B) < 0.03] = 0  # generations that have ended
    else:  # a few long requests among short ones
        lens = np.minimum(longest, new + (longest * 0.05 * rs.rand(B)).astype(np.int64))
        lens[rs.randint(0, B)] = longest
    return lens.astype(np.int64)


def _pages_for(lens, page):
    return (lens + page - 1) // page


def _round_codes(x, kv):
    """Scaled values in 32 bits to the nearest codes."""
    x = x.clamp(-MOST[kv], MOST[kv])
    return torch.round(x).to(torch.int8) if kv == "i8" else x.to(torch.float8_e4m3fn)


def _written(x, block, kv):
    """A pool [N, page, H, D] of values as a cache holds them: codes, and a
    scale for each block and head [N, page / block, H]."""
    N, page, H, D = x.shape
    x = x.view(N, page // block, block, H, D)
    s = x.abs().amax((2, 4)).float() / MOST[kv]
    codes = _round_codes(x.float() * (1.0 / s)[:, :, None, :, None], kv)
    return codes.view(N, page, H, D), s


def _cache(s, g, N, page, H, D, block, kv, dev):
    # A few channels of keys are far larger than the others.
    gain = 1.0 + 4.0 * (torch.rand(2, H, D, generator=g, device=dev) < 0.04).float()
    gain[1] = 1.0
    for i, name in enumerate(("k", "v")):
        x = torch.randn(N, page, H, D, generator=g, device=dev, dtype=torch.bfloat16)
        s[name + "_pool"], s[name + "_scale"] = _written(x * gain[i].to(x.dtype), block, kv)
    if own:
        from scriptonait_amd.kv_blocks import BlockKVCache

        s["cache"] = BlockKVCache(_handle(), s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"])
    return gain


def prepare(case, seed):
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(seed)
    rs = np.random.RandomState((seed * 15485863 + 3) % (1 << 31))
    s = {"append": _prepare_append, "read": _prepare_read, "attend": _prepare_attend}[case["op"]](case, seed, dev, g, rs)
    s["case"] = case
    return s


def _append_slots(case, rs):
    """Slots and positions of the new tokens, and the pool's pages."""
    T, page = case["T"], case["page"]
    if case["mode"] == "decode":  # each request's next token, somewhere in a page
        N = T + 3
        order = rs.permutation(N)
        return order[:T] * page + rs.randint(0, page, T), rs.randint(0, case["far"], T), N
    # Three prompts behind what their caches hold, the first of them from an
    # empty one; behind each some padding.
    run = -(-T // 3)
    first = rs.randint(0, max(1, case["far"] - run), 3)
    first[0] = 0
    N = 3 * (run // page + 2) + 3
    order = rs.permutation(N).reshape(3, -1)
    at = np.arange(T)
    pos = first[at // run] + at % run
    place = first[at // run] % page + at % run
    slots = order[at // run, place // page] * page + place % page
    slots[at % run >= run - run // 50] = -1
    return slots, pos, N


def _prepare_append(case, seed, dev, g, rs):
    T, Hq, Hkv, D = case["T"], case["Hq"], case["Hkv"], case["D"]
    slots, pos, N = _append_slots(case, rs)
    s = {}
    gain = _cache(s, g, N, case["page"], Hkv, D, case["block"], case["kv"], dev)
    # The projections' output: queries, keys and values of a token in one row.
    # Some tokens' keys and values pass all that their blocks hold.
    qkv = torch.randn(T, Hq + 2 * Hkv, D, generator=g, device=dev)
    qkv[:, Hq:] *= gain.view(2 * Hkv, D) * (0.6 + torch.rand(T, 2 * Hkv, 1, generator=g, device=dev))
    back = DTYPES["bf16" if case["q"] == "f32" else case["q"]]
    rows = N * case["page"]
    s |= dict(qkv=qkv.to(DTYPES[case["q"]]), slots=torch.from_numpy(slots.astype(np.int64)).to(dev),
              positions=torch.from_numpy(pos.astype(np.int32)).to(dev), theta=50000.0,
              out_q=torch.zeros(T, Hq, D, dtype=DTYPES[case["q"]], device=dev), every=torch.arange(rows, device=dev),
              out_k=torch.zeros(rows, Hkv, D, dtype=back, device=dev), out_v=torch.zeros(rows, Hkv, D, dtype=back, device=dev))
    if own:
        from scriptonait_amd.kv import Rope

        s["rope"] = Rope(dims=case["dims"], theta=s["theta"], style=case["style"]) if case["dims"] else None
    return s


def _prepare_read(case, seed, dev, g, rs):
    T, Hkv, D, page = case["T"], case["Hkv"], case["D"], case["page"]
    N = -(-T // page) + 3
    s = {}
    _cache(s, g, N, page, Hkv, D, case["block"], case["kv"], dev)
    # Runs of tokens in shuffled pages, some padding behind them.
    order = rs.permutation(N)
    at = np.arange(T)
    slots = order[at // page] * page + at % page
    slots[T - T // 50:] = -1
    s |= dict(slots=torch.from_numpy(slots.astype(np.int64)).to(dev))
    s |= {n: torch.zeros(T, Hkv, D, dtype=DTYPES[case["q"]], device=dev) for n in ("out_k", "out_v")}
    return s


def _prepare_attend(case, seed, dev, g, rs):
    B, new, Hq, Hkv, D, page = case["B"], case["new"], case["Hq"], case["Hkv"], case["D"], case["page"]
    lens = _lens(case, seed)
    pages = _pages_for(lens, page)
    N = int(pages.sum()) + 3
    P = max(1, int(_pages_for(np.array([case["longest"]]), page)[0]))
    order = rs.permutation(N)
    table = np.zeros((B, P), dtype=np.int64)
    table[np.arange(P)[None, :] < pages[:, None]] = order[:int(pages.sum())]
    s = {}
    _cache(s, g, N, page, Hkv, D, case["block"], case["kv"], dev)
    # Queries that attend to some tokens far more than to others: scores of
    # a spread of two or more.
    shape = (B, Hq, D) if new == 1 else (B, new, Hq, D)
    qs = (2.0 * torch.randn(*shape, generator=g, device=dev)).to(DTYPES[case["q"]])
    s |= dict(q=qs, lens=torch.from_numpy(lens.astype(np.int32)).to(dev), table=torch.from_numpy(table.astype(np.int32)).to(dev),
              scale=1.0 / math.sqrt(D), out=torch.zeros_like(qs), lse=torch.zeros(shape[:-1], dtype=torch.float32, device=dev))
    if own:
        s["workspace"] = s["cache"].workspace(Hq, new)
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(s):
    if s["case"]["op"] == "append":
        return _own_append(s) if own else _plain_append(s)
    if s["case"]["op"] == "read":
        return _own_read(s) if own else _plain_read(s)
    return _own_attend(s) if own else _plain_attend(s)


def _own_append(s):
    Hq, Hkv = s["case"]["Hq"], s["case"]["Hkv"]
    x = s["qkv"]
    s["cache"].append(x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], s["slots"], q=x[:, :Hq], out_q=s["out_q"], positions=s["positions"],
                      rope=s["rope"])
    s["cache"].read(s["every"], s["out_k"], s["out_v"])
    return dict(q=s["out_q"], k=s["out_k"], v=s["out_v"], k_scale=s["k_scale"], v_scale=s["v_scale"])


def _own_read(s):
    s["cache"].read(s["slots"], s["out_k"], s["out_v"])
    return dict(k=s["out_k"], v=s["out_v"])


def _own_attend(s):
    s["cache"].attend(s["q"], s["table"], s["lens"], s["out"], s["workspace"], window=s["case"]["window"], scale=s["scale"],
                      out_lse=s["lse"])
    return dict(out=s["out"], lse=s["lse"])


def _plain_rotate(x, positions, dims, theta, style):
    """x [T, H, D] in 32 bits, its first `dims` values rotated by their positions."""
    if not dims:
        return x
    half = dims // 2
    i = torch.arange(half, device=x.device, dtype=torch.float64)
    angle = positions.double()[:, None] * torch.pow(torch.tensor(theta, dtype=torch.float64, device=x.device), -2.0 * i / dims)
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    if style == "halves":
        a, b = x[..., :half], x[..., half:dims]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., dims:]], -1)
    a, b = x[..., 0:dims:2], x[..., 1:dims:2]
    turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([turned, x[..., dims:]], -1)


def _plain_write(pool, scale, x, slots, kv):
    """New rows x [T, H, D] in 32 bits into their slots."""
    N, page, H, D = pool.shape
    block = page // scale.shape[1]
    rows, blocks = N * page, N * scale.shape[1]
    live = slots >= 0
    of = torch.where(live, slots // block, blocks)
    # Of each block: the largest new value, and where its new tokens begin.
    top = x.new_zeros(blocks + 1, H).scatter_reduce_(0, of[:, None].expand(-1, H), x.abs().amax(-1), "amax")[:blocks]
    begin = torch.full((blocks + 1,), block, device=x.device).scatter_reduce_(0, of, torch.where(live, slots % block, block), "amin")
    begin = begin[:blocks, None]
    old = scale.view(blocks, H)
    s = torch.where(begin > 0, torch.maximum(old, top / MOST[kv]), top / MOST[kv])
    # Kept tokens of blocks whose scale grew, then the new ones.
    place = torch.arange(block, device=x.device)
    kept = (place < begin)[:, :, None] & (s > old)[:, None] & (begin < block)[:, None]
    codes = pool.view(blocks, block, H, D)
    again = _round_codes(codes.float() * torch.where(s > 0, old / s, 0.0)[:, None, :, None], kv)
    codes = torch.where(kept[..., None], again.view(torch.uint8), codes.view(torch.uint8)).view(rows, H * D)
    r = torch.where(s > 0, 1.0 / s, 0.0)
    token = torch.full((rows + 1,), -1, device=x.device).scatter_(0, torch.where(live, slots, rows),
                                                                 torch.arange(len(x), device=x.device))[:rows]
    new = _round_codes(x * r[of.clamp(max=blocks - 1)][:, :, None], kv).view(torch.uint8).view(len(x), H * D)
    pool.view(torch.uint8).view(rows, H * D).copy_(torch.where(token[:, None] >= 0, new[token.clamp(min=0)], codes))
    scale.copy_(torch.where(begin < block, s, old).view(scale.shape))


def _plain_values(pool, scale, slots, dtype):
    """The tokens' values; zeros for padding."""
    N, page, H, D = pool.shape
    block = page // scale.shape[1]
    at = slots.clamp(min=0)
    codes = pool.view(torch.uint8).view(N * page, H, D)[at].view(pool.dtype)
    x = codes.float() * scale.view(-1, H)[at // block][:, :, None]
    return torch.where((slots >= 0)[:, None, None], x, 0.0).to(dtype)


def _plain_append(s):
    c = s["case"]
    Hq, Hkv = c["Hq"], c["Hkv"]
    x = s["qkv"].float()
    turned = _plain_rotate(x[:, :Hq + Hkv], s["positions"], c["dims"], s["theta"], c["style"])
    _plain_write(s["k_pool"], s["k_scale"], turned[:, Hq:], s["slots"], c["kv"])
    _plain_write(s["v_pool"], s["v_scale"], x[:, Hq + Hkv:], s["slots"], c["kv"])
    k, v = (_plain_values(s[n + "_pool"], s[n + "_scale"], s["every"], s["out_k"].dtype) for n in "kv")
    return dict(q=turned[:, :Hq].to(s["qkv"].dtype), k=k, v=v, k_scale=s["k_scale"], v_scale=s["v_scale"])


def _plain_read(s):
    k, v = (_plain_values(s[n + "_pool"], s[n + "_scale"], s["slots"], s["out_k"].dtype) for n in "kv")
    return dict(k=k, v=v)


def _plain_attend(s):
    c = s["case"]
    B, new, Hq, Hkv, D, page = c["B"], c["new"], c["Hq"], c["Hkv"], c["D"], c["page"]
    G = Hq // Hkv
    table = s["table"].long()
    L = table.shape[1] * page
    q = s["q"].float().view(B, new, Hkv, G, D).transpose(1, 2).reshape(B, Hkv, new * G, D)
    t = torch.arange(L, device=q.device)
    # The newest tokens' own lengths: the last one sees all of the request.
    ends = s["lens"].long()[:, None] - new + 1 + torch.arange(new, device=q.device)
    seen = t < ends[..., None]
    if c["window"]:
        seen = seen & (t >= ends[..., None] - c["window"])
    any_seen = seen.any(1)
    seen = seen[:, None, :, None].expand(B, 1, new, G, L).reshape(B, 1, new * G, L)

    def rows(name):  # [B, Hkv, L, D]; what no query may see reads as zero
        pool, scale = s[name + "_pool"], s[name + "_scale"]
        block = page // scale.shape[1]
        x = pool.view(torch.uint8)[table].view(pool.dtype).view(B, -1, block, Hkv, D).float()
        x = (x * scale[table].view(B, -1, 1, Hkv, 1)).view(B, L, Hkv, D).transpose(1, 2)
        return torch.where(any_seen[:, None, :, None], x, 0.0)

    scores = torch.matmul(q, rows("k").transpose(-1, -2)) * s["scale"]
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e, rows("v")) / torch.where(total == 0, 1.0, total)

    def back(x):  # [B, Hkv, new * G, ...] to [B, new, Hq, ...]
        return x.view(B, Hkv, new, G, -1).transpose(1, 2).reshape(B, new, Hq, -1)

    return dict(out=back(o).to(s["q"].dtype).view(s["q"].shape), lse=back(top + torch.log(total)).view(s["lse"].shape))


# ---------------------------------------------------------------------------
# What a pass cannot do without, and its outputs from the definitions
# ---------------------------------------------------------------------------
def work(case):
    Hkv, D = case["Hkv"], case["D"]
    if case["op"] == "append":
        T, Hq, q = case["T"], case["Hq"], BYTES[case["q"]]
        rs = np.random.RandomState(3)
        rows = _append_slots(case, rs)[2] * case["page"]
        # queries, keys and values in, queries out; codes written; the cache's values out
        x = T * D * ((2 * Hq + 2 * Hkv) * q + 2 * Hkv)
        return {"bytes": x + 12 * T + 2 * rows * Hkv * (2 * D + 4.0 / case["block"]), "flops": 3 * T * case["dims"] * (Hq + Hkv)}
    if case["op"] == "read":
        T = case["T"]
        return {"bytes": T * (8 + 2 * Hkv * (D * (1 + BYTES[case["q"]]) + 4.0 / case["block"])), "flops": 2 * T * Hkv * D}
    lens = _lens(case, 0)
    if case["window"]:
        lens = np.minimum(lens, case["window"] + case["new"] - 1)
    tokens, n = int(lens.sum()), case["new"] * case["Hq"]
    return {"bytes": 2 * tokens * Hkv * (D + 4.0 / case["block"]) + case["B"] * n * (2 * D * BYTES[case["q"]] + 4),
            "flops": 4 * tokens * n * D}


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"append": _exact_append, "read": _exact_read, "attend": _exact_attend}[case["op"]](case, s)


def _exact_codes(x, kv):
    if kv == "i8":
        return torch.round(x).clamp(-127, 127)
    # E4M3: three bits behind the leading one, steps of 2^-9 at the least.
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0**-6))) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _exact_write(pool, scale, x, slots, kv):
    """Block by block, as a program on the host would write them. The pool's
    values and the scales, in 64 bits."""
    N, page, H, D = pool.shape
    block = page // scale.shape[1]
    codes = pool.double().view(-1, block, H, D).clone()
    scale = scale.double().view(-1, H).clone()
    at = slots.cpu().numpy()
    if block == 1 or not (np.diff(at[at >= 0]) == 1).any():  # one token in each block: all at once
        t = torch.from_numpy(np.flatnonzero(at >= 0)).to(x.device)
        b, o = slots[t] // block, slots[t] % block
        top = x[t].abs().amax(-1) / MOST[kv]
        s = torch.where((o > 0)[:, None] & (scale[b] > top), scale[b], top)
        grown = (torch.arange(block, device=x.device) < o[:, None])[:, :, None] & (s > scale[b])[:, None]
        codes[b] = torch.where(grown[..., None], _exact_codes(codes[b] * (scale[b] / s)[:, None, :, None], kv), codes[b])
        codes[b, o] = _exact_codes(x[t] / s[:, :, None], kv)
        scale[b] = s
    else:
        t = 0
        while t < len(at):
            n = 1
            while t + n < len(at) and at[t] >= 0 and at[t + n] == at[t] + n and at[t + n] % block:
                n += 1
            if at[t] >= 0:
                b, o = int(at[t]) // block, int(at[t]) % block
                s = x[t:t + n].abs().amax((0, 2)) / MOST[kv]
                if o:
                    s = torch.maximum(s, scale[b])
                    if o and bool((s > scale[b]).any()):
                        grown = (s > scale[b])[:, None]
                        codes[b, :o] = torch.where(grown, _exact_codes(codes[b, :o] * (scale[b] / s)[:, None], kv), codes[b, :o])
                codes[b, o:o + n] = _exact_codes(x[t:t + n] / s[:, None], kv)
                scale[b] = s
            t += n
    return (codes * scale[:, None, :, None]).view(N * page, H, D), scale.view(N, page // block, H)


def _exact_append(case, s):
    Hq, Hkv, dims = case["Hq"], case["Hkv"], case["dims"]
    x = s["qkv"].double()
    turned = x[:, :Hq + Hkv].clone()
    if dims:
        half = dims // 2
        freq = torch.tensor([s["theta"] ** (-2.0 * i / dims) for i in range(half)], dtype=torch.float64, device=x.device)
        # A pair as a complex number, turned by its position's angle.
        at = torch.arange(half, device=x.device)
        first = at if case["style"] == "halves" else 2 * at
        second = at + half if case["style"] == "halves" else 2 * at + 1
        z = torch.complex(turned[..., first], turned[..., second])
        angle = s["positions"].double()[:, None, None] * freq
        z = z * torch.polar(torch.ones_like(angle), angle)
        turned[..., first], turned[..., second] = z.real, z.imag
    k, k_scale = _exact_write(s["k_pool"], s["k_scale"], turned[:, Hq:], s["slots"], case["kv"])
    v, v_scale = _exact_write(s["v_pool"], s["v_scale"], x[:, Hq + Hkv:], s["slots"], case["kv"])
    return dict(q=turned[:, :Hq], k=k, v=v, k_scale=k_scale, v_scale=v_scale)


def _exact_read(case, s):
    found = {}
    for name in "kv":
        scale = s[name + "_scale"].double().repeat_interleave(case["block"], 1)  # of each token
        x = s[name + "_pool"].double() * scale[..., None]
        out = torch.zeros(case["T"], case["Hkv"], case["D"], dtype=torch.float64, device=x.device)
        live = s["slots"] >= 0
        out[live] = x.flatten(0, 1)[s["slots"][live]]
        found[name] = out
    return found


def _exact_attend(case, s):
    """Request by request and token by token, over the rows that it may see."""
    B, new, Hq, Hkv, D, page, block = (case[k] for k in ("B", "new", "Hq", "Hkv", "D", "page", "block"))
    G = Hq // Hkv
    out = torch.zeros(B, new, Hq, D, dtype=torch.float64, device=s["q"].device)
    lse = torch.full((B, new, Hq), -math.inf, dtype=torch.float64, device=out.device)
    q = s["q"].view(B, new, Hq, D)
    pools = [s[n + "_pool"].view(torch.uint8).view(-1, Hkv, D) for n in "kv"]
    scales = [s[n + "_scale"].view(-1, Hkv) for n in "kv"]
    for b, n in enumerate(s["lens"].cpu().tolist()):
        if n == 0:
            continue
        begin = max(0, n - new + 1 - case["window"]) if case["window"] else 0
        t = torch.arange(begin, n, device=out.device)
        slot = s["table"][b].long()[t // page] * page + t % page
        k, v = (p[slot].view(DTYPES[case["kv"]]).double() * c[slot // block].double()[:, :, None] for p, c in zip(pools, scales))
        for j in range(new):
            hi = n - new + 1 + j
            lo = max(0, hi - case["window"]) if case["window"] else 0
            if hi <= lo:
                continue
            for h in range(Hkv):
                heads = slice(h * G, (h + 1) * G)
                x = (q[b, j, heads].double() @ k[lo - begin:hi - begin, h].t().contiguous()) * s["scale"]
                lse[b, j, heads] = torch.logsumexp(x, -1)
                out[b, j, heads] = torch.softmax(x, -1) @ v[lo - begin:hi - begin, h].contiguous()
    return dict(out=out.view(s["q"].shape), lse=lse.view(s["lse"].shape))
