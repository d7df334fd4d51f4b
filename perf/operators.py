"""The work around a decode step's key-value cache, as measurable cases.

Three operators that a serving loop calls between two sampling steps. A
case's "op" names its operator:

  plan    PagePool.plan    pages for the tokens that each request adds: block
                           tables, slot map, positions, the free pages
  append  KVCache.append   rotary positions on the new queries and keys, keys
                           and values into their pages
  attend  KVCache.attend   attention of one new token for each request over
                           its pages

`run` computes them in plain torch operations where `own` is false and
through the library where it is true, on the same state.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
BYTES = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1}
E4M3_MAX = 448.0

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
def _plan(name, R, page, table, mode, T, tight=False):
    return dict(name=name, op="plan", R=R, page=page, table=table, mode=mode, T=T, tight=tight)


def _append(name, T, Hq, Hkv, D, page, q, kv, style, dims, far):
    return dict(name=name, op="append", T=T, Hq=Hq, Hkv=Hkv, D=D, page=page, q=q, kv=kv, style=style, dims=dims, far=far)


def _attend(name, B, Hq, Hkv, D, page, longest, lens, window, q, kv):
    return dict(name=name, op="attend", B=B, Hq=Hq, Hkv=Hkv, D=D, page=page, longest=longest, lens=lens, window=window, q=q,
                kv=kv)


def listed():
    return [
        # A decode step of a small server batch: latency.
        _plan("plan_decode_64", 64, 16, 256, "decode", 64),
        # A decode step of a large batch, some of whose generations have ended.
        _plan("plan_decode_1000", 1000, 16, 512, "decode", 1024),
        # New prompts beside running generations, packed into one token batch.
        _plan("plan_prompts", 300, 16, 512, "mixed", 65536),
        # One generation of a small binary32 model, neighbouring pairs rotated.
        _append("append_one_f32", 1, 8, 2, 64, 16, "f32", "f32", "neighbours", 64, 1024),
        # A decode step's new tokens, grouped heads.
        _append("append_decode_256", 256, 32, 8, 128, 16, "bf16", "bf16", "halves", 128, 131072),
        # Prompts into an 8-bit cache, an odd number of tokens.
        _append("append_e4m3_2047", 2047, 32, 8, 128, 16, "bf16", "e4m3", "halves", 128, 8192),
        # A full batch of prompt tokens.
        _append("append_prompt", 16384, 32, 8, 128, 64, "bf16", "bf16", "halves", 128, 32768),
        # One generation of a small binary32 model with a sliding window.
        _attend("attend_one_f32", 1, 8, 2, 64, 16, 700, "equal", 512, "f32", "f32"),
        # One head for each cache head, head size 80, pages of 24, a window.
        _attend("attend_heads_f16", 37, 12, 12, 80, 24, 2000, "ragged", 1000, "f16", "f16"),
        # A server batch of ragged lengths.
        _attend("attend_64", 64, 32, 8, 128, 16, 4096, "ragged", 0, "bf16", "bf16"),
        # One generation over a very long context.
        _attend("attend_long", 1, 32, 8, 128, 64, 131072, "equal", 0, "bf16", "bf16"),
        # A large batch over an 8-bit cache.
        _attend("attend_256_e4m3", 256, 32, 8, 128, 16, 8192, "ragged", 0, "bf16", "e4m3"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend"])
    if op == "plan":
        mode = rng.choice(["decode", "mixed"])
        R = _log(rng, 1, 1500)
        page = rng.choice([1, 8, 16, 24, 32, 64, 128])
        table = max(1, 8192 // page) if R <= 512 else max(1, 4096 // page)
        T = R + rng.randrange(1, 65) if mode == "decode" else _log(rng, 512, 65536)
        return dict(op=op, R=R, page=page, table=table, mode=mode, T=T, tight=rng.random() < 0.25)
    Hkv = rng.choice([1, 2, 3, 4, 8, 12])
    G = rng.choice([1, 2, 4, 5, 7, 8, 12, 16])
    if Hkv * G > 48:
        G = rng.choice([1, 2, 4])
    D = rng.choice([16, 32, 64, 80, 96, 112, 128, 192, 256])
    page = rng.choice([1, 8, 16, 20, 24, 32, 64, 128, 256])
    q, kv = rng.choice([("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "e4m3"), ("f16", "e4m3")])
    if op == "append":
        most = min(16384, 200_000_000 // ((G + 2) * Hkv * D * BYTES[q]))
        dims = rng.choice([D, D, D // 2, 0])
        return dict(op=op, T=_log(rng, 1, most), Hq=Hkv * G, Hkv=Hkv, D=D, page=page, q=q, kv=kv,
                    style=rng.choice(["halves", "neighbours"]), dims=dims, far=rng.choice([512, 8192, 131072, 1048576]))
    most = 1_000_000_000 // (2 * Hkv * D * max(2, BYTES[kv]))
    B = _log(rng, 1, 300)
    longest = _log(rng, 1, max(1, min(131072, most // B)))
    return dict(op=op, B=B, Hq=Hkv * G, Hkv=Hkv, D=D, page=page, longest=longest,
                lens=rng.choice(["equal", "ragged", "ragged", "skewed"]), window=rng.choice([0, 0, 128, 1000]), q=q, kv=kv)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _lens(case, seed):
    """The requests' cache lengths: on the host, from the seed."""
    rs = np.random.RandomState((seed * 7919 + 17) % (1 << 31))
    B, longest = case["B"], case["longest"]
    if case["lens"] == "equal":
        lens = np.full(B, longest)
    elif case["lens"] == "ragged":
        lens = rs.randint(1, longest + 1, B)
        lens[rs.rand(B) < 0.03] = 0  # generations that have ended
    else:  # a few long requests among short ones
        lens = np.minimum(longest, 1 + (longest * 0.05 * rs.rand(B)).astype(np.int64))
        lens[rs.randint(0, B)] = longest
    return lens.astype(np.int64)


def _pages_for(lens, page):
    return (lens + page - 1) // page


def _plan_host(case, seed):
    rs = np.random.RandomState((seed * 104729 + 5) % (1 << 31))
    R, page, table, T = case["R"], case["page"], case["table"], case["T"]
    cap = page * table
    lens = rs.randint(0, cap, R)
    release = np.zeros(R, dtype=np.int64)
    new = None
    if case["mode"] == "decode":
        release[rs.rand(R) < 0.03] = 1
        need = _pages_for(lens + 1, page) - _pages_for(lens, page)
        need[release == 1] = 0
    else:
        fresh = rs.rand(R) < 0.2
        fresh[rs.randint(0, R)] = True
        lens[fresh] = 0
        # Most of the token batch belongs to the prompts; the rest decode.
        share = rs.rand(R) * fresh
        new = np.where(fresh, 1 + (share / share.sum() * max(0, T - 2 * R)).astype(np.int64), 1)
        need = _pages_for(lens + new, page) - _pages_for(lens, page)
    used = int(_pages_for(lens, page).sum())
    free = int(need.sum() * (0.5 if case["tight"] else 1.5)) + 1
    return rs, lens, release, new, used, free


def prepare(case, seed):
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(seed)
    if case["op"] == "plan":
        s = _prepare_plan(case, seed, dev)
    elif case["op"] == "append":
        s = _prepare_append(case, seed, dev, g)
    else:
        s = _prepare_attend(case, seed, dev, g)
    s["case"] = case
    return s


def _prepare_plan(case, seed, dev):
    rs, lens, release, new, used, free = _plan_host(case, seed)
    R, page, table, T = case["R"], case["page"], case["table"], case["T"]
    N = R * table + 2 * (R + T // page) + 8  # the pool serves more requests than these
    order = rs.permutation(N)
    have = _pages_for(lens, page)
    rows = np.zeros((R, table), dtype=np.int64)
    rows[np.arange(table)[None, :] < have[:, None]] = order[:used]
    head = int(rs.randint(0, N))
    ring = np.zeros(N, dtype=np.int64)
    ring[(head + np.arange(free)) % N] = order[used:used + free]

    def i32(x):
        return torch.from_numpy(np.asarray(x, dtype=np.int32)).to(dev)

    s = dict(lens=i32(lens), release=i32(release) if new is None else None, new=None if new is None else i32(new),
             table=i32(rows), ring=i32(ring), free=i32([head, free]))
    # The outputs that a serving loop keeps from step to step.
    s |= dict(out_lens=torch.zeros(R, dtype=torch.int32, device=dev), granted=torch.zeros(R, dtype=torch.int32, device=dev),
              start=torch.zeros(R + 1, dtype=torch.int32, device=dev), slots=torch.zeros(T, dtype=torch.int64, device=dev),
              positions=torch.zeros(T, dtype=torch.int32, device=dev), out_free=torch.zeros(2, dtype=torch.int32, device=dev))
    if own:
        from scriptonait_amd.kv import PagePool

        s["pool"] = PagePool(_handle(), N, page, free_ring=s["ring"], free_state=s["free"])
    return s


def _store(x, kv, scale=None):
    """Values as the cache's type holds them; scale: one for each head."""
    if kv == "e4m3":
        return (x.float() / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(DTYPES[kv])
    return x.to(DTYPES[kv])


def _prepare_append(case, seed, dev, g):
    T, Hq, Hkv, D, page = case["T"], case["Hq"], case["Hkv"], case["D"], case["page"]
    q, kv = case["q"], case["kv"]
    rs = np.random.RandomState((seed * 15485863 + 3) % (1 << 31))
    # The projections' output: queries, keys and values of a token in one row.
    qkv = torch.randn(T, Hq + 2 * Hkv, D, generator=g, device=dev).to(DTYPES[q])
    N = (T + page - 1) // page + 3
    scales = None
    if kv == "e4m3":
        scales = [torch.rand(Hkv, generator=g, device=dev) * 0.02 + 0.005 for _ in range(2)]
    pool = [_store(torch.randn(N, page, Hkv, D, generator=g, device=dev), kv, scales and scales[i]) for i in range(2)]
    # Runs of consecutive positions (prompts) in shuffled pages; a token in
    # fifty is a batch's padding.
    order = rs.permutation(N)
    at = np.arange(T)
    slots = order[at // page] * page + at % page
    slots[rs.rand(T) < 0.02] = -1
    run_len = max(1, T // 3)
    first = rs.randint(0, max(1, case["far"] - run_len), T // run_len + 1)
    positions = first[at // run_len] + at % run_len
    s = dict(qkv=qkv, k_pool=pool[0], v_pool=pool[1], scales=scales,
             slots=torch.from_numpy(slots.astype(np.int64)).to(dev),
             positions=torch.from_numpy(positions.astype(np.int32)).to(dev), theta=50000.0,
             out_q=torch.zeros(T, Hq, D, dtype=DTYPES[q], device=dev))
    if own:
        from scriptonait_amd.kv import KVCache, Rope

        s["cache"] = KVCache(_handle(), pool[0], pool[1], *(scales or ()))
        s["rope"] = Rope(dims=case["dims"], theta=s["theta"], style=case["style"]) if case["dims"] else None
    return s


def _prepare_attend(case, seed, dev, g):
    B, Hq, Hkv, D, page = case["B"], case["Hq"], case["Hkv"], case["D"], case["page"]
    q, kv = case["q"], case["kv"]
    rs = np.random.RandomState((seed * 32452843 + 9) % (1 << 31))
    lens = _lens(case, seed)
    pages = _pages_for(lens, page)
    N = int(pages.sum()) + 3
    P = max(1, int(_pages_for(np.array([case["longest"]]), page)[0]))
    order = rs.permutation(N)
    table = np.zeros((B, P), dtype=np.int64)
    table[np.arange(P)[None, :] < pages[:, None]] = order[:int(pages.sum())]
    scales = None
    if kv == "e4m3":
        scales = [torch.rand(Hkv, generator=g, device=dev) * 0.02 + 0.005 for _ in range(2)]
    pool = [_store(torch.randn(N, page, Hkv, D, generator=g, device=dev, dtype=torch.float32 if kv == "f32" else torch.bfloat16), kv,
                   scales and scales[i]) for i in range(2)]
    # Queries that attend to some tokens far more than to others: scores of
    # a spread of two.
    qs = (2.0 * torch.randn(B, Hq, D, generator=g, device=dev)).to(DTYPES[q])
    s = dict(q=qs, k_pool=pool[0], v_pool=pool[1], scales=scales, lens=torch.from_numpy(lens.astype(np.int32)).to(dev),
             table=torch.from_numpy(table.astype(np.int32)).to(dev), scale=1.0 / math.sqrt(D), out=torch.zeros_like(qs),
             lse=torch.zeros(B, Hq, dtype=torch.float32, device=dev))
    if own:
        from scriptonait_amd.kv import KVCache

        s["cache"] = KVCache(_handle(), pool[0], pool[1], *(scales or ()))
        s["workspace"] = s["cache"].workspace(Hq)
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(s):
    if s["case"]["op"] == "plan":
        return _own_plan(s) if own else _plain_plan(s)
    if s["case"]["op"] == "append":
        return _own_append(s) if own else _plain_append(s)
    return _own_attend(s) if own else _plain_attend(s)


def _own_plan(s):
    s["pool"].plan(s["lens"], s["table"], s["out_lens"], s["granted"], s["start"], s["slots"], s["positions"],
                   new_tokens=s["new"], release=s["release"], out_free_state=s["out_free"])
    return dict(lens=s["out_lens"], granted=s["granted"], start=s["start"], slots=s["slots"], positions=s["positions"],
                table=s["table"], ring=s["ring"], free=s["out_free"])


def _own_append(s):
    Hq, Hkv = s["case"]["Hq"], s["case"]["Hkv"]
    x = s["qkv"]
    s["cache"].append(x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], s["slots"], q=x[:, :Hq], out_q=s["out_q"], positions=s["positions"],
                      rope=s["rope"])
    return dict(q=s["out_q"], k=s["k_pool"], v=s["v_pool"])


def _own_attend(s):
    s["cache"].attend(s["q"], s["table"], s["lens"], s["out"], s["workspace"], window=s["case"]["window"], scale=s["scale"],
                      out_lse=s["lse"])
    return dict(out=s["out"], lse=s["lse"])


def _plain_plan(s):
    page, T = s["case"]["page"], s["case"]["T"]
    R, table = s["table"].shape
    N = s["ring"].numel()
    lens = s["lens"].long()
    head, free = s["free"].long()
    gone = torch.zeros_like(lens, dtype=torch.bool) if s["release"] is None else s["release"] != 0
    base = torch.where(gone, 0, lens)
    n = (~gone).long() if s["new"] is None else s["new"].long()
    end = torch.cumsum(n, 0)
    start = end - n
    fits = (base + n <= table * page) & (end <= T)
    have = (base + page - 1) // page
    need = torch.where(fits, (base + n + page - 1) // page - have, 0)
    upto = torch.cumsum(need, 0)
    ok = fits & ((need == 0) | (upto <= free))
    took = torch.where(ok, need, 0)
    granted = torch.where(ok, n, 0)
    # Released pages go behind the free ones, in the requests' order.
    p = torch.arange(table, device=lens.device)
    back = torch.where(gone, (lens + page - 1) // page, 0)
    back_end = torch.cumsum(back, 0)
    to = (head + free + (back_end - back)[:, None] + p) % N
    ring = torch.cat([s["ring"], s["ring"].new_zeros(1)])
    ring.scatter_(0, torch.where(p < back[:, None], to, N).reshape(-1), s["table"].reshape(-1))
    # New pages from the front.
    j = p - have[:, None]
    at = (head + (upto - need)[:, None] + j) % N
    s["table"].copy_(torch.where((j >= 0) & (j < took[:, None]), s["ring"][at], s["table"]))
    s["ring"].copy_(ring[:N])
    # Each token's request, position and slot.
    t = torch.arange(T, device=lens.device)
    r = torch.clamp(torch.searchsorted(end, t, right=True), max=R - 1)
    live = (t < end[-1]) & ok[r]
    pos = torch.where(live, base[r] + t - start[r], 0)
    slots = torch.where(live, s["table"][r, pos // page].long() * page + pos % page, -1)
    state = torch.stack([(head + took.sum()) % N, free - took.sum() + back.sum()])
    return dict(lens=(base + granted).int(), granted=granted.int(), start=torch.cat([start.new_zeros(1), end]).int(), slots=slots,
                positions=pos.int(), table=s["table"], ring=s["ring"], free=state.int())


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


def _plain_append(s):
    c = s["case"]
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    x = s["qkv"].float()
    turned = _plain_rotate(x[:, :Hq + Hkv], s["positions"], c["dims"], s["theta"], c["style"])
    # Which token each of the pool's rows takes, if any. A padding token's key
    # and value go nowhere; its query is as any other's.
    rows = s["k_pool"].shape[0] * c["page"]
    t = torch.arange(len(x), device=x.device)
    token = torch.full((rows + 1,), -1, device=x.device).scatter_(0, torch.where(s["slots"] < 0, rows, s["slots"]), t)[:rows]
    for pool, new, scale in ((s["k_pool"], turned[:, Hq:], 0), (s["v_pool"], x[:, Hq + Hkv:], 1)):
        new = _store(new, c["kv"], s["scales"] and s["scales"][scale]).contiguous().view(torch.uint8).view(len(x), -1)
        raw = pool.view(torch.uint8).view(rows, -1)
        raw.copy_(torch.where(token[:, None] >= 0, new[token.clamp(min=0)], raw))
    return dict(q=turned[:, :Hq].to(s["qkv"].dtype), k=s["k_pool"], v=s["v_pool"])


def _plain_attend(s):
    c = s["case"]
    B, Hq, Hkv, D = c["B"], c["Hq"], c["Hkv"], c["D"]
    G = Hq // Hkv
    table = s["table"].long()
    L = table.shape[1] * c["page"]
    q = s["q"].float().view(B, Hkv, G, D)
    t = torch.arange(L, device=q.device)
    lens = s["lens"].long()[:, None]
    seen = t < lens
    if c["window"]:
        seen = seen & (t >= lens - c["window"])

    def rows(pool, scale):  # [B, Hkv, L, D]; what no query may see reads as zero
        x = pool.view(torch.uint8)[table].view(pool.dtype).view(B, L, Hkv, D).transpose(1, 2).float()
        if scale is not None:
            x = x * scale[:, None, None]
        return torch.where(seen[:, None, :, None], x, 0.0)

    scores = torch.matmul(q, rows(s["k_pool"], s["scales"] and s["scales"][0]).transpose(-1, -2)) * s["scale"]
    scores = torch.where(seen[:, None, None], scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e, rows(s["v_pool"], s["scales"] and s["scales"][1])) / torch.where(total == 0, 1.0, total)
    lse = (top + torch.log(total)).view(B, Hq)
    return dict(out=o.view(B, Hq, D).to(s["q"].dtype), lse=lse)


# ---------------------------------------------------------------------------
# What a pass cannot do without, and its outputs from the definitions
# ---------------------------------------------------------------------------
def work(case):
    if case["op"] == "plan":
        _, lens, release, new, _, _ = _plan_host(case, 0)
        page, R, T = case["page"], case["R"], case["T"]
        n = np.where(release == 1, 0, 1) if new is None else new
        pages = int((_pages_for(lens * (1 - release) + n, page) - _pages_for(lens * (1 - release), page)).sum())
        back = int((_pages_for(lens, page) * release).sum())
        # lengths, counts or flags in; lengths, grants and starts out; slots and
        # positions; a free page read and a table entry written
        return {"bytes": 4 * 2 * R + 4 * 3 * R + 12 * T + 8 * (pages + back), "flops": 0}
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    if case["op"] == "append":
        T = case["T"]
        rows = T * D * ((2 * Hq + 2 * Hkv) * BYTES[case["q"]] + 2 * Hkv * BYTES[case["kv"]])
        return {"bytes": rows + 12 * T, "flops": 3 * T * case["dims"] * (Hq + Hkv)}
    lens = _lens(case, 0)
    if case["window"]:
        lens = np.minimum(lens, case["window"])
    tokens = int(lens.sum())
    return {"bytes": 2 * tokens * Hkv * D * BYTES[case["kv"]] + case["B"] * Hq * (2 * D * BYTES[case["q"]] + 4),
            "flops": 4 * tokens * Hq * D}


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "plan":
        return _exact_plan(case, s)
    return _exact_append(case, s) if case["op"] == "append" else _exact_attend(case, s)


def _exact_plan(case, s):
    """The requests one after the other, as a program on the host would serve them."""
    page, T = case["page"], case["T"]
    lens, table, ring = (s[k].cpu().numpy().astype(np.int64) for k in ("lens", "table", "ring"))
    release = np.zeros_like(lens) if s["release"] is None else s["release"].cpu().numpy()
    head, free = s["free"].cpu().tolist()
    N = len(ring)
    before = ring.copy()
    tail, left, taken, asked, stop = head + free, free, 0, 0, False
    slots, positions = np.full(T, -1), np.zeros(T, dtype=np.int64)
    out_lens, granted, start = lens.copy(), np.zeros_like(lens), [0]
    for r in range(len(lens)):
        if release[r]:
            have = -(-lens[r] // page)
            for p in range(have):
                ring[tail % N] = table[r, p]
                tail += 1
            out_lens[r] = 0
        n = int(s["new"][r]) if s["new"] is not None else int(not release[r])
        first = asked
        asked += n
        start.append(asked)
        base = int(out_lens[r])
        if base + n > table.shape[1] * page or asked > T:
            continue
        have, want = -(-base // page), -(-(base + n) // page)
        if want > have and (stop or want - have > left):
            stop = True
            continue
        for p in range(have, want):
            table[r, p] = before[(head + taken) % N]
            taken += 1
            left -= 1
        granted[r], out_lens[r] = n, base + n
        pos = base + np.arange(n)
        positions[first:first + n] = pos
        slots[first:first + n] = table[r, pos // page] * page + pos % page
    state = [(head + taken) % N, tail - head - taken]
    return dict(lens=out_lens, granted=granted, start=np.array(start), slots=slots, positions=positions, table=table, ring=ring,
                free=np.array(state))


def _exact_append(case, s):
    Hq, Hkv, D, dims = case["Hq"], case["Hkv"], case["D"], case["dims"]
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
    pools = []
    for i, (pool, rows) in enumerate(((s["k_pool"], turned[:, Hq:]), (s["v_pool"], x[:, Hq + Hkv:]))):
        p = pool.double().view(-1, Hkv, D).clone()
        if case["kv"] == "e4m3":
            rows = (rows / s["scales"][i].double()[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
        live = s["slots"] >= 0
        p.index_copy_(0, s["slots"][live], rows[live])
        pools.append(p.view(pool.shape))
    return dict(q=turned[:, :Hq], k=pools[0], v=pools[1])


def _exact_attend(case, s):
    """Request by request, over the rows that it may see."""
    Hq, Hkv, D, page = case["Hq"], case["Hkv"], case["D"], case["page"]
    G = Hq // Hkv
    out = torch.zeros(case["B"], Hq, D, dtype=torch.float64, device=s["q"].device)
    lse = torch.full((case["B"], Hq), -math.inf, dtype=torch.float64, device=s["q"].device)
    kb, vb = (p.view(torch.uint8).view(-1, Hkv, D * BYTES[case["kv"]]) for p in (s["k_pool"], s["v_pool"]))
    for b, n in enumerate(s["lens"].cpu().tolist()):
        if n == 0:
            continue
        t = torch.arange(max(0, n - case["window"]) if case["window"] else 0, n, device=out.device)
        slot = s["table"][b].long()[t // page] * page + t % page
        k, v = (x[slot].view(DTYPES[case["kv"]]).double() for x in (kb, vb))
        if s["scales"]:
            k, v = k * s["scales"][0].double()[:, None], v * s["scales"][1].double()[:, None]
        for h in range(Hkv):
            q = s["q"][b, h * G:(h + 1) * G].double()
            x = (q @ k[:, h].t().contiguous()) * s["scale"]
            lse[b, h * G:(h + 1) * G] = torch.logsumexp(x, -1)
            out[b, h * G:(h + 1) * G] = torch.softmax(x, -1) @ v[:, h].contiguous()
    return dict(out=out, lse=lse)
