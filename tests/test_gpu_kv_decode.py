"""GPU: the paged cache's operators together, in the decode loop of
examples/paged_decode.py, and a step of them recorded into a graph."""
import sys
from pathlib import Path

import pytest

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))

pytestmark = pytest.mark.gpu


def _dense(m, tokens, t):
    """Hidden state after tokens[: t + 1] of one request, without a cache:
    all positions at once in binary64, the weights as they are."""
    import torch

    n = t + 1
    x = m.embed[tokens[:n].long()].double()
    H, K, D = m.heads, m.kv_heads, m.dim
    norm = lambda y: y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-5)  # noqa: E731
    half = D // 2
    angle = torch.arange(n, device=x.device).double()[:, None, None] * torch.tensor(m.rope.freqs, device=x.device, dtype=torch.float64)
    c, s = torch.cos(angle), torch.sin(angle)
    turn = lambda y: torch.cat([y[..., :half] * c - y[..., half:] * s, y[..., half:] * c + y[..., :half] * s], -1)  # noqa: E731
    i = torch.arange(n, device=x.device)
    seen = (i[None] <= i[:, None]) & (i[None] > i[:, None] - m.window)
    for w in m.layers:
        w = {k: v.double() for k, v in w.items()}
        rows = (norm(x) @ w["qkv"]).view(n, -1, D)
        q, k, v = turn(rows[:, :H]), turn(rows[:, H:H + K]), rows[:, H + K:]
        k, v = k.repeat_interleave(H // K, 1), v.repeat_interleave(H // K, 1)
        o = torch.empty_like(q)
        for h in range(H):
            sc = q[:, h] @ k[:, h].t().contiguous() * D**-0.5
            o[:, h] = torch.softmax(sc.masked_fill(~seen, float("-inf")), -1) @ v[:, h].contiguous()
        x = x + o.reshape(n, -1) @ w["o"]
        y = norm(x)
        x = x + (torch.nn.functional.silu(y @ w["gate"]) * (y @ w["up"])) @ w["down"]
    return norm(x)[-1]


# A hidden state is normalized to 1. Through 2 layers of about 8 roundings
# each, of at most half a step of the type relative to values of a few units,
# its error stays below 50 half steps; an 8-bit cache's own half step, 2^-4 of
# keys and values, comes in through averages over tokens and scores.
@pytest.mark.parametrize("dtype,tol", [("f32", 50 * 2.0**-20), ("f16", 50 * 2.0**-11), ("bf16", 50 * 2.0**-8), ("e4m3", 0.8)])
def test_decode_loop_equals_the_dense_model(sampler, dtype, tol):
    import paged_decode
    import torch

    steps = 70
    prompts = [([1, 2, 3], steps), ([10, 11, 12, 13, 14], 33), ([7], steps), ([5, 6], 49)]
    kept = []
    out, m = paged_decode.generate(sampler, prompts, steps, dtype=dtype, on_step=lambda t, h: kept.append(h.clone()))
    assert [len(o) for o in out] == [steps, 33, steps, 49]
    for t in (0, 16, 32, 48, 69):
        for b, o in enumerate(out):
            if t < len(o):
                want = _dense(m, torch.tensor(o, device="cuda"), t)
                err = float((kept[t][b].double() - want).abs().max())
                assert err <= tol, (t, b, err)
    again, _ = paged_decode.generate(sampler, prompts, steps, dtype=dtype)
    assert again == out
    # Two ended and gave their pages back; the others hold 70 tokens each.
    assert int(m.pool.free_state[1]) == m.pool.pages - 2 * 5
    held = set(m.table[0, :5].tolist()) | set(m.table[2, :5].tolist())
    head, free = m.pool.free_state.tolist()
    ring = m.pool.free_ring.tolist()
    assert held | {ring[(head + i) % m.pool.pages] for i in range(free)} == set(range(m.pool.pages))


def test_pages_run_out_and_come_back(sampler):
    """More requests than the pool can hold: the refused tokens get no slot,
    and a released request's pages serve the next call."""
    import torch

    from scriptonait_amd.kv import PagePool

    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    pool = PagePool(sampler, 3, 4)
    lens, granted, start, table = i32(4), i32(4), i32(5), i32(4, 2)
    slots, pos = torch.zeros(4, dtype=torch.int64, device="cuda"), i32(4)
    pool.plan(lens, table, lens, granted, start, slots, pos)
    assert granted.tolist() == [1, 1, 1, 0] and slots.tolist()[3] == -1 and pool.free_state.tolist()[1] == 0
    gone = torch.tensor([0, 1, 0, 0], dtype=torch.int32, device="cuda")
    pool.plan(lens, table, lens, granted, start, slots, pos, release=gone)
    assert lens.tolist() == [2, 0, 2, 0] and granted.tolist() == [1, 0, 1, 0] and pool.free_state.tolist()[1] == 1
    pool.plan(lens, table, lens, granted, start, slots, pos, new_tokens=torch.tensor([1, 0, 1, 1], dtype=torch.int32, device="cuda"))
    assert lens.tolist() == [3, 0, 3, 1] and sampler.status().flags == 0


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
def test_a_step_in_a_graph(sampler, kv):
    """plan, append and attend recorded once and replayed, with the program's
    own work between the replays: every step equals the eager one."""
    import torch

    from scriptonait_amd.kv import KVCache, PagePool, Rope

    dev, B, Hq, Hkv, D, page, P = torch.device("cuda:0"), 70, 8, 2, 64, 16, 6
    g = torch.Generator().manual_seed(0)
    cached = torch.bfloat16 if kv == "bf16" else torch.float8_e4m3fn
    rope = Rope(D)

    def state():
        i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)  # noqa: E731
        s = dict(lens=i32(B), table=i32(B, P), granted=i32(B), start=i32(B + 1), slots=torch.zeros(B, dtype=torch.int64, device=dev),
                 pos=i32(B), x=torch.zeros(B, Hq + 2 * Hkv, D, dtype=torch.bfloat16, device=dev), lse=torch.zeros(B, Hq, device=dev))
        s["q"] = torch.zeros(B, Hq, D, dtype=torch.bfloat16, device=dev)
        s["out"] = torch.zeros_like(s["q"])
        s["pool"] = PagePool(sampler, B * P, page)
        scales = [torch.full((Hkv,), 0.01, device=dev) for _ in range(2)] if kv == "e4m3" else []
        s["cache"] = KVCache(sampler, *[torch.zeros(B * P, page, Hkv, D, device=dev).to(cached) for _ in range(2)], *scales)
        s["ws"] = s["cache"].workspace(Hq)
        return s

    def step(s):
        s["pool"].plan(s["lens"], s["table"], s["lens"], s["granted"], s["start"], s["slots"], s["pos"])
        x = s["x"]
        s["cache"].append(x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], s["slots"], q=x[:, :Hq], out_q=s["q"], positions=s["pos"], rope=rope)
        s["cache"].attend(s["q"], s["table"], s["lens"], s["out"], s["ws"], window=40, out_lse=s["lse"])

    eager, played = state(), state()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(played)
    for n in range(60):
        x = torch.randn(B, Hq + 2 * Hkv, D, generator=g).bfloat16()
        for s in (eager, played):
            s["x"].copy_(x)
        step(eager)
        graph.replay()
        if n % 7 == 0:
            torch.cuda.synchronize()
            torch.ones(1000, device=dev).sum().item()
        for k in ("lens", "table", "slots", "pos", "q", "out", "lse"):
            assert torch.equal(eager[k], played[k]), (n, k)
    assert eager["lens"].tolist() == [60] * B and sampler.status().flags == 0
