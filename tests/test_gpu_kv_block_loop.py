"""GPU: the 8-bit cache's operators together: in the decode loop of
examples/paged_decode.py, with draft tokens that are taken back, recorded into
a graph, on two streams at once, and far into a large pool."""
import sys
from pathlib import Path

import numpy as np
import pytest

import kv_block_oracle
import kv_oracle
from test_gpu_kv_block_append import make_pools, same, to_cuda, to_host

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))

pytestmark = pytest.mark.gpu

STEPS = (0, 1, 15, 16, 33, 47, 48, 49, 64, 69)


def test_calls_of_a_decode_loop(sampler, monkeypatch):
    """Each append and attend on what it was really given."""
    import paged_decode
    import torch

    from scriptonait_amd.kv_blocks import BlockKVCache

    at = dict(step=0, calls=0)
    append, attend = BlockKVCache.append, BlockKVCache.attend

    def checked_append(self, k, v, slots, q=None, out_q=None, positions=None, rope=None, stream=None):
        if at["step"] not in STEPS:
            return append(self, k, v, slots, q, out_q, positions, rope, stream)
        before = [to_host(x) for x in (self.k_pool, self.v_pool, self.k_scale, self.v_scale)]
        host = [t.double().cpu() for t in (q, k)]
        append(self, k, v, slots, q, out_q, positions, rope, stream)
        pos, where = positions.cpu(), slots.tolist()
        want = kv_oracle.rotate(host[0], pos, rope.freqs, rope.style)
        tol = kv_oracle.rotate_bound(host[0], rope.freqs, rope.style) * 1.01 + kv_oracle.HALF_STEP[q.dtype] * want.abs() + 2.0**-25
        assert ((out_q.double().cpu() - want).abs() <= tol).all()
        pool, scale = kv_block_oracle.write(before[1], before[3], v.float().cpu(), where)
        same(to_host(self.v_pool), pool)
        same(to_host(self.v_scale), scale)
        want = kv_oracle.rotate(host[1], pos, rope.freqs, rope.style)
        err = kv_oracle.rotate_bound(host[1], rope.freqs, rope.style) * 1.01
        got = kv_block_oracle.values(to_host(self.k_pool), to_host(self.k_scale)).flatten(0, 1)
        for t, slot in enumerate(where):
            if slot >= 0:
                s = self.k_scale[slot // self.page_size, slot % self.page_size // self.block_size].double().cpu()
                tol = kv_block_oracle.half_step(want[t], s[:, None], torch.int8) + err[t] * 1.1
                assert ((got[slot] - want[t]).abs() <= tol).all()
        at["calls"] += 1

    def checked_attend(self, q, table, lens, out, workspace, window=0, scale=None, out_lse=None, stream=None):
        attend(self, q, table, lens, out, workspace, window, scale, out_lse, stream)
        if at["step"] not in STEPS:
            return
        state = [to_host(x) for x in (self.k_pool, self.v_pool, self.k_scale, self.v_scale)]
        want, _, tol, _ = kv_block_oracle.attend(q.cpu()[:, None], state[:2], state[2:], table.cpu(), lens.cpu(), window,
                                                 self.head_dim**-0.5)
        assert ((out.double().cpu() - want[:, 0]).abs() <= tol[:, 0]).all()
        at["calls"] += 1

    monkeypatch.setattr(BlockKVCache, "append", checked_append)
    monkeypatch.setattr(BlockKVCache, "attend", checked_attend)
    steps = 70
    prompts = [([1, 2, 3], steps), ([10, 11, 12, 13, 14], 33), ([7], steps), ([5, 6], 49)]
    out, m = paged_decode.generate(sampler, prompts, steps, dtype="i8", on_step=lambda t, h: at.update(step=t + 1))
    assert at["calls"] == 2 * 2 * len(STEPS)
    assert [len(o) for o in out] == [steps, 33, steps, 49]
    assert int(m.pool.free_state[1]) == m.pool.pages - 2 * 5


class Loop:
    """Requests that add `new` tokens a step, of which some are taken back."""

    def __init__(self, sampler, B, new, Hq, H, D, page, block, P, kv="i8", q="bfloat16"):
        import torch

        from scriptonait_amd.kv import PagePool, Rope
        from scriptonait_amd.kv_blocks import BlockKVCache

        dev, X = torch.device("cuda:0"), getattr(torch, q)
        i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)  # noqa: E731
        self.B, self.new, self.Hq, self.H = B, new, Hq, H
        self.lens, self.granted, self.start, self.table = i32(B), i32(B), i32(B + 1), i32(B, P)
        self.want, self.slots, self.pos = i32(B) + new, torch.zeros(B * new, dtype=torch.int64, device=dev), i32(B * new)
        self.x = torch.zeros(B * new, Hq + 2 * H, D, dtype=X, device=dev)
        self.q, self.out = (torch.zeros(B, new, Hq, D, dtype=X, device=dev) for _ in range(2))
        self.lse = torch.zeros(B, new, Hq, device=dev)
        self.k, self.v = (torch.zeros(B * new, H, D, dtype=X, device=dev) for _ in range(2))
        self.pool, self.rope = PagePool(sampler, B * P, page), Rope(D)
        codes = torch.int8 if kv == "i8" else torch.float8_e4m3fn
        self.cache = BlockKVCache(sampler, *[torch.zeros(B * P, page, H, D, device=dev).to(codes) for _ in range(2)],
                                  *[torch.full((B * P, page // block, H), float("nan"), device=dev) for _ in range(2)])
        self.ws = self.cache.workspace(Hq, new)

    def step(self, stream=None):
        Hq, H, x = self.Hq, self.H, self.x
        self.pool.plan(self.lens, self.table, self.lens, self.granted, self.start, self.slots, self.pos, new_tokens=self.want,
                       stream=stream)
        self.cache.append(x[:, Hq:Hq + H], x[:, Hq + H:], self.slots, q=x[:, :Hq], out_q=self.q.view(-1, Hq, x.shape[-1]),
                          positions=self.pos, rope=self.rope, stream=stream)
        self.cache.attend(self.q, self.table, self.lens, self.out, self.ws, window=60, out_lse=self.lse, stream=stream)
        self.cache.read(self.slots, self.k, self.v, stream=stream)

    NAMES = ("lens", "table", "slots", "pos", "q", "out", "lse", "k", "v")


@pytest.mark.parametrize("kv", ["i8", "e4m3"])
def test_draft_tokens_that_are_taken_back(sampler, kv):
    """Three draft tokens a step, none to three of which stay: the next step
    writes over the others, in the middle of their blocks."""
    import torch

    rs, g = np.random.RandomState(0), torch.Generator().manual_seed(0)
    m = Loop(sampler, 9, 3, 8, 2, 64, 16, 8, 5, kv)
    for n in range(20):
        before = [to_host(t) for t in (m.cache.v_pool, m.cache.v_scale)]
        x = torch.randn(27, 12, 64, generator=g).bfloat16()
        m.x.copy_(x)
        m.step()
        torch.cuda.synchronize()
        assert (m.granted == 3).all()
        pool, scale = kv_block_oracle.write(*before, x[:, 10:].float(), m.slots.tolist())
        same(to_host(m.cache.v_pool), pool)
        seen = ~torch.isnan(scale)
        same(to_host(m.cache.v_scale)[seen], scale[seen])
        # What the draft tokens read back as is what attention saw.
        want = kv_block_oracle.values(pool, scale).flatten(0, 1)[m.slots.cpu()].float().bfloat16()
        assert torch.equal(m.v.cpu(), want)
        state = [to_host(t) for t in (m.cache.k_pool, m.cache.v_pool, m.cache.k_scale, m.cache.v_scale)]
        out, lse, out_tol, lse_tol = kv_block_oracle.attend(m.q.cpu(), state[:2], state[2:], m.table.cpu(), m.lens.cpu(), 60, 0.125)
        assert ((m.out.double().cpu() - out).abs() <= out_tol).all()
        assert ((m.lse.double().cpu() - lse).abs() <= lse_tol).all()
        m.lens -= torch.from_numpy(rs.randint(0, 4, 9)).int().cuda()
    assert sampler.status().flags == 0


@pytest.mark.parametrize("new,block", [(1, 16), (3, 8), (2, 1)])
def test_a_step_in_a_graph(sampler, new, block):
    """Recorded once and replayed, with the program's own work between the
    replays: every step equals the eager one."""
    import torch

    g = torch.Generator().manual_seed(1)
    eager, played = (Loop(sampler, 70, new, 8, 2, 64, 16, block, 8) for _ in range(2))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        played.step()
    steps = 40
    for n in range(steps):
        x = torch.randn(eager.x.shape, generator=g).bfloat16()
        for m in (eager, played):
            m.x.copy_(x)
        eager.step()
        graph.replay()
        if n % 7 == 0:
            torch.cuda.synchronize()
            torch.ones(1000, device="cuda").sum().item()
        for k in Loop.NAMES:
            assert torch.equal(getattr(eager, k), getattr(played, k)), (n, k)
    for k in ("k_pool", "v_pool", "k_scale", "v_scale"):
        a, b = (to_host(getattr(m.cache, k)) for m in (eager, played))
        if a.is_floating_point():
            a, b = a.nan_to_num(-1.0), b.nan_to_num(-1.0)
        assert torch.equal(a, b)
    assert eager.lens.tolist() == [steps * new] * 70 and sampler.status().flags == 0


def test_two_streams_at_once(sampler):
    """Two loops on streams of their own, with workspaces of their own."""
    import torch

    g = torch.Generator().manual_seed(2)
    alone, one, two = (Loop(sampler, 33, 2, 8, 2, 128, 16, 16, 4) for _ in range(3))
    xs = [torch.randn(alone.x.shape, generator=g).bfloat16().cuda() for _ in range(25)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for x in xs:
        for m, s in ((one, streams[0]), (two, streams[1])):
            with torch.cuda.stream(s):
                m.x.copy_(x)
                m.step()
    for x in xs:
        alone.x.copy_(x)
        alone.step()
    torch.cuda.synchronize()
    for k in Loop.NAMES:
        for m in (one, two):
            assert torch.equal(getattr(alone, k), getattr(m, k)), k


@pytest.mark.parametrize("kv", ["i8", "e4m3"])
def test_offsets_past_32_bits(sampler, kv):
    """The last pages of a pool of 4.6 GB: the same as those of a small one."""
    import torch

    from scriptonait_amd.kv_blocks import BlockKVCache

    N, few, page, H, D, block = 70000, 8, 64, 8, 128, 32
    g = torch.Generator().manual_seed(3)
    pools, scales = make_pools(g, few, page, H, D, block, kv)
    codes = torch.int8 if kv == "i8" else torch.float8_e4m3fn
    small = [to_cuda(x) for x in (*pools, *scales)]
    large = [torch.zeros(N, page, H, D, dtype=torch.uint8, device="cuda").view(codes) for _ in range(2)]
    large += [torch.zeros(N, page // block, H, device="cuda") for _ in range(2)]
    for a, b in zip(large, small):
        kv_block_oracle.raw(a)[-few:].copy_(kv_block_oracle.raw(b))
    q = torch.randn(2, 2, 16, D, generator=g).bfloat16().cuda()
    x = torch.randn(100, 2 * H, D, generator=g).bfloat16().cuda()
    lens = torch.tensor([250, 190], dtype=torch.int32, device="cuda")
    got = []
    for state, far in ((small, 0), (large, N - few)):
        cache = BlockKVCache(sampler, *state)
        slots = torch.arange(60, 160, device="cuda") + far * page
        table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4) + far
        out, rows = torch.zeros_like(q), torch.zeros(100, H, D, device="cuda")
        ws = cache.workspace(16, 2)
        cache.append(x[:, :H], x[:, H:], slots)
        cache.attend(q, table, lens, out, ws)
        cache.read(slots, rows)
        torch.cuda.synchronize()
        got.append([out.cpu(), rows.cpu(), *[to_host(kv_block_oracle.raw(t)[-few:]) for t in state]])
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert (kv_block_oracle.raw(large[0])[:-few] == 0).all() and sampler.status().flags == 0
