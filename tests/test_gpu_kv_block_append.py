"""GPU: llmhip_kv_block_append against the rule of its blocks: bit for bit where
no rotation comes before the codes, within half a step where one does."""
import numpy as np
import pytest

import kv_block_oracle
import kv_oracle

pytestmark = pytest.mark.gpu

Q = dict(f32="float32", bf16="bfloat16", f16="float16")
KV = dict(i8="int8", e4m3="float8_e4m3fn")


def to_cuda(x):
    import torch

    y = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device="cuda")
    kv_block_oracle.raw(y).copy_(kv_block_oracle.raw(x))
    return y


def to_host(x):
    return kv_block_oracle.raw(x).cpu().view(x.dtype)


def make_pools(g, N, page, H, D, block, kv, layout="tokens"):
    """Codes and scales of a cache that was written before; its views are laid
    out with tokens or heads before."""
    import torch

    P = getattr(torch, KV[kv])
    pools, scales = [], []
    for _ in range(2):
        x = torch.randint(-127, 128, (N, page, H, D), generator=g).float()
        x = x.to(P) if kv == "i8" else (x * 3.5).to(P)
        s = torch.rand(N, page // block, H, generator=g) * 0.02 + 0.001
        if layout == "heads":
            x = kv_block_oracle.raw(x).transpose(1, 2).contiguous().transpose(1, 2).view(P)
            s = s.transpose(1, 2).contiguous().transpose(1, 2)
        pools.append(x)
        scales.append(s)
    return pools, scales


def make_slots(rs, lens, page, N):
    """Slots of several requests' new tokens (first position, tokens), as a plan
    gives them, with padding behind each."""
    order, at, slots, positions = rs.permutation(N), 0, [], []
    for first, n in lens:
        pages = (first % page + n + page - 1) // page
        for i in range(n):
            place = first % page + i
            slots.append(int(order[at + place // page]) * page + place % page)
            positions.append(first + i)
        at += pages
        slots.append(-1)
        positions.append(0)
    assert at <= N
    return np.array(slots), np.array(positions)


def run_append(sampler, pools, scales, k, v, slots, q=None, positions=None, rope=None, stream=None, out_q=None):
    import torch

    from scriptonait_amd.kv_blocks import BlockKVCache

    state = [to_cuda(x) for x in (*pools, *scales)]
    cache = BlockKVCache(sampler, *state)
    out = None
    if q is not None:
        out = torch.full(q.shape, 77.0, dtype=q.dtype, device="cuda") if out_q is None else out_q
    cache.append(k, v, torch.from_numpy(slots).long().cuda(), q=q, out_q=out,
                 positions=None if positions is None else torch.from_numpy(positions).int().cuda(), rope=rope, stream=stream)
    torch.cuda.synchronize()
    return [to_host(x) for x in state], None if out is None else out.cpu()


def same(a, b):
    import torch

    a, b = kv_block_oracle.raw(a), kv_block_oracle.raw(b)
    if a.is_floating_point():
        a, b = a.view(torch.int32), b.view(torch.int32)
    assert torch.equal(a, b), int((a != b).sum())


LAYOUTS = [
    ([(0, 1)], 8, 2, 64, 16, 16, "tokens"),
    ([(5, 1), (0, 1), (31, 1), (16, 1), (46, 1)], 8, 2, 64, 32, 16, "tokens"),
    ([(0, 100), (7, 33), (64, 1)], 4, 4, 128, 16, 16, "heads"),
    ([(3, 70)], 12, 12, 80, 24, 8, "tokens"),
    ([(0, 40), (19, 41)], 5, 1, 96, 20, 4, "tokens"),
    ([(2, 30), (1, 9)], 20, 1, 256, 64, 64, "heads"),
    ([(0, 300), (100, 77)], 6, 3, 112, 256, 256, "tokens"),
    ([(1, 200)], 2, 1, 256, 128, 128, "tokens"),
    ([(4, 9), (0, 3)], 33, 11, 40, 7, 7, "tokens"),
    ([(4, 9), (6, 23)], 9, 9, 8, 7, 1, "heads"),
    ([(10, 64), (33, 2)], 16, 16, 16, 12, 2, "tokens"),
    ([(i, 1) for i in range(40)], 8, 8, 128, 16, 1, "tokens"),
    ([(0, 150), (40, 260), (0, 1700)], 3, 1, 32, 64, 32, "tokens"),
]


@pytest.mark.parametrize("kv", ["i8", "e4m3"])
@pytest.mark.parametrize("q", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lens,Hq,H,D,page,block,layout", LAYOUTS)
def test_codes_and_scales_without_a_rotation(sampler, q, kv, lens, Hq, H, D, page, block, layout):
    import torch

    g, rs = torch.Generator().manual_seed(D + page), np.random.RandomState(page + len(lens))
    N = sum((f % page + n) // page + 1 for f, n in lens) + 3
    pools, scales = make_pools(g, N, page, H, D, block, kv, layout)
    slots, _ = make_slots(rs, lens, page, N)
    x = (torch.randn(len(slots), Hq + 2 * H, D, generator=g) * (0.2 + 4 * torch.rand(len(slots), 1, 1, generator=g))).to(getattr(torch, Q[q]))
    on = x.cuda()
    got, out_q = run_append(sampler, pools, scales, on[:, Hq:Hq + H], on[:, Hq + H:], slots, q=on[:, :Hq])
    same(out_q, x[:, :Hq])
    for i in range(2):
        new = x[:, Hq + i * H:Hq + (i + 1) * H].float()
        pool, scale = kv_block_oracle.write(pools[i], scales[i], new, slots.tolist())
        same(got[2 + i], scale)
        same(got[i], pool)
    assert sampler.status().flags == 0


@pytest.mark.parametrize("style", ["halves", "neighbours"])
@pytest.mark.parametrize("q,kv", [("f32", "i8"), ("bf16", "i8"), ("f16", "e4m3"), ("f32", "e4m3")])
@pytest.mark.parametrize("lens,Hq,H,D,dims,page,block", [
    ([(0, 1)], 8, 2, 64, 64, 16, 16),
    ([(1000005, 1), (0, 1), (31, 1)], 4, 2, 128, 64, 16, 8),
    ([(0, 100), (70, 33)], 12, 12, 80, 80, 16, 16),
    ([(3, 140)], 2, 1, 256, 256, 64, 64),
    ([(9, 33)], 3, 9, 40, 36, 11, 11),
    ([(5, 20)], 6, 2, 24, 6, 4, 4),
    ([(0, 513)], 1, 1, 16, 16, 256, 128),
    ([(5, 2500)], 2, 33, 64, 64, 32, 16),
    ([(0, 300), (17, 270)], 1, 2, 256, 128, 256, 256),
])
def test_rotated_keys_and_queries(sampler, q, kv, style, lens, Hq, H, D, dims, page, block):
    import torch

    from scriptonait_amd.kv import Rope

    g, rs = torch.Generator().manual_seed(D), np.random.RandomState(D)
    N = sum((f % page + n) // page + 1 for f, n in lens) + 2
    pools, scales = make_pools(g, N, page, H, D, block, kv)
    slots, pos = make_slots(rs, lens, page, N)
    T, X = len(slots), getattr(torch, Q[q])
    q_rows, k, v = ((3 * torch.randn(T, h, D, generator=g)).to(X) for h in (Hq, H, H))
    rope = Rope(dims, 10000.0, style)
    got, out_q = run_append(sampler, pools, scales, k.cuda(), v.cuda(), slots, q=q_rows.cuda(), positions=pos, rope=rope)
    positions = torch.from_numpy(pos)
    want = kv_oracle.rotate(q_rows.double(), positions, rope.freqs, style)
    err = kv_oracle.rotate_bound(q_rows.double(), rope.freqs, style) * 1.01
    assert ((out_q.double() - want).abs() <= err + kv_oracle.HALF_STEP[X] * want.abs() + 2.0**-25).all()

    same(got[1], kv_block_oracle.write(pools[1], scales[1], v.float(), slots.tolist())[0])
    want = kv_oracle.rotate(k.double(), positions, rope.freqs, style)
    err = kv_oracle.rotate_bound(k.double(), rope.freqs, style) * 1.01
    got_values, old_values = kv_block_oracle.values(got[0], got[2]), kv_block_oracle.values(pools[0], scales[0])
    untouched = torch.ones(N, page, dtype=torch.bool)
    kind, most = pools[0].dtype, float(kv_block_oracle.MOST[pools[0].dtype])
    for t, n in kv_block_oracle.runs(slots.tolist(), block):
        p, at = divmod(int(slots[t]), page)
        b, place = divmod(at, block)
        s = got[2][p, b].double()
        top = want[t:t + n].abs().amax((0, 2)) / most
        if place:
            top = torch.maximum(top, scales[0][p, b].double())
        assert ((s - top).abs() <= err[t:t + n].amax((0, 2)) / most + 2 * kv_oracle.F32 * top).all()
        new = got_values[p, at:at + n]
        tol = kv_block_oracle.half_step(want[t:t + n], s[:, None], kind) + err[t:t + n] * 1.1
        assert ((new - want[t:t + n]).abs() <= tol).all()
        old, kept = old_values[p, b * block:at], got_values[p, b * block:at]
        grown = (s > scales[0][p, b].double())[:, None]
        tol = torch.where(grown, kv_block_oracle.half_step(old, s[:, None], kind), 0.0)
        assert ((kept - old).abs() <= tol).all()
        untouched[p, b * block:at + n] = False
    same(got[0].contiguous()[untouched], pools[0].contiguous()[untouched])


@pytest.mark.parametrize("kv", ["i8", "e4m3"])
def test_a_block_filled_token_by_token(sampler, kv):
    """Each token raises some heads' scales and not others'; then the block is
    begun again, and its scales fall."""
    import torch

    g = torch.Generator().manual_seed(3)
    pools, scales = make_pools(g, 3, 16, 3, 32, 8, kv)
    for step in range(24):
        x = torch.randn(1, 6, 32, generator=g) * (1.5**(step % 16) if step % 3 else 0.3)
        slots = np.array([16 + step % 16])
        on = x.cuda()
        got, _ = run_append(sampler, pools, scales, on[:, :3], on[:, 3:], slots)
        for i in range(2):
            pools[i], scales[i] = kv_block_oracle.write(pools[i], scales[i], x[:, 3 * i:3 * i + 3], slots.tolist())
            same(got[i], pools[i])
            same(got[2 + i], scales[i])


@pytest.mark.parametrize("kv", ["i8", "e4m3"])
def test_values_that_have_no_code(sampler, kv):
    """Infinities, NaN, zeros and the smallest numbers; scales that no call has
    written are not looked at where a block begins."""
    import torch

    g = torch.Generator().manual_seed(4)
    pools, scales = make_pools(g, 8, 8, 1, 16, 4, kv)
    for s in scales:
        s[...] = float("nan")
    inf, nan = float("inf"), float("nan")
    x = torch.randn(32, 2, 16, generator=g)
    x[0:4] = 0.0
    x[4, :, 3], x[5, :, 4] = inf, -inf
    x[8, :, 0] = nan
    x[12:16] = nan
    x[16:20] = 1e-37
    x[20:24] = 0.0
    x[20, :, 1] = inf
    x[24:28] *= 1e37
    x[28:32] *= 2.0**-118
    slots = np.arange(8, 40)
    on = x.cuda()
    got, _ = run_append(sampler, pools, scales, on[:, :1], on[:, 1:], slots)
    for i in range(2):
        pool, scale = kv_block_oracle.write(pools[i], scales[i], x[:, i:i + 1], slots.tolist())
        same(got[2 + i], scale)
        if kv == "e4m3":  # (NaN's sign is not fixed)
            nans = torch.isnan(pool.float())
            assert torch.equal(nans, torch.isnan(got[i].float())) and nans.any()
            same(kv_block_oracle.raw(got[i])[~nans], kv_block_oracle.raw(pool)[~nans])
        else:
            same(got[i], pool)


def test_slots_past_the_pool_are_flagged_and_skipped(sampler):
    import torch

    g = torch.Generator().manual_seed(5)
    pools, scales = make_pools(g, 2, 16, 2, 64, 16, "i8")
    k, v = (torch.randn(5, 2, 64, generator=g) for _ in range(2))
    slots = np.array([3, 32, 1 << 40, -1, 20])
    assert sampler.status().flags == 0
    got, _ = run_append(sampler, pools, scales, k.cuda(), v.cuda(), slots)
    assert sampler.status().flags == 2
    for i, x in enumerate((k, v)):
        pool, scale = kv_block_oracle.write(pools[i], scales[i], x, slots.tolist())
        same(got[i], pool)
        same(got[2 + i], scale)


def test_rows_of_any_place_and_a_query_in_place(sampler):
    """Operands that start at odd places of wider rows, out_q that is q, another
    stream; no tokens at all."""
    import torch

    from scriptonait_amd.kv import Rope

    g = torch.Generator().manual_seed(6)
    pools, scales = make_pools(g, 4, 16, 2, 64, 16, "i8")
    x = torch.randn(20, 7, 3 + 64 + 2, generator=g).to(torch.bfloat16)
    on = x.cuda()[:, :, 3:67]
    slots, pos = make_slots(np.random.RandomState(1), [(0, 15), (7, 3)], 16, 4)
    rope = Rope(64)
    plain = x[:, :, 3:67].contiguous().cuda()
    want, want_q = run_append(sampler, pools, scales, plain[:, 3:5], plain[:, 5:], slots, q=plain[:, :3], positions=pos, rope=rope)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    got, got_q = run_append(sampler, pools, scales, on[:, 3:5], on[:, 5:], slots, q=on[:, :3], positions=pos, rope=rope, stream=stream,
                            out_q=on[:, :3])
    same(got_q.contiguous(), want_q)
    for a, b in zip(got, want):
        same(a, b)
    empty = torch.zeros(0, 2, 64, device="cuda")
    got, _ = run_append(sampler, pools, scales, empty, empty, np.zeros(0, np.int64))
    for a, b in zip(got, (*pools, *scales)):
        same(a, b)


@pytest.mark.parametrize("kv", ["i8", "e4m3"])
def test_more_heads_and_tokens_than_workgroups(sampler, kv):
    """Workgroups that take several heads of several blocks, one after the other."""
    import torch

    g = torch.Generator().manual_seed(9)
    T, H, D, page, block = 3000, 41, 32, 32, 16
    pools, scales = make_pools(g, 100, page, H, D, block, kv)
    slots, _ = make_slots(np.random.RandomState(9), [(5, 1700), (0, 1), (40, 1296)], page, 100)
    x = torch.randn(len(slots), 2 * H, D, generator=g).to(torch.bfloat16)
    on = x.cuda()
    got, _ = run_append(sampler, pools, scales, on[:, :H], on[:, H:], slots)
    for i in range(2):
        pool, scale = kv_block_oracle.write(pools[i], scales[i], x[:, i * H:(i + 1) * H].float(), slots.tolist())
        same(got[2 + i], scale)
        same(got[i], pool)
    assert T <= len(slots)


@pytest.mark.parametrize("H", [1, 3, 40])
def test_a_batch_is_its_tokens_one_by_one(sampler, H):
    """Decoding requests far apart in a padded batch, with rotations: what each
    writes does not depend on the others."""
    import torch

    from scriptonait_amd.kv import Rope

    g, rs = torch.Generator().manual_seed(H), np.random.RandomState(H)
    T, D, page, block = 200, 256, 64, 64
    pools, scales = make_pools(g, T, page, H, D, block, "i8")
    slots, pos = np.full(T, -1), rs.randint(0, 1 << 20, T)
    live = [0, 1, 30, 55, 63, 64, 100, 127, 128, 190, 199]
    slots[live] = rs.permutation(T)[:len(live)] * page + rs.randint(0, page, len(live))
    k, v = (torch.randn(T, H, D, generator=g).bfloat16().cuda() for _ in range(2))
    rope = Rope(D)
    whole, _ = run_append(sampler, pools, scales, k, v, slots, positions=pos, rope=rope)
    state = [*pools, *scales]
    for t in live:
        state, _ = run_append(sampler, state[:2], state[2:], k[t:t + 1], v[t:t + 1], slots[t:t + 1], positions=pos[t:t + 1], rope=rope)
    for a, b in zip(whole, state):
        same(a, b)
