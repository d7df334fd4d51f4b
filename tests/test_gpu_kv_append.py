"""GPU: llmhip_kv_append against the rotation in binary64, with the bounds
that kv_oracle derives; rows that no token goes to keep every bit."""
import numpy as np
import pytest

import kv_oracle

pytestmark = pytest.mark.gpu


def _dtypes(q, kv):
    import torch

    names = dict(f32=torch.float32, bf16=torch.bfloat16, f16=torch.float16, e4m3=torch.float8_e4m3fn)
    return names[q], names[kv]


def _pool(kind, N, page, Hkv, D, dtype, g):
    """Two pools [N, page, Hkv, D] of one of the layouts that strides allow."""
    import torch

    n = dict(plain=2, heads_first=2, interleaved=1)[kind]
    shape = dict(plain=(N, page, Hkv, D), heads_first=(N, Hkv, page, D), interleaved=(N, page, Hkv, 2, D))[kind]
    raw = [torch.randn(shape, generator=g).clamp(-400, 400).to(dtype).cuda() for _ in range(n)]
    if kind == "plain":
        return raw
    if kind == "heads_first":
        return [r.transpose(1, 2) for r in raw]
    return [raw[0][:, :, :, i] for i in range(2)]


def _bytes(t):
    import torch

    return t.contiguous().view(torch.uint8)


@pytest.mark.parametrize("q,kv", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "e4m3"), ("f16", "e4m3"),
                                  ("f32", "e4m3")])
@pytest.mark.parametrize("T,Hq,Hkv,D,page,dims,style,layout,packed", [
    (1, 8, 2, 64, 16, 64, "neighbours", "plain", True), (1, 1, 1, 8, 1, 8, "halves", "plain", False),
    (3, 4, 4, 80, 24, 40, "halves", "heads_first", True), (17, 5, 1, 128, 20, 128, "halves", "plain", False),
    (64, 7, 7, 112, 16, 56, "neighbours", "interleaved", True), (33, 6, 2, 96, 64, 96, "halves", "interleaved", False),
    (100, 32, 8, 128, 16, 128, "halves", "plain", True), (257, 3, 3, 256, 8, 254, "neighbours", "heads_first", False),
    (50, 10, 5, 24, 5, 10, "halves", "plain", True), (41, 0, 3, 192, 32, 96, "halves", "plain", False),
    (41, 2, 1, 40, 7, 0, "halves", "plain", True)])
def test_append(sampler, q, kv, T, Hq, Hkv, D, page, dims, style, layout, packed):
    import torch

    from scriptonait_amd.kv import KVCache, Rope

    X, P = _dtypes(q, kv)
    g = torch.Generator().manual_seed(T * 1000 + D)
    rs = np.random.default_rng(T)
    N = T // page + 3
    pools = _pool(layout, N, page, Hkv, D, P, g)
    scales = [(torch.rand(Hkv, generator=g) * 0.02 + 0.005).cuda() for _ in range(2)] if kv == "e4m3" else []
    x = torch.randn(T, Hq + 2 * Hkv, D + 8, generator=g).to(X)
    x[0, -1, 0] = 1e4 if X != torch.float16 else 6e4  # past an 8-bit cache's range
    x = x.cuda()
    if packed:
        x = x[:, :, :D]
        parts = x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]
    else:
        parts = [t.contiguous() for t in (x[:, :Hq, :D], x[:, Hq:Hq + Hkv, :D], x[:, Hq + Hkv:, :D])]
    slots = rs.permutation(N * page)[:T]
    slots[rs.random(T) < 0.1] = -1
    slots_d = torch.from_numpy(slots).cuda()
    positions = torch.from_numpy(rs.integers(0, 1 << 30 if T > 50 else 5000, T).astype(np.int32))
    rope = Rope(dims, 10000.0, style) if dims else None
    before = [_bytes(p).cpu() for p in pools]
    cache = KVCache(sampler, *pools, *scales)
    out_q = torch.full((T, Hq, D), 7.0, dtype=X, device="cuda") if Hq else None
    cache.append(parts[1], parts[2], slots_d, q=parts[0] if Hq else None, out_q=out_q, positions=positions.cuda(), rope=rope)
    torch.cuda.synchronize()
    assert sampler.status().flags == 0
    freqs = rope.freqs if rope else ()
    host = [p.double().cpu() for p in parts]
    live = slots >= 0
    if Hq:
        want = kv_oracle.rotate(host[0], positions, freqs, style)
        tol = kv_oracle.rotate_bound(host[0], freqs, style) * 1.01 + kv_oracle.HALF_STEP[X] * want.abs() + 2.0**-25
        assert ((out_q.double().cpu() - want).abs() <= tol).all()
    for i, (pool, was) in enumerate(zip(pools, before)):
        want = kv_oracle.rotate(host[1], positions, freqs, style) if i == 0 else host[2]
        tol = kv_oracle.rotate_bound(host[1], freqs, style) * 1.01 if i == 0 else torch.zeros_like(want)
        got = pool.double().cpu().reshape(N * page, Hkv, D)[slots[live]]
        want, tol = want[live], tol[live]
        if kv == "e4m3":
            s = scales[i].double().cpu()[:, None]
            # One division; the smallest steps are 2^-9, half of that at most off.
            want, tol = (want / s).clamp(-448, 448), tol / s + kv_oracle.F32 * (want / s).abs()
            tol = tol + torch.maximum(kv_oracle.HALF_STEP[P] * (want.abs() + tol), torch.tensor(2.0**-10, dtype=torch.float64))
        else:
            tol = tol + kv_oracle.HALF_STEP[P] * want.abs() * 1.01 + (2.0**-25 if kv == "f16" else 0.0)
            if i == 1:
                assert (got == host[2][live]).all()  # values are moved as they are
        assert ((got - want).abs() <= tol).all()
        rest = np.ones(N * page, bool)
        rest[slots[live]] = False
        now = _bytes(pool).cpu().reshape(N * page, -1)
        assert torch.equal(now[torch.from_numpy(rest)], was.reshape(N * page, -1)[torch.from_numpy(rest)])


@pytest.mark.parametrize("style", ["halves", "neighbours"])
@pytest.mark.parametrize("q,kv", [("f32", "f32"), ("bf16", "bf16"), ("f16", "e4m3")])
def test_rows_of_any_alignment(sampler, q, kv, style):
    """Operands that start at an odd value give the bits that aligned ones give."""
    import torch

    from scriptonait_amd.kv import KVCache, Rope

    X, P = _dtypes(q, kv)
    T, H, D = 19, 3, 40
    g = torch.Generator().manual_seed(8)
    scales = [torch.full((H,), 0.25, device="cuda") for _ in range(2)] if kv == "e4m3" else []
    x = torch.randn(T, 3 * H, D + 1, generator=g).to(X).cuda()
    odd = [x[:, i * H:(i + 1) * H, 1:] for i in range(3)]
    slots, pos = torch.arange(T, device="cuda"), torch.arange(T, dtype=torch.int32, device="cuda") * 37
    results = []
    for parts, out in [(odd, torch.zeros(T, H, D + 1, dtype=X, device="cuda")[:, :, 1:]),
                       ([p.contiguous() for p in odd], torch.zeros(T, H, D, dtype=X, device="cuda"))]:
        pools = [torch.zeros(2, 16, H, D, device="cuda").to(P) for _ in range(2)]
        KVCache(sampler, *pools, *scales).append(parts[1], parts[2], slots, q=parts[0], out_q=out, positions=pos,
                                                 rope=Rope(D, 10000.0, style))
        results.append([_bytes(t) for t in (out, *pools)])
    assert all(torch.equal(a, b) for a, b in zip(*results)) and int(results[0][0].count_nonzero()) > 0
    assert sampler.status().flags == 0


def test_in_place_queries_nan_and_bad_slots(sampler):
    import torch

    from scriptonait_amd.kv import KSTATUS_BAD_INDEX, KVCache, Rope

    T, H, D = 6, 2, 64
    g = torch.Generator().manual_seed(5)
    q = torch.randn(T, H, D, generator=g).cuda()
    k, v = torch.randn(T, H, D, generator=g).cuda(), torch.randn(T, H, D, generator=g).cuda()
    v[0, 0, 3] = float("nan")
    pools = [torch.zeros(4, 4, H, D, device="cuda") for _ in range(2)]
    cache = KVCache(sampler, *pools)
    pos = torch.arange(T, dtype=torch.int32, device="cuda") * 100
    slots = torch.tensor([0, 16, 1 << 40, -1, -(1 << 60), 15], device="cuda")
    out = torch.empty_like(q)
    sampler.status()
    cache.append(k, v, slots, q=q, out_q=out, positions=pos, rope=Rope(D))
    assert sampler.status().flags == KSTATUS_BAD_INDEX
    assert torch.isnan(pools[1][0, 0, 0, 3]) and int(torch.isnan(pools[1]).sum()) == 1
    used = torch.zeros(16, dtype=torch.bool)
    used[[0, 15]] = True
    assert torch.equal((pools[0].reshape(16, -1) != 0).any(1).cpu(), used)
    cache.append(k, v, slots.clamp(max=-1), q=q, out_q=q, positions=pos, rope=Rope(D))
    assert torch.equal(q, out) and sampler.status().flags == 0
    e4m3 = [torch.zeros(4, 4, H, D, device="cuda").to(torch.float8_e4m3fn) for _ in range(2)]
    KVCache(sampler, *e4m3, torch.ones(H, device="cuda"), torch.ones(H, device="cuda")).append(k, v, slots.clamp(max=15))
    assert torch.isnan(e4m3[1].float()[0, 0, 0, 3]) and not torch.isnan(e4m3[0].float()).any()


def test_far_positions_are_exact(sampler):
    """Angles near 2^31 radians: binary32 would be off by a hundred turns."""
    import torch

    from scriptonait_amd.kv import KVCache, Rope

    T, D = 64, 128
    x = torch.ones(T, 1, D, device="cuda")
    pos = torch.arange(2**31 - T, 2**31, dtype=torch.int64).int()
    pools = [torch.zeros(1, T, 1, D, device="cuda") for _ in range(2)]
    rope = Rope(D, 50000.0)
    KVCache(sampler, *pools).append(x, x, torch.arange(T, device="cuda"), positions=pos.cuda(), rope=rope)
    host = x.double().cpu()
    want = kv_oracle.rotate(host, pos, rope.freqs, "halves")
    # The oracle's own angle is rounded in 64 bits: 2^31 * 2^-53.
    tol = kv_oracle.rotate_bound(host, rope.freqs, "halves") + kv_oracle.F32 * want.abs() + 2 * 2.0**-22
    assert ((pools[0][0].double().cpu() - want).abs() <= tol).all()


def test_no_token(sampler):
    import torch

    from scriptonait_amd.kv import KVCache

    pools = [torch.zeros(1, 4, 1, 64, device="cuda") for _ in range(2)]
    e = torch.zeros(0, 1, 64, device="cuda")
    KVCache(sampler, *pools).append(e, e, torch.zeros(0, dtype=torch.int64, device="cuda"))
    torch.cuda.synchronize()
