"""GPU: llmhip_kv_attend against the definition in binary64, with the bounds
that kv_oracle derives from the types."""
import numpy as np
import pytest

import kv_oracle

pytestmark = pytest.mark.gpu

TYPES = dict(f32="float32", bf16="bfloat16", f16="float16", e4m3="float8_e4m3fn")


def _make(seed, lens, Hq, Hkv, D, page, q, kv, layout="plain", spare=2, spread=2.0):
    """Inputs whose every place that no request may see holds NaN or wild page ids."""
    import torch

    rs = np.random.default_rng(seed)
    g = torch.Generator().manual_seed(seed)
    X, P = getattr(torch, TYPES[q]), getattr(torch, TYPES[kv])
    lens = np.asarray(lens)
    B, pages = len(lens), -(-lens // page)
    N = max(1, int(pages.sum())) + 3
    width = max(1, int(pages.max(initial=0))) + spare
    order = rs.permutation(N)
    table = rs.choice([-1, 1 << 30, -(1 << 31), N], (B, width)).astype(np.int64)
    seen = np.zeros((N, page), bool)
    at = 0
    for b in range(B):
        ids = order[at:at + pages[b]]
        at += pages[b]
        table[b, :pages[b]] = ids
        t = np.arange(lens[b])
        seen[ids[t // page] if len(t) else [], t % page] = True
    pools = []
    for i in range(2):
        shape = dict(plain=(N, page, Hkv, D), heads_first=(N, Hkv, page, D))[layout]
        x = torch.randn(shape, generator=g)
        if i == 0 and seed % 2:
            x = x * 3
        x = x if layout == "plain" else x.transpose(1, 2)
        x[torch.from_numpy(~seen)] = float("nan")
        x = x.to(P)
        pools.append(x if layout == "plain" else x.transpose(1, 2).contiguous().transpose(1, 2))
    scales = [torch.rand(Hkv, generator=g) * 0.3 + 0.5 for _ in range(2)] if kv == "e4m3" else [None, None]
    qs = (spread * torch.randn(B, Hq, D, generator=g)).to(X)
    return dict(q=qs, k_pool=pools[0], v_pool=pools[1], k_scale=scales[0], v_scale=scales[1],
                table=torch.from_numpy(table.astype(np.int32)), lens=torch.from_numpy(lens.astype(np.int32)))


def _cuda(x, layout=None):
    import torch

    if x is None:
        return None
    y = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device="cuda")
    if x.element_size() == 1:
        y.view(torch.uint8).copy_(x.view(torch.uint8))
    else:
        y.copy_(x)
    return y


def _attend(sampler, c, window=0, scale=None, want_lse=True, q=None, out=None, stream=None, pool_bytes=0):
    import torch

    from scriptonait_amd.kv import KVCache

    pools = [_cuda(c["k_pool"]), _cuda(c["v_pool"])]
    if pool_bytes:  # more pages behind those that are used
        for i, p in enumerate(pools):
            page = p[0].numel() * p.element_size()
            raw = torch.full((pool_bytes // page + 1, page), 255, dtype=torch.uint8, device="cuda")
            raw[:len(p)] = p.contiguous().view(torch.uint8).reshape(len(p), page)
            pools[i] = raw.view(p.dtype).view(-1, *p.shape[1:])
    cache = KVCache(sampler, *pools, _cuda(c["k_scale"]), _cuda(c["v_scale"]))
    q = _cuda(c["q"]) if q is None else q
    B, Hq, D = q.shape
    out = torch.full((B, Hq, D), 77.0, dtype=q.dtype, device="cuda") if out is None else out
    lse = torch.full((B, Hq), 77.0, device="cuda") if want_lse else None
    ws = cache.workspace(Hq)
    ws.fill_(255)  # whatever it held
    table, lens = _cuda(c["table"]), _cuda(c["lens"])
    torch.cuda.synchronize()
    cache.attend(q, table, lens, out, ws, window=window, scale=scale, out_lse=lse, stream=stream)
    torch.cuda.synchronize()
    return out.double().cpu(), None if lse is None else lse.double().cpu()


def _check(c, got, window=0, scale=None):
    scale = c["q"].shape[2] ** -0.5 if scale is None else scale
    out, lse, out_tol, lse_tol = kv_oracle.attend(c["q"], c["k_pool"], c["v_pool"], c["table"], c["lens"], window, scale,
                                                  c["k_scale"], c["v_scale"])
    assert ((got[0] - out).abs() <= out_tol).all(), float(((got[0] - out).abs() - out_tol).max())
    if got[1] is not None:
        none = lse == -np.inf
        assert (got[1][none] == -np.inf).all()
        assert ((got[1] - lse).abs()[~none] <= lse_tol[~none]).all()


PAIRS = [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "e4m3"), ("f16", "e4m3")]


@pytest.mark.parametrize("q,kv", PAIRS)
@pytest.mark.parametrize("lens,Hq,Hkv,D,page,window,layout", [
    ([1], 1, 1, 64, 16, 0, "plain"),
    ([0, 1, 2, 31, 32, 33, 0], 8, 2, 64, 16, 0, "plain"),
    ([63, 64, 65, 127, 129, 7], 4, 4, 128, 16, 0, "heads_first"),
    ([700], 8, 2, 64, 16, 512, "plain"),
    ([5, 100, 37, 90, 41], 12, 12, 80, 24, 40, "plain"),
    ([333, 1, 258], 16, 1, 128, 64, 0, "plain"),
    ([45, 46, 200], 20, 1, 96, 20, 0, "plain"),
    ([77, 130], 33, 3, 40, 7, 33, "heads_first"),
    ([65, 300], 14, 2, 112, 1, 100, "plain"),
    ([90, 17, 255], 6, 3, 256, 8, 0, "plain"),
    ([64, 10], 6, 2, 192, 128, 0, "heads_first"),
    ([19, 150, 33], 5, 1, 8, 3, 1, "plain"),
    ([100, 77], 4, 2, 16, 32, 0, "plain"),
    ([500, 499], 2, 2, 32, 256, 300, "plain"),
    ([121, 122], 40, 2, 136, 12, 0, "plain"),
    ([4000], 32, 8, 128, 16, 0, "plain"),
    ([2600, 3], 7, 7, 24, 16, 0, "plain")])
def test_attend(sampler, q, kv, lens, Hq, Hkv, D, page, window, layout):
    c = _make(len(lens) + D, lens, Hq, Hkv, D, page, q, kv, layout)
    _check(c, _attend(sampler, c, window), window)
    assert sampler.status().flags == 0


@pytest.mark.parametrize("q,kv", PAIRS)
def test_many_ragged_requests(sampler, q, kv):
    """More requests than a workgroup has threads, most of them short."""
    rs = np.random.default_rng(3)
    lens = rs.integers(0, 60, 700)
    lens[::97] = 900
    c = _make(4, lens, 4, 2, 64, 16, q, kv)
    _check(c, _attend(sampler, c, want_lse=True))
    _check(c, _attend(sampler, c, 50, want_lse=False), 50)


@pytest.mark.parametrize("q,kv", [("f32", "f32"), ("bf16", "bf16"), ("f16", "e4m3")])
@pytest.mark.parametrize("B,Hq,Hkv,D,longest", [(2100, 2, 1, 64, 90), (65, 4, 4, 128, 300), (3, 2100, 2100, 8, 40),
                                                (2, 96, 24, 32, 700)])
def test_batches_and_heads_beyond_one_cut(sampler, q, kv, B, Hq, Hkv, D, longest):
    """More requests than are cut into ranges, than a wave has lanes; more
    heads than workgroups fill the card with, and teams of 8."""
    rs = np.random.default_rng(B)
    c = _make(B, rs.integers(0, longest, B), Hq, Hkv, D, 16, q, kv)
    _check(c, _attend(sampler, c))
    assert sampler.status().flags == 0


@pytest.mark.parametrize("q,kv", PAIRS)
@pytest.mark.parametrize("wide", [False, True])
def test_wide_tables_and_long_requests_beside_short_ones(sampler, q, kv, wide):
    c = _make(6, [20000, 5, 0, 900], 8, 2, 128, 16, q, kv, spare=8000 if wide else 2)
    got = _attend(sampler, c)
    _check(c, got)
    again = _attend(sampler, c)
    assert (got[0] == again[0]).all() and (got[1] == again[1]).all()  # the same bits every time


@pytest.mark.parametrize("q,kv", PAIRS)
def test_views_scale_and_large_scores(sampler, q, kv):
    """Queries out of a packed tensor, an output with gaps, a scale of its own
    whose scores are past what exp takes without its maximum, also falling
    and rising along the cache."""
    import torch

    c = _make(9, [300, 40], 4, 2, 64, 16, q, kv, spread=30.0)
    packed = torch.zeros(2, 9, 64, dtype=c["q"].dtype, device="cuda")
    packed[:, 3:7] = c["q"].cuda()
    gaps = torch.full((2, 4, 80), 5.0, dtype=c["q"].dtype, device="cuda")
    got = _attend(sampler, c, scale=2.0, q=packed[:, 3:7], out=gaps[:, :, :64])
    _check(c, got, scale=2.0)
    assert (gaps[:, :, 64:] == 5).all()
    odd = torch.zeros(2 * 4 * 65 + 1, dtype=c["q"].dtype, device="cuda")[1:].view(2, 4, 65)[:, :, :64]
    odd.copy_(c["q"])
    odd_out = torch.zeros(2 * 4 * 65 + 1, dtype=c["q"].dtype, device="cuda")[1:].view(2, 4, 65)[:, :, :64]
    again = _attend(sampler, c, scale=2.0, q=odd, out=odd_out)
    assert (got[0] == again[0]).all() and (got[1] == again[1]).all()


@pytest.mark.parametrize("q,kv", PAIRS)
@pytest.mark.parametrize("page", [4, 16])
def test_bad_pages_and_lengths_are_left_out(sampler, q, kv, page):
    import torch

    from scriptonait_amd.kv import KSTATUS_BAD_INDEX

    c = _make(12, [200, 64, 90, 16], 4, 2, 64, page, q, kv, spare=0)
    c["table"][0, 1] = -1
    c["table"][1, :] = c["k_pool"].shape[0]  # no page is left
    sampler.status()
    _check(c, _attend(sampler, c))
    assert sampler.status().flags == KSTATUS_BAD_INDEX
    c = _make(13, [208, 64], 4, 2, 64, page, q, kv, spare=0)
    c["lens"] = torch.tensor([2**31 - 1, -3], dtype=torch.int32)
    _check(c, _attend(sampler, c))
    assert sampler.status().flags == KSTATUS_BAD_INDEX


@pytest.mark.parametrize("Hq,spare", [(1, 0), (8, 0), (8, 500)])
@pytest.mark.parametrize("bad", [0, 63, 64, 70, 299])
def test_one_bad_length_among_many_is_flagged(sampler, bad, Hq, spare):
    """Whichever of a workgroup's threads reads it, in ranges and whole."""
    from scriptonait_amd.kv import KSTATUS_BAD_INDEX

    lens = np.arange(300) % 40
    lens[bad] = 0
    c = _make(21, lens, Hq, Hq, 64, 16, "bf16", "bf16", spare=spare)
    _check(c, _attend(sampler, c))
    assert sampler.status().flags == 0
    c["lens"][bad] = -1
    got = _attend(sampler, c)
    assert sampler.status().flags == KSTATUS_BAD_INDEX
    c["lens"][bad] = 0
    _check(c, got)


def test_infinite_scores(sampler):
    """Keys of -inf drop their token, all of them leave a row of zeros."""
    import torch

    for q, kv in [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16")]:
        c = _make(14, [70, 40], 2, 1, 64, 16, q, kv)
        c["q"] = c["q"].abs() + 0.1
        c["k_pool"][c["table"][0, 0].item(), 3] = float("-inf")
        c["k_pool"][c["table"][1, :3].long()] = float("-inf")
        out, lse = _attend(sampler, c)
        assert (out[1] == 0).all() and (lse[1] == -np.inf).all()
        keep = torch.tensor([t for t in range(70) if t != 3])
        ids = c["table"][0].long()[keep // 16]
        k, v = c["k_pool"][ids, keep % 16, 0].double(), c["v_pool"][ids, keep % 16, 0].double()
        p = torch.softmax(c["q"][0].double() @ k.T / 8, -1)
        assert torch.allclose(out[0], p @ v, rtol=0, atol=0.02)


def test_caches_past_32_bits(sampler):
    """Pools of more than 2^32 bytes and 2^31 values: pages at their ends."""
    import torch

    from scriptonait_amd.kv import KVCache

    D, H, page = 128, 8, 64
    N = (2**31 + 2**27) // (D * H * page)
    pools = [torch.empty(N, page, H, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    ids = torch.tensor([[N - 1, 0, N - 2, N // 2]], dtype=torch.int32)
    g = torch.Generator().manual_seed(1)
    small = [torch.randn(4, page, H, D, generator=g).bfloat16() for _ in range(2)]
    for p, s in zip(pools, small):
        p[ids[0].long().cuda()] = s.cuda()
    q = torch.randn(1, 2 * H, D, generator=g).bfloat16()
    cache = KVCache(sampler, *pools)
    out, lse = torch.zeros_like(q, device="cuda"), torch.zeros(1, 2 * H, device="cuda")
    lens = torch.tensor([4 * page - 5], dtype=torch.int32)
    cache.attend(q.cuda(), ids.cuda(), lens.cuda(), out, cache.workspace(2 * H), out_lse=lse)
    c = dict(q=q, k_pool=small[0], v_pool=small[1], k_scale=None, v_scale=None, table=torch.arange(4, dtype=torch.int32)[None],
             lens=lens)
    _check(c, (out.double().cpu(), lse.double().cpu()))
    # And slots there.
    x = torch.randn(2, H, D, generator=g).bfloat16().cuda()
    cache.append(x, -x, torch.tensor([N * page - 1, N * page - page], device="cuda"))
    assert torch.equal(pools[0][N - 1, [page - 1, 0]], x) and torch.equal(pools[1][N - 1, [page - 1, 0]], -x)
    del pools, cache
    torch.cuda.empty_cache()


@pytest.mark.parametrize("q,kv", PAIRS)
@pytest.mark.parametrize("D,page", [(64, 16), (80, 16), (128, 8), (256, 32), (192, 64), (128, 20)])
def test_large_pools(sampler, q, kv, D, page):
    """Pools that no cache of the card holds: their values are read another way."""
    c = _make(D + page, [300, 0, 77, 33], 8, 4, D, page, q, kv)
    got = _attend(sampler, c, 200, pool_bytes=80 << 20)
    _check(c, got, 200)
    small = _attend(sampler, c, 200)
    assert (got[0] == small[0]).all() and (got[1] == small[1]).all()


def test_no_request_and_empty_table(sampler):
    import torch

    from scriptonait_amd.kv import KVCache

    cache = KVCache(sampler, *[torch.zeros(2, 16, 1, 64, device="cuda") for _ in range(2)])
    ws = cache.workspace(1)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    cache.attend(torch.zeros(0, 1, 64, device="cuda"), i(0, 3), i(0), torch.zeros(0, 1, 64, device="cuda"), ws)
    out, lse = torch.ones(2, 1, 64, device="cuda"), torch.ones(2, 1, device="cuda")
    cache.attend(torch.ones(2, 1, 64, device="cuda"), i(2, 0), i(2), out, ws, out_lse=lse)
    assert (out == 0).all() and (lse == -np.inf).all()


def test_other_stream(sampler):
    import torch

    c = _make(15, [500, 20], 8, 2, 64, 16, "bf16", "bf16")
    _check(c, _attend(sampler, c, stream=torch.cuda.Stream()))
