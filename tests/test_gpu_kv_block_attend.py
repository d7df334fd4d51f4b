"""GPU: llmhip_kv_block_attend against the definition in binary64, with the
bounds that kv_oracle derives from the types."""
import numpy as np
import pytest

import kv_block_oracle
from test_gpu_kv_block_append import KV, Q, to_cuda

pytestmark = pytest.mark.gpu

PAIRS = [("bf16", "i8"), ("f16", "i8"), ("bf16", "e4m3"), ("f16", "e4m3")]


def make(seed, lens, new, Hq, H, D, page, block, q, kv, layout="tokens", spare=2, spread=2.0):
    """Inputs whose every place that no request may see holds the worst codes,
    scales or page ids."""
    import torch

    rs = np.random.default_rng(seed)
    g = torch.Generator().manual_seed(seed)
    P = getattr(torch, KV[kv])
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
    some = torch.from_numpy(seen.reshape(N, page // block, block).any(2))
    seen = torch.from_numpy(seen)
    pools, scales = [], []
    for i in range(2):
        x = torch.randn(N, page, H, D, generator=g) * (30 if kv == "i8" else 60)
        x = x.round().clamp(-127, 127) if kv == "i8" else x.clamp(-448, 448)
        x[~seen] = -128.0 if kv == "i8" else float("nan")
        s = (torch.rand(N, page // block, H, generator=g) + 0.2) / (30 if kv == "i8" else 60) * (3 if i == 0 and seed % 2 else 1)
        s[~some] = float("nan")
        if layout == "heads":
            x = x.transpose(1, 2).contiguous().transpose(1, 2)
            s = s.transpose(1, 2).contiguous().transpose(1, 2)
        pools.append(x.to(P))
        scales.append(s)
    qs = (spread * torch.randn(B, new, Hq, D, generator=g)).to(getattr(torch, Q[q]))
    return dict(q=qs, pools=pools, scales=scales, table=torch.from_numpy(table.astype(np.int32)),
                lens=torch.from_numpy(lens.astype(np.int32)))


def attend(sampler, c, window=0, scale=None, want_lse=True, q=None, out=None, stream=None, flat=False):
    import torch

    from scriptonait_amd.kv_blocks import BlockKVCache

    cache = BlockKVCache(sampler, *[to_cuda(x) for x in (*c["pools"], *c["scales"])])
    q = to_cuda(c["q"]) if q is None else q
    B, new, Hq, D = q.shape
    out = torch.full(q.shape, 77.0, dtype=q.dtype, device="cuda") if out is None else out
    lse = torch.full((B, new, Hq), 77.0, device="cuda") if want_lse else None
    ws = cache.workspace(Hq, new)
    ws.fill_(255)  # whatever it held
    table, lens = to_cuda(c["table"]), to_cuda(c["lens"])
    args = (q[:, 0], out[:, 0], lse[:, 0] if want_lse else None) if flat else (q, out, lse)
    torch.cuda.synchronize()
    cache.attend(args[0], table, lens, args[1], ws, window=window, scale=scale, out_lse=args[2], stream=stream)
    torch.cuda.synchronize()
    return out.double().cpu(), lse.double().cpu() if want_lse else None


def check(c, got, window=0, scale=None):
    scale = c["q"].shape[-1] ** -0.5 if scale is None else scale
    out, lse, out_tol, lse_tol = kv_block_oracle.attend(c["q"], c["pools"], c["scales"], c["table"], c["lens"], window, scale)
    assert ((got[0] - out).abs() <= out_tol).all(), float(((got[0] - out).abs() - out_tol).max())
    if got[1] is not None:
        none = lse == -np.inf
        assert (got[1][none] == -np.inf).all()
        assert ((got[1] - lse).abs()[~none] <= lse_tol[~none]).all()


@pytest.mark.parametrize("q,kv", PAIRS)
@pytest.mark.parametrize("lens,new,Hq,H,D,page,block,window,layout", [
    ([1], 1, 1, 1, 64, 16, 16, 0, "tokens"),
    ([0, 1, 2, 31, 32, 33, 0], 1, 8, 2, 64, 16, 8, 0, "tokens"),
    ([63, 64, 65, 127, 129, 7], 1, 4, 4, 128, 16, 16, 0, "heads"),
    ([63, 64, 65, 127, 129, 7], 1, 4, 4, 128, 16, 1, 0, "tokens"),
    ([700], 1, 8, 2, 64, 16, 16, 512, "tokens"),
    ([5, 100, 37, 90, 41], 1, 12, 12, 80, 24, 12, 40, "tokens"),
    ([5, 100, 37, 90, 41], 2, 12, 12, 80, 24, 24, 40, "heads"),
    ([333, 1, 258], 1, 16, 1, 128, 64, 64, 0, "tokens"),
    ([45, 46, 200], 3, 20, 1, 96, 20, 4, 0, "tokens"),
    ([77, 130], 1, 33, 3, 40, 7, 7, 33, "heads"),
    ([65, 300], 1, 14, 2, 112, 1, 1, 100, "tokens"),
    ([90, 17, 255], 5, 6, 3, 256, 8, 8, 0, "tokens"),
    ([90, 17, 255], 1, 6, 3, 256, 8, 2, 0, "tokens"),
    ([64, 10], 1, 6, 2, 192, 128, 128, 0, "heads"),
    ([64, 10], 16, 6, 2, 192, 20, 10, 7, "tokens"),
    ([19, 150, 33], 1, 5, 1, 8, 3, 3, 1, "tokens"),
    ([100, 77], 4, 4, 2, 16, 32, 32, 0, "tokens"),
    ([500, 499], 8, 2, 2, 32, 256, 256, 300, "tokens"),
    ([121, 122], 1, 40, 2, 136, 12, 4, 0, "tokens"),
    ([121, 122], 2, 40, 2, 136, 16, 16, 0, "tokens"),
    ([97, 40], 1, 4, 2, 104, 8, 4, 0, "heads"),
    ([4000], 1, 32, 8, 128, 16, 16, 0, "tokens"),
    ([4000, 2000], 4, 32, 8, 128, 16, 1, 0, "tokens"),
    ([2600, 3], 1, 7, 7, 24, 16, 16, 0, "tokens")])
def test_attend(sampler, q, kv, lens, new, Hq, H, D, page, block, window, layout):
    c = make(len(lens) + D, lens, new, Hq, H, D, page, block, q, kv, layout)
    check(c, attend(sampler, c, window, flat=new == 1), window)
    assert sampler.status().flags == 0


@pytest.mark.parametrize("q,kv", PAIRS)
@pytest.mark.parametrize("block", [16, 2])
def test_requests_shorter_than_their_new_tokens(sampler, q, kv, block):
    """Lengths of 0 and below the number of queries: the first of them see nothing."""
    c = make(9, [0, 1, 3, 7, 8, 9, 40, 0], 8, 6, 3, 64, 16, block, q, kv)
    check(c, attend(sampler, c))
    check(c, attend(sampler, c, 2), 2)
    check(c, attend(sampler, c, 1, want_lse=False), 1)


@pytest.mark.parametrize("q,kv", PAIRS)
@pytest.mark.parametrize("new", [1, 3])
def test_many_ragged_requests(sampler, q, kv, new):
    """More requests than a workgroup has threads, most of them short."""
    rs = np.random.default_rng(3)
    lens = rs.integers(0, 60, 700)
    lens[::97] = 900
    c = make(4, lens, new, 4, 2, 64, 16, 8, q, kv)
    check(c, attend(sampler, c))
    check(c, attend(sampler, c, 50, want_lse=False), 50)


@pytest.mark.parametrize("q,kv", PAIRS)
@pytest.mark.parametrize("B,Hq,H,D,longest,new", [(2100, 2, 1, 64, 90, 1), (65, 4, 4, 128, 300, 2), (3, 2100, 2100, 8, 40, 1)])
def test_many_requests_or_heads(sampler, q, kv, B, Hq, H, D, longest, new):
    lens = np.random.default_rng(B).integers(0, longest, B)
    c = make(B, lens, new, Hq, H, D, 16, 16, q, kv)
    check(c, attend(sampler, c))


@pytest.mark.parametrize("kv", ["i8", "e4m3"])
@pytest.mark.parametrize("block", [16, 1])
def test_one_long_request_over_all_ranges(sampler, kv, block):
    c = make(6, [30011], 2, 8, 2, 64, 16, block, "bf16", kv)
    check(c, attend(sampler, c))
    check(c, attend(sampler, c, 29000), 29000)


@pytest.mark.parametrize("kv", ["i8", "e4m3"])
def test_bad_lengths_and_pages_are_flagged(sampler, kv):
    """Tokens on pages outside the pool are left out, lengths are clamped; what
    is there of their scales is not used."""
    c = make(3, [40, 70, 33], 2, 4, 2, 64, 16, 8, "bf16", kv)
    c["table"][1, 2] = -7
    c["table"][2, 0] = 1 << 20
    check(c, attend(sampler, c))
    assert sampler.status().flags == 2
    c = make(3, [48, 70], 2, 4, 2, 64, 16, 8, "bf16", kv, spare=0)
    c["lens"][0] = -5
    assert c["table"].shape[1] == 5
    c["table"][1, 4] = c["table"][1, 0]  # the last page's other tokens are seen once the length is clamped
    c["lens"][1] = 1 << 30
    check(c, attend(sampler, c))
    assert sampler.status().flags == 2


def test_rows_of_any_place_and_another_stream(sampler):
    import torch

    c = make(8, [50, 7, 300], 3, 6, 2, 96, 16, 8, "f16", "i8")
    wide_q = torch.zeros(3, 3, 7, 99, dtype=torch.float16, device="cuda")
    q = wide_q[:, :, 1:, 3:]
    q.copy_(c["q"])
    wide = torch.full((3, 7, 3, 101), 5.0, dtype=torch.float16, device="cuda")  # heads before tokens
    out = wide[:, :6, :, 5:].transpose(1, 2)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    check(c, attend(sampler, c, q=q, out=out, stream=stream))
    out.fill_(5.0)
    assert (wide == 5.0).all()


@pytest.mark.parametrize("block", [16, 1])
def test_scores_far_from_zero(sampler, block):
    """Large queries: the largest scores are in the thousands."""
    c = make(5, [100, 333], 1, 8, 2, 128, 16, block, "bf16", "i8", spread=400.0)
    check(c, attend(sampler, c))
