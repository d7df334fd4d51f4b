"""GPU: codes of an E4M3 cache with block scales that are no numbers: they reach
the queries that see their token, and no others, whatever else a tile holds."""
import numpy as np
import pytest

import kv_block_oracle
from test_gpu_kv_block_attend import attend, make

pytestmark = pytest.mark.gpu


def place(c, kind, head, b, t, columns):
    """Codes of request b's token t and a cache head that become NaN."""
    page = c["pools"][0].shape[1]
    rows = kv_block_oracle.raw(c["pools"][kind])
    rows[int(c["table"][b, t // page]), t % page, head][list(columns)] = 0x7F if t % 2 else 0xFF


def check(c, got, window=0):
    """Every output of a query is NaN where the definition's is, and near it elsewhere."""
    import torch

    D = c["q"].shape[-1]
    out, lse, out_tol, lse_tol = kv_block_oracle.attend(c["q"], c["pools"], c["scales"], c["table"], c["lens"], window, D**-0.5)
    for x, want, tol in ((got[0], out, out_tol), (got[1], lse, lse_tol)):
        nan, none = torch.isnan(want), want == -np.inf
        assert torch.equal(torch.isnan(x), nan), (int(torch.isnan(x).sum()), int(nan.sum()))
        assert (x[none] == -np.inf).all()
        fine = ~nan & ~none
        assert ((x - want).abs()[fine] <= tol[fine]).all()
    return torch.isnan(out)


CASES = [
    ([40], 2, 4, 2, 64, 16, 16, 0),
    ([3, 0, 64, 65], 4, 6, 3, 128, 16, 8, 0),
    ([90, 17, 255, 2], 5, 6, 3, 256, 8, 2, 33),
    ([45, 46, 200], 3, 20, 1, 96, 20, 4, 40),
    ([77, 130], 16, 33, 3, 40, 7, 7, 33),
    ([64, 10], 16, 6, 2, 192, 20, 10, 7),
    ([100, 77], 4, 4, 2, 16, 32, 32, 1),
    ([19, 150, 33], 7, 5, 1, 8, 3, 3, 0),
    ([121, 122], 2, 40, 2, 136, 16, 16, 50),
    ([97, 40], 8, 4, 2, 104, 8, 8, 0),
    ([500, 499], 8, 2, 2, 32, 256, 256, 300),
    ([333, 1, 258], 1, 16, 1, 128, 64, 64, 100),
    ([65, 300], 3, 14, 2, 112, 1, 1, 100),
    ([4000, 2000], 4, 32, 8, 128, 16, 1, 0),
    ([9000], 3, 8, 2, 64, 16, 16, 8500),
    ([2600, 3], 2, 7, 7, 24, 16, 16, 70)]


@pytest.mark.parametrize("q", ["bf16", "f16"])
@pytest.mark.parametrize("lens,new,Hq,H,D,page,block,window", CASES)
def test_values(sampler, q, lens, new, Hq, H, D, page, block, window):
    """In the newest tokens, which the ones before them do not see, in tokens
    that windows leave, and in the middle, each in columns of its own."""
    c = make(len(lens) + D, lens, new, Hq, H, D, page, block, q, "e4m3")
    rs = np.random.default_rng(D + new)
    for b, n in enumerate(lens):
        for i, t in enumerate({n - 1, n - 2, n - new + 1, n - new + 1 - window, n - window, n // 2} & set(range(n))):
            place(c, 1, int(rs.integers(H)), b, t, rs.integers(0, D, 1 + i % 2))
    got = attend(sampler, c, window)
    nan = check(c, got, window)
    assert nan.any() and not nan.all()
    assert sampler.status().flags == 0


@pytest.mark.parametrize("window", [0, 9])
def test_whole_rows_of_the_newest_token(sampler, window):
    """Only the newest token's own queries are NaN, also of requests of which
    the tokens before it see nothing."""
    import torch

    c = make(7, [1, 2, 3, 8, 31, 32, 33, 200], 3, 8, 2, 80, 24, 12, "bf16", "e4m3")
    for b, n in enumerate(c["lens"].tolist()):
        for head in range(2):
            place(c, 1, head, b, n - 1, range(80))
    got = attend(sampler, c, window)
    check(c, got, window)
    assert torch.isnan(got[0][:, 2]).all() and not torch.isnan(got[0][:, :2]).any() and not torch.isnan(got[1]).any()
    assert (got[0][0, :2] == 0).all() and (got[0][1, 0] == 0).all()


@pytest.mark.parametrize("q", ["bf16", "f16"])
def test_keys(sampler, q):
    c = make(5, [50, 300, 4], 4, 8, 2, 128, 16, 8, q, "e4m3")
    for b, t in ((0, 49), (1, 298), (2, 1)):
        place(c, 0, b % 2, b, t, [3 * b])
    nan = check(c, attend(sampler, c, 100), 100)
    assert nan.any() and not nan.all()


def test_draft_tokens_of_which_one_is_no_number(sampler):
    """Through the append: a draft token's values are NaN, the tokens before it
    keep their answers bit for bit."""
    import torch

    from scriptonait_amd.kv_blocks import BlockKVCache

    g = torch.Generator().manual_seed(1)
    page, H, D, new = 16, 2, 64, 4
    k, v = (torch.randn(50, H, D, generator=g).bfloat16().cuda() for _ in range(2))
    q = torch.randn(1, new, 8, D, generator=g).bfloat16().cuda()
    slots = torch.arange(page, page + 50, device="cuda")
    table = torch.arange(1, 5, dtype=torch.int32, device="cuda")[None]
    lens = torch.full((1,), 50, dtype=torch.int32, device="cuda")
    out = {}
    for bad in (False, True):
        cache = BlockKVCache(sampler, *[torch.zeros(6, page, H, D, device="cuda").to(torch.float8_e4m3fn) for _ in range(2)],
                             *[torch.zeros(6, 2, H, device="cuda") for _ in range(2)])
        values = v.clone()
        if bad:  # (in a place that is not the block's largest, so that no scale changes)
            values[48, 1, 5] = float("nan")
        else:
            values[48, 1, 5] = 0.0
        cache.append(k, values, slots)
        out[bad] = torch.zeros_like(q)
        cache.attend(q, table, lens, out[bad], cache.workspace(8, new))
    torch.cuda.synchronize()
    nan = torch.zeros(1, new, 8, D, dtype=torch.bool)
    nan[:, 2:, 4:, 5] = True  # tokens 48 and 49, the second cache head's queries
    assert torch.equal(torch.isnan(out[True]).cpu(), nan)
    assert torch.equal(out[True].cpu()[:, :2], out[False].cpu()[:, :2])
