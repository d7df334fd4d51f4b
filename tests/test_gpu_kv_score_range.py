"""GPU: attention scores far from 0, up to those that binary32 does not hold."""
import numpy as np
import pytest

import kv_oracle
from test_gpu_kv_attend import _attend, _make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q,kv,size", [("f32", "f32", s) for s in (16, 22, 26, 30, 34, 60, 120)]
                         + [("bf16", "bf16", s) for s in (22, 26, 30, 34, 120)]
                         + [("f16", "f16", s) for s in (18, 22, 24, 26, 28, 30)] + [("f16", "e4m3", s) for s in (20, 22)]
                         + [("bf16", "e4m3", s) for s in (22, 40, 100)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("n,B", [(40, 16), (3000, 16), (700, 300)])
def test_large_scores(sampler, q, kv, size, sign, n, B):
    """Scores of 2^size / 8 and thereabouts, all exact, with gaps of a 32nd of
    them: the tokens that share the largest one share the weight."""
    import torch

    D, H, page = 16, 2, 16
    c = _make(40, [n], H, H, D, page, q, kv, spare=0)
    k_bits = dict(f16=15, e4m3=8).get(kv, size // 2)
    steps = torch.arange(n) % 7 / (8 if kv == "e4m3" else 32)
    t = torch.arange(n)
    ids = c["table"][0].long()[t // page]

    def rows(pool):
        raw = pool.view(torch.uint8) if kv == "e4m3" else pool
        return raw[ids, t % page].view(pool.dtype).double()

    keys = (2.0**k_bits * (1 + steps)).to(c["k_pool"].dtype)
    if kv == "e4m3":
        c["k_pool"].view(torch.uint8)[ids, t % page, :, 0] = keys.view(torch.uint8)[:, None]
        c["k_scale"], c["v_scale"] = torch.ones(H), torch.ones(H)
    else:
        c["k_pool"][ids, t % page, :, 0] = keys[:, None]
    # All requests read the same pages; their queries differ.
    c["table"], c["lens"] = c["table"].expand(B, -1).contiguous(), c["lens"].expand(B).contiguous()
    first = sign * 2.0 ** (size - k_bits) * (1 + torch.arange(B) % 13 / 64)
    c["q"] = torch.zeros(B, H, D, dtype=c["q"].dtype)
    c["q"][..., 0] = first[:, None]
    got = _attend(sampler, c, scale=0.125)
    k, v = rows(c["k_pool"])[:, 0, 0], rows(c["v_pool"])
    for b in range(B):
        s = k * c["q"][b, 0, 0].double() * 0.125
        top = s == s.max()
        assert n < 7 or float((s.max() - s[~top]).min()) > 200  # the others have no weight
        want = v[top].mean(0)
        rel = 2 * (8 + n) * kv_oracle.F32 + 2.0**-16
        tol = rel * v[top].abs().mean(0) + kv_oracle.HALF_STEP[c["q"].dtype] * want.abs() * 1.01 + 2.0**-24
        assert ((got[0][b] - want).abs() <= tol).all(), b
        lse = float(s.max()) + np.log(int(top.sum()))
        assert ((got[1][b] - lse).abs() <= 2.0**-20 * abs(lse)).all(), b


@pytest.mark.parametrize("B,n", [(1, 1), (1, 40), (2, 3000), (1, 200)])
def test_scores_past_binary32_give_nan(sampler, B, n):
    """A score that binary32 does not hold is no weight of 0, whichever part
    of its request it is in."""
    import torch

    D = 64
    c = _make(33, [n] * B, 2, 1, D, 16, "f32", "f32")
    c["q"] = torch.zeros_like(c["q"])
    c["q"][..., 0] = 1e19
    live = ~c["k_pool"][..., 0].isnan()
    c["k_pool"][..., 0][live] = 1e15
    id, at = int(c["table"][0, n // 2 // 16]), n // 2 % 16
    c["k_pool"][id, at, 0, 0] = 3e19  # 3e38, times log2(e) past the largest number
    got = _attend(sampler, c, scale=1.0)
    assert got[0][0].isnan().all() and got[1][0].isnan().all()
    assert got[0][1:].isfinite().all() and got[1][1:].isfinite().all()
