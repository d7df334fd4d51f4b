"""GPU: infinite values in attention. A value that a request sees with a
weight above 0 decides its column alone, however the request is cut over waves
and workgroups: infinity gives infinity, both signs and NaN give NaN."""
import pytest

import kv_oracle
from test_gpu_kv_attend import _attend, _make

pytestmark = pytest.mark.gpu

TYPES = [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16")]
INF = float("inf")


def _place(c, b, t):
    page = c["k_pool"].shape[1]
    return int(c["table"][b, t // page]), t % page


def _want(c, b):
    """Request b's output by its definition in binary64, infinities and all."""
    import torch

    B, Hq, D = c["q"].shape
    page, Hkv = c["k_pool"].shape[1:3]
    t = torch.arange(int(c["lens"][b]))
    ids = c["table"][b].long()[t // page]
    k, v = (c[x][ids, t % page].double() for x in ("k_pool", "v_pool"))
    out = torch.zeros(Hq, D, dtype=torch.float64)
    for h in range(Hq):
        p = torch.softmax(k[:, h * Hkv // Hq] @ c["q"][b, h].double() * D**-0.5, 0)
        assert (p > 0).all()
        out[h] = (p[:, None] * v[:, h * Hkv // Hq]).sum(0)
    return out


def _check(c, got):
    import torch

    out, _, tol, _ = kv_oracle.attend(c["q"], c["k_pool"], c["v_pool"], c["table"], c["lens"], 0, c["q"].shape[2] ** -0.5)
    for b in range(len(c["lens"])):
        want = _want(c, b)
        finite = want.isfinite()
        assert torch.equal(got[0][b].isnan(), want.isnan()), b
        inf = want.isinf()
        assert torch.equal(got[0][b][inf], want[inf]), b
        assert ((got[0][b] - out[b]).abs() <= tol[b])[finite].all(), b


@pytest.mark.parametrize("q,kv", TYPES)
@pytest.mark.parametrize("lens,Hq,Hkv,D,page,spare", [
    ([1], 1, 1, 64, 16, 2),           # a single token, whose weight is 1
    ([40, 3, 70], 8, 2, 64, 16, 0),   # parts of several waves, joined in LDS
    ([33, 100], 16, 8, 128, 16, 0),   # a wave for each head
    ([3000, 40], 8, 2, 64, 16, 0),    # parts of several workgroups
    ([900, 5, 77, 300], 4, 4, 128, 20, 4000),
    ([2000], 20, 1, 80, 16, 0), ([700, 40], 6, 3, 256, 8, 0), ([50, 900], 2, 2, 24, 7, 0)])
def test_infinite_values(sampler, q, kv, lens, Hq, Hkv, D, page, spare):
    c = _make(30 + D + len(lens), lens, Hq, Hkv, D, page, q, kv, spare=spare)
    v = c["v_pool"]
    for b, n in enumerate(lens):
        last = _place(c, b, n - 1)
        v[last[0], last[1], :, 3] = INF
        v[last[0], last[1], :, D - 1] = -INF
        mid = _place(c, b, n // 2)
        v[mid[0], mid[1], :, 3] = INF
        first = _place(c, b, 0)
        v[first[0], first[1], :, 5] = INF
        v[last[0], last[1], :, 5] = -INF if n > 1 else INF
        v[first[0], first[1], 0, 7] = float("nan")
    _check(c, _attend(sampler, c))
    assert sampler.status().flags == 0


@pytest.mark.parametrize("q,kv", TYPES)
@pytest.mark.parametrize("below", [4.0, 18.0, 25.0, 40.0])
def test_infinite_values_of_small_weights(sampler, q, kv, below):
    """A token `below` nats under the largest score, of a weight that binary32
    still has, with an infinite value."""
    import torch

    D, n = 64, 300
    c = _make(31, [n, n], 2, 1, D, 16, q, kv)
    c["q"] = torch.zeros_like(c["q"])
    c["q"][..., 0] = 8.0
    for b in range(2):
        for t in range(n):
            id, at = _place(c, b, t)
            c["k_pool"][id, at, :, 0] = below if t == 100 else 0.0  # scores of `below` and 0
        id, at = _place(c, b, 250)
        c["v_pool"][id, at, 0, 9] = INF
        c["v_pool"][id, at, 0, 10] = -INF
    got = _attend(sampler, c)
    assert (got[0][:, :, 9] == INF).all() and (got[0][:, :, 10] == -INF).all()
    _check(c, got)


@pytest.mark.parametrize("q,kv", TYPES)
def test_one_requests_infinity_stays_its_own(sampler, q, kv):
    import torch

    c = _make(32, [500, 90, 40, 700], 8, 4, 64, 16, q, kv)
    clean = _attend(sampler, c)
    id, at = _place(c, 1, 60)
    c["v_pool"][id, at, 2, 11] = INF
    got = _attend(sampler, c)
    hit = torch.zeros_like(got[0], dtype=torch.bool)
    hit[1, 4:6, 11] = True
    assert (got[0][hit] == INF).all()
    assert torch.equal(got[0][~hit], clean[0][~hit]) and torch.equal(got[1], clean[1])
