"""GPU: attention where one token outweighs all others together, so that the
many small weights are the answer. A weight of 2^-25 is the size of half of
float16's smallest step: a type that holds the weights themselves, with the
largest one at 1, loses them or doubles them."""
import pytest

import kv_oracle
from test_gpu_kv_attend import TYPES, _attend

pytestmark = pytest.mark.gpu

# Queries and keys that every type holds exactly: 16 times 1 and times these
# are 17.375, 17, 16.5 and 20 nats apart.
BELOW = [-0.0859375, -0.0625, -0.03125, -0.25]


def _make(q, kv, B, tokens, H, D, below, first):
    """B equal requests over the same pages: token 0 has the value `first` and
    the largest score by far."""
    import torch

    X, P = getattr(torch, TYPES[q]), getattr(torch, TYPES[kv])
    g = torch.Generator().manual_seed(tokens + D)
    page = 64
    N = -(-tokens // page)
    k, v = torch.zeros(N, page, H, D), torch.rand(N, page, H, D, generator=g) * 0.5 + 0.5
    k[..., 0] = below
    k[0, 0, :, 0] = 1.0
    v[0, 0] = first
    qs = torch.zeros(B, H, D)
    qs[..., 0] = 16.0
    ones = [torch.ones(H) if kv == "e4m3" else None for _ in range(2)]
    return dict(q=qs.to(X), k_pool=k.to(P), v_pool=v.to(P), k_scale=ones[0], v_scale=ones[1],
                table=torch.arange(N, dtype=torch.int32).expand(B, N).contiguous(),
                lens=torch.full((B,), tokens, dtype=torch.int32))


def _check(sampler, c):
    one = {k: x[:1] if k in ("q", "table", "lens") else x for k, x in c.items()}
    out, lse, out_tol, lse_tol = kv_oracle.attend(one["q"], one["k_pool"], one["v_pool"], one["table"], one["lens"], 0, 1.0,
                                                  one["k_scale"], one["v_scale"])
    got = _attend(sampler, c, scale=1.0)
    over = float(((got[0] - out).abs() / out_tol).max())
    assert over <= 1.0, (over, got[0][0, 0, :4].tolist(), out[0, 0, :4].tolist())
    assert ((got[1] - lse).abs() <= lse_tol).all()


@pytest.mark.parametrize("q,kv", [("f16", "f16"), ("f16", "e4m3"), ("bf16", "bf16"), ("bf16", "e4m3")])
@pytest.mark.parametrize("below", BELOW)
@pytest.mark.parametrize("first", [0.0, 1.0])
@pytest.mark.parametrize("B,H,tokens", [(256, 8, 8192), (1, 1, 8192), (3, 2, 500)])
def test_small_weights_keep_their_bits(sampler, q, kv, below, first, B, H, tokens):
    """Requests that one wave reads, that many share, and that a workgroup
    reads whole; the first token's value is nothing, or like the others."""
    _check(sampler, _make(q, kv, B, tokens, H, 64, below, first))


@pytest.mark.parametrize("q,kv", [("f16", "f16"), ("f16", "e4m3")])
def test_small_weights_of_a_long_context(sampler, q, kv):
    _check(sampler, _make(q, kv, 256, 131072, 8, 16, BELOW[0], 0.0))
