"""GPU: values near the largest that attention's binary32 sums can hold. Weights
are below 2^8 before they are divided, so values whose magnitudes sum to less
than 2^119 over a request's tokens leave every partial sum below 2^128."""
import pytest

import kv_block_oracle
import kv_oracle
from test_gpu_kv_block_attend import attend, check, make
from test_gpu_kv_block_append import to_cuda

pytestmark = pytest.mark.gpu

LENS = [64, 1, 33, 500]


@pytest.mark.parametrize("kv", ["i8", "e4m3"])
@pytest.mark.parametrize("new,page,block", [(1, 16, 16), (3, 16, 1), (3, 20, 4)])
def test_blocks(sampler, kv, new, page, block):
    c = make(11, LENS, new, 8, 2, 64, page, block, "bf16", kv)
    c["scales"][1] *= 2.0**108 / 4  # 500 tokens of up to 4 * 2^108 / 4 * 1.2: below 2^119
    values = kv_block_oracle.values(c["pools"][1], c["scales"][1])
    top = values.nan_to_num(0.0).abs().amax()
    assert top * max(LENS) < 2.0**119 and top > 2.0**107
    check(c, attend(sampler, c))


@pytest.mark.parametrize("kind", ["bfloat16", "float32"])
def test_values_as_they_are(sampler, kind):
    import torch

    from scriptonait_amd.kv import KVCache

    X = getattr(torch, kind)
    g = torch.Generator().manual_seed(2)
    pools = [torch.randn(40, 16, 2, 64, generator=g).to(X) for _ in range(2)]
    pools[1] = (pools[1].float() * 2.0**107).to(X)
    assert float(pools[1].float().abs().amax()) * max(LENS) < 2.0**119
    q = torch.randn(4, 8, 64, generator=g).to(X)
    table = torch.randperm(40, generator=g)[:39].int()
    table = torch.stack([torch.roll(table, 3 * b)[:32] for b in range(4)])
    lens = torch.tensor(LENS, dtype=torch.int32)
    cache = KVCache(sampler, *[to_cuda(p) for p in pools])
    out, lse = torch.zeros_like(q, device="cuda"), torch.zeros(4, 8, device="cuda")
    cache.attend(q.cuda(), table.cuda(), lens.cuda(), out, cache.workspace(8), out_lse=lse)
    torch.cuda.synchronize()
    want, _, tol, _ = kv_oracle.attend(q, *pools, table, lens, 0, 0.125)
    assert ((out.double().cpu() - want).abs() <= tol).all()
