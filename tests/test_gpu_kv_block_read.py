"""GPU: llmhip_kv_block_read: each code times its scale, rounded once."""
import numpy as np
import pytest

import kv_block_oracle
from test_gpu_kv_block_append import Q, make_pools, to_cuda

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["i8", "e4m3"])
@pytest.mark.parametrize("q", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,H,D,page,block,layout", [
    (1, 1, 8, 1, 1, "tokens"), (700, 2, 64, 16, 16, "tokens"), (33, 12, 80, 24, 8, "heads"), (100, 3, 256, 20, 4, "tokens"),
    (65, 1, 16, 7, 7, "heads"), (2, 40, 128, 256, 256, "tokens"), (5000, 1, 8, 64, 2, "tokens"), (129, 8, 128, 12, 12, "heads")])
def test_read(sampler, q, kv, T, H, D, page, block, layout):
    import torch

    from scriptonait_amd.kv_blocks import BlockKVCache

    g, rs = torch.Generator().manual_seed(T), np.random.RandomState(T)
    N = T // page // 2 + 2
    pools, scales = make_pools(g, N, page, H, D, block, kv, layout)
    cache = BlockKVCache(sampler, *[to_cuda(x) for x in (*pools, *scales)])
    slots = rs.randint(-2, N * page, T)  # any order, some of them twice, some padding
    X = getattr(torch, Q[q])
    on = torch.from_numpy(slots).cuda()
    wide = torch.full((T, 2 * H + 1, D + 3), 55.0, dtype=X, device="cuda")
    out = [wide[:, :H, 1:1 + D], wide[:, H:2 * H, 1:1 + D]]
    cache.read(on, *out)
    only = [torch.full((T, H, D), 55.0, dtype=X, device="cuda") for _ in range(2)]
    cache.read(on, out_k=only[0])
    cache.read(on, out_v=only[1])
    torch.cuda.synchronize()
    for i in range(2):
        x = kv_block_oracle.values(pools[i], scales[i]).flatten(0, 1)
        # The product of a code of 8 bits and a binary32 scale is exact in
        # binary64: rounded to binary32 and then to the rows' type.
        want = torch.where(torch.from_numpy(slots >= 0)[:, None, None], x[torch.from_numpy(slots.clip(0))], 0.0).float().to(X)
        assert torch.equal(out[i].cpu(), want) and torch.equal(only[i].cpu(), want)
        out[i].fill_(55.0)
    assert (wide == 55.0).all()
    assert sampler.status().flags == 0


def test_slots_past_the_pool_give_zeros_and_are_flagged(sampler):
    import torch

    from scriptonait_amd.kv_blocks import BlockKVCache

    pools, scales = make_pools(torch.Generator().manual_seed(1), 2, 16, 2, 32, 8, "e4m3")
    cache = BlockKVCache(sampler, *[to_cuda(x) for x in (*pools, *scales)])
    out = torch.full((3, 2, 32), 9.0, device="cuda")
    cache.read(torch.tensor([5, 32, 1 << 50], device="cuda"), out_v=out)
    torch.cuda.synchronize()
    assert sampler.status().flags == 2
    assert torch.equal(out[0].cpu().double(), kv_block_oracle.values(pools[1], scales[1])[0, 5].float().double())
    assert (out[1:] == 0).all()
