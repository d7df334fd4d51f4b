"""GPU: blocks whose scale is 0, as nothing in them is a finite number above the
smallest ones: what they are read back as, and what attention makes of them."""
import pytest

import kv_block_oracle
from test_gpu_kv_block_append import KV

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["i8", "e4m3"])
def test_infinite_values_read_back_as_zeros_and_nan_as_what_it_is(sampler, kv):
    import torch

    from scriptonait_amd.kv_blocks import BlockKVCache

    P, inf = getattr(torch, KV[kv]), float("inf")
    cache = BlockKVCache(sampler, *[torch.zeros(3, 8, 1, 16, device="cuda").to(P) for _ in range(2)],
                         *[torch.full((3, 2, 1), float("nan"), device="cuda") for _ in range(2)])
    x = torch.zeros(8, 1, 16, device="cuda")
    x[0, 0, :3] = torch.tensor([inf, -inf, 1e-40])
    x[1, 0, 5] = float("nan")
    x[2, 0, 4] = -1e-37
    x[4:, 0, 2] = 3.0  # the second block's scale is no 0
    x[5, 0, 3] = inf
    slots = torch.arange(8, 16, device="cuda")
    cache.append(x, x, slots)
    rows = [torch.empty(8, 1, 16, device="cuda") for _ in range(2)]
    cache.read(slots, *rows)
    q = torch.ones(1, 4, 2, 16, dtype=torch.bfloat16, device="cuda")
    out, lse = torch.zeros_like(q), torch.zeros(1, 4, 2, device="cuda")
    table = torch.tensor([[1]], dtype=torch.int32, device="cuda")
    cache.attend(q, table, torch.tensor([4], dtype=torch.int32, device="cuda"), out, cache.workspace(2, 4), out_lse=lse)
    torch.cuda.synchronize()
    want = torch.zeros(8, 16)
    want[4:, 2] = want[5, 3] = 3.0
    if kv == "e4m3":
        want[1, 5] = float("nan")
    most = float(kv_block_oracle.MOST[P])
    for pool, scale, got in ((cache.k_pool, cache.k_scale, rows[0]), (cache.v_pool, cache.v_scale, rows[1])):
        assert (scale[1, 0] == 0).all() and torch.equal(scale[1, 1].cpu(), torch.tensor([3.0]) / most)
        assert pool[1, 0, 0].float()[:3].tolist() == [most, -most, 0.0]
        # (3 / MAX is rounded, and so is its product with MAX: by 2^-24 each.)
        assert torch.allclose(got[:, 0].cpu(), want, rtol=2.0**-23 * 1.001, atol=0, equal_nan=True)
    # Token 1's key and value are no number for the queries that see it.
    nan = kv == "e4m3"
    assert (out[0, 0] == 0).all() and (lse[0, 0] == 0).all()
    assert torch.isnan(lse[0, 1:]).all() if nan else torch.allclose(lse[0].cpu(), torch.log(torch.arange(1.0, 5))[:, None].expand(-1, 2), atol=1e-6)
    assert torch.isnan(out[0, 1:]).all() if nan else (out == 0).all()
    assert sampler.status().flags == 0
