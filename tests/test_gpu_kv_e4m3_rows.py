"""GPU: E4M3 caches whose rows start on any multiple of 8 bytes, as the pools'
strides allow: heads beside gaps, pages of an odd number of 8s."""
import pytest

from test_gpu_kv_attend import TYPES, _check, _make

pytestmark = pytest.mark.gpu


def _spread(pool, gap, start):
    """The pool's rows `gap` bytes apart, the first `start` bytes into its memory."""
    import torch

    N, page, H, D = pool.shape
    raw = torch.full((N * page * H * (D + gap) + start,), 255, dtype=torch.uint8, device="cuda")
    rows = raw[start:].view(N, page, H, D + gap)[..., :D]
    rows.copy_(pool.view(torch.uint8))
    return rows.view(torch.float8_e4m3fn)


@pytest.mark.parametrize("q", ["bf16", "f16"])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 16), (128, 20), (96, 16), (80, 5), (256, 8), (192, 32), (48, 16), (16, 16),
                                    (40, 16)])
@pytest.mark.parametrize("gap,start", [(8, 0), (24, 8), (0, 8)])
def test_rows_on_8_bytes(sampler, q, D, page, gap, start):
    import torch

    from scriptonait_amd.kv import KVCache

    lens = [300, 1, 0, 77]
    c = _make(D + page + gap, lens, 6, 3, D, page, q, "e4m3")
    pools = [_spread(c[k], gap, start) for k in ("k_pool", "v_pool")]
    assert any(p.stride(2) % 16 or p.data_ptr() % 16 for p in pools) or D % 16
    cache = KVCache(sampler, *pools, c["k_scale"].cuda(), c["v_scale"].cuda())
    out = torch.full(c["q"].shape, 77.0, dtype=getattr(torch, TYPES[q]), device="cuda")
    lse = torch.full(out.shape[:2], 77.0, device="cuda")
    cache.attend(c["q"].cuda(), c["table"].cuda(), c["lens"].cuda(), out, cache.workspace(6), out_lse=lse)
    torch.cuda.synchronize()
    _check(c, (out.double().cpu(), lse.double().cpu()))
    assert sampler.status().flags == 0


@pytest.mark.parametrize("style", ["halves", "neighbours"])
@pytest.mark.parametrize("gap,start", [(8, 0), (24, 8)])
def test_appends_to_rows_on_8_bytes(sampler, style, gap, start):
    """What is stored there is what aligned rows get, and the gaps keep their bytes."""
    import torch

    from scriptonait_amd.kv import KVCache, Rope

    T, H, D, page = 20, 3, 64, 16
    g = torch.Generator().manual_seed(3)
    x = torch.randn(T, 2 * H, D, generator=g).bfloat16().cuda()
    slots, pos = torch.arange(T, device="cuda"), torch.arange(T, dtype=torch.int32, device="cuda") * 11
    scale = torch.full((H,), 0.25, device="cuda")
    plain = [torch.zeros(2, page, H, D, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)]
    spread = [_spread(p, gap, start) for p in plain]
    for pools in (plain, spread):
        KVCache(sampler, *pools, scale, scale).append(x[:, :H], x[:, H:], slots, positions=pos, rope=Rope(D, style=style))
    torch.cuda.synchronize()
    for p, s in zip(plain, spread):
        assert torch.equal(p.view(torch.uint8), s.view(torch.uint8)) and int(p.view(torch.uint8).count_nonzero()) > 0
        whole = s.view(torch.uint8)
        whole = whole.as_strided((2, page, H, gap), whole.stride(), whole.storage_offset() + D)
        assert (whole == 255).all()
    assert sampler.status().flags == 0
