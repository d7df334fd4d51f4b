"""GPU: appends and attention inside the decode loop of
examples/paged_decode.py, each against the oracle on what it was really given,
with the bounds of its own roundings alone."""
import sys
from pathlib import Path

import pytest

import kv_oracle

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))

pytestmark = pytest.mark.gpu

STEPS = (0, 1, 15, 16, 33, 47, 48, 49, 64, 69)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16", "e4m3"])
def test_calls_of_a_decode_loop(sampler, dtype, monkeypatch):
    import paged_decode
    import torch

    from scriptonait_amd.kv import KVCache

    at = dict(step=0, calls=0)
    append, attend = KVCache.append, KVCache.attend

    def checked_append(self, k, v, slots, q=None, out_q=None, positions=None, rope=None, stream=None):
        if at["step"] not in STEPS:
            return append(self, k, v, slots, q, out_q, positions, rope, stream)
        host = [t.double().cpu() for t in (q, k, v)]
        append(self, k, v, slots, q, out_q, positions, rope, stream)
        live = (slots >= 0).cpu()
        pos = positions.cpu()
        want = kv_oracle.rotate(host[0], pos, rope.freqs, rope.style)
        tol = kv_oracle.rotate_bound(host[0], rope.freqs, rope.style) * 1.01 + kv_oracle.HALF_STEP[q.dtype] * want.abs() + 2.0**-25
        assert ((out_q.double().cpu() - want).abs() <= tol).all()
        for i, pool in enumerate((self.k_pool, self.v_pool)):
            want = kv_oracle.rotate(host[1], pos, rope.freqs, rope.style) if i == 0 else host[2]
            tol = kv_oracle.rotate_bound(host[1], rope.freqs, rope.style) * 1.01 if i == 0 else torch.zeros_like(want)
            if self.k_scale is not None:
                s = (self.k_scale, self.v_scale)[i].double().cpu()[:, None]
                want, tol = (want / s).clamp(-448, 448), tol / s + kv_oracle.F32 * (want / s).abs()
            half = kv_oracle.HALF_STEP[pool.dtype]
            tol = tol + torch.clamp(half * (want.abs() + tol), min=2.0**-10 if half == 2.0**-4 else 2.0**-25)
            got = pool.double().cpu().flatten(0, 1)[slots.cpu()[live]]
            assert ((got - want[live]).abs() <= tol[live]).all()
        at["calls"] += 1

    def checked_attend(self, q, table, lens, out, workspace, window=0, scale=None, out_lse=None, stream=None):
        attend(self, q, table, lens, out, workspace, window, scale, out_lse, stream)
        if at["step"] not in STEPS:
            return
        host = lambda t: None if t is None else t.cpu()  # noqa: E731
        want, _, tol, _ = kv_oracle.attend(q.cpu(), self.k_pool.cpu(), self.v_pool.cpu(), table.cpu(), lens.cpu(), window,
                                           self.head_dim**-0.5, host(self.k_scale), host(self.v_scale))
        assert ((out.double().cpu() - want).abs() <= tol).all()
        at["calls"] += 1

    monkeypatch.setattr(KVCache, "append", checked_append)
    monkeypatch.setattr(KVCache, "attend", checked_attend)
    steps = 70
    prompts = [([1, 2, 3], steps), ([10, 11, 12, 13, 14], 33), ([7], steps), ([5, 6], 49)]
    paged_decode.generate(sampler, prompts, steps, dtype=dtype, on_step=lambda t, h: at.update(step=t + 1))
    assert at["calls"] == 2 * 2 * len(STEPS)
