"""A cache, a pool of pages and a stream belong to the sampler's device. Shown
on the CPU with tensors that name another device."""
import pytest
import torch

from scriptonait_amd import kv
from scriptonait_amd import sampler as smp


class _Sampler:
    ctx = None

    def __init__(self, device):
        self.device = device


class _OnGpu1(torch.Tensor):
    device = property(lambda self: torch.device("cuda:1"))


def _gpu1(*shape, dtype=torch.int32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_OnGpu1)


def test_a_sampler_names_its_device(monkeypatch):
    class Library:
        llmhip_ctx_create = staticmethod(lambda device, ctx: 0)

    monkeypatch.setattr(smp, "load_library", Library)
    assert smp.Sampler(3).device == 3


def test_caches_of_another_device_are_refused():
    pools = [_gpu1(4, 16, 2, 64, dtype=torch.bfloat16) for _ in range(2)]
    with pytest.raises(ValueError, match="cuda:1.*cuda:0"):
        kv.KVCache(_Sampler(0), *pools)
    assert kv.KVCache(_Sampler(1), *pools).device == torch.device("cuda:1")


def test_pages_of_another_device_are_refused():
    with pytest.raises(ValueError, match="cuda:1.*cuda:0"):
        kv.PagePool(_Sampler(0), 8, 16, _gpu1(8), _gpu1(2))
    assert kv.PagePool(_Sampler(1), 8, 16, _gpu1(8), _gpu1(2)).device == torch.device("cuda:1")


def test_pages_start_out_on_the_samplers_device(monkeypatch):
    asked = []
    arange, tensor = torch.arange, torch.tensor

    def made(make):
        def f(*a, device=None, **k):
            asked.append(torch.device(device))
            return make(*a, **k).as_subclass(_OnGpu1)
        return f

    monkeypatch.setattr(kv.torch, "arange", made(arange))
    monkeypatch.setattr(kv.torch, "tensor", made(tensor))
    assert kv.PagePool(_Sampler(1), 8, 16).device == torch.device("cuda:1")
    assert asked == [torch.device("cuda:1")] * 2
    with pytest.raises(ValueError, match="cuda:1.*cuda:0"):
        kv.PagePool(_Sampler(0), 8, 16, device="cuda:1")


class _Stream:
    cuda_stream = 0

    def __init__(self, device):
        self.device = torch.device(device)


def test_streams_of_another_device_are_refused():
    device = torch.device("cuda:0")
    with pytest.raises(ValueError, match="stream.*cuda:1"):
        kv._on(_Stream("cuda:1"), device, ())
    assert kv._on(_Stream("cuda:0"), device, ()) == 0
