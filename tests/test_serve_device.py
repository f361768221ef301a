"""The serving bindings take no tensor that the GPU cannot read: the checks come before any CUDA call, so they are tried
here without a GPU."""
import pytest
import torch

import lnsb200

I32, F32, F16 = torch.int32, torch.float32, torch.float16


class Elsewhere:
    """a stand-in for a tensor on another device: everything but the device is the CPU tensor's"""

    def __init__(self, t, device):
        self.__dict__.update(_t=t, _device=device)

    def __getattr__(self, name):
        return getattr(self._t, name)

    def get_device(self):
        return self._device


class Refuses:
    """a library whose calls must not be reached"""

    def __getattr__(self, name):
        raise AssertionError("%s was called" % name)


@pytest.fixture
def ks(monkeypatch):
    k = object.__new__(lnsb200.KernelSet)
    k.lib = Refuses()
    lnsb200._load_types()
    monkeypatch.setattr(lnsb200, "_current_device", lambda: 0)
    return k


def _append():
    kc, k, q = torch.zeros(4, 16, 2, 64, dtype=F16), torch.zeros(3, 2, 64), torch.zeros(3, 4, 64)
    return dict(k=k, v=k.clone(), k_cache=kc, v_cache=kc.clone(), page_table=torch.zeros(1, 4, dtype=I32),
                q_start=torch.zeros(2, dtype=I32), kv_len=torch.zeros(1, dtype=I32), max_kv=10, q=q, q_out=q.half(),
                cos_sin=torch.zeros(10, 32, 2))


def _attn():
    a, q = _append(), torch.zeros(3, 4, 64, dtype=F16)
    a = {n: a[n] for n in ("k_cache", "v_cache", "page_table", "q_start", "kv_len", "max_kv")}
    return dict(a, q=q, max_q=3, dst=q.clone(), work=torch.zeros(8))


def _sample():
    f = lambda: torch.zeros(2)  # noqa: E731
    return dict(logits=torch.zeros(2, 50), u=f(), token=torch.zeros(2, dtype=I32), prob=f(), temperature=f(),
                top_k=torch.zeros(2, dtype=I32), top_p=f(), min_p=f())


CALLS = {"paged_append": _append, "paged_attn": _attn, "sample": _sample}
TENSORS = [(call, n) for call, make in CALLS.items() for n, t in make().items() if isinstance(t, torch.Tensor)]


@pytest.mark.parametrize("call", sorted(CALLS))
def test_host_tensors_refused(ks, call):
    with pytest.raises(ValueError, match="device"):
        getattr(ks, call)(**CALLS[call]())


@pytest.mark.parametrize("call,name", TENSORS, ids=lambda v: str(v))
@pytest.mark.parametrize("device", (-1, 1))
def test_one_tensor_elsewhere_refused(ks, call, name, device):
    """any single tensor on the host or on another GPU"""
    args = {n: Elsewhere(t, device if n == name else 0) if isinstance(t, torch.Tensor) else t for n, t in CALLS[call]().items()}
    with pytest.raises(ValueError, match="device"):
        getattr(ks, call)(**args)


@pytest.mark.parametrize("call", sorted(CALLS))
def test_another_current_device_refused(ks, call):
    """all on one GPU, which is not the current one"""
    args = {n: Elsewhere(t, 1) if isinstance(t, torch.Tensor) else t for n, t in CALLS[call]().items()}
    with pytest.raises(ValueError, match="device"):
        getattr(ks, call)(**args)


@pytest.mark.parametrize("call", sorted(CALLS))
def test_tensors_in_place_reach_the_library(ks, call):
    args = {n: Elsewhere(t, 0) if isinstance(t, torch.Tensor) else t for n, t in CALLS[call]().items()}
    with pytest.raises(AssertionError, match="was called"):
        getattr(ks, call)(**args)
