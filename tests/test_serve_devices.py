"""The front ends of the serving operators and devices, on stand-ins for tensors:
calls launch with their tensors' device current and on its stream, and refuse
tensors of another one."""
import contextlib
from types import SimpleNamespace

import pytest
import torch

from cllm_inference_b200 import _lib, kv4, scoring


class Tensor:
    """As much of a CUDA tensor as the front ends look at."""

    def __init__(self, shape, dtype, device):
        self.shape, self.dtype, self.device = tuple(shape), dtype, device

    @property
    def is_cuda(self):
        return self.device >= 0

    def get_device(self):
        return self.device

    def is_contiguous(self):
        return True

    def dim(self):
        return len(self.shape)

    def numel(self):
        n = 1
        for x in self.shape:
            n *= x
        return n

    def stride(self, i=None):
        steps = (self.shape[1], 1)
        return steps if i is None else steps[i]

    def data_ptr(self):
        return 256

    def new_empty(self, shape):
        return Tensor(shape if isinstance(shape, tuple) else (shape,), self.dtype, self.device)


def ints(*shape, device=1):
    return Tensor(shape, torch.int32, device)


def floats(*shape, device=1):
    return Tensor(shape, torch.float32, device)


@pytest.fixture
def calls(monkeypatch):
    """(C function, current device, stream) of every call; device 0 is current."""
    now, seen = [0], []

    @contextlib.contextmanager
    def device(index):
        before, now[0] = now[0], index
        yield
        now[0] = before

    def function(name):
        def call(*args):
            seen.append((name, now[0], args[-1]))
            return 0
        return call

    fake = SimpleNamespace(**{n: function(n) for n in (
        "cllm_cuda_kv4_append", "cllm_cuda_kv4_attention", "cllm_cuda_kv4_fork", "cllm_cuda_kv4_compact",
        "cllm_cuda_token_scores")})
    monkeypatch.setattr(_lib, "load", lambda: fake)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch, "empty_like", lambda t, dtype=None: Tensor(t.shape, dtype or t.dtype, t.device))
    monkeypatch.setattr(kv4, "_dense_like", lambda t: Tensor(t.shape, t.dtype, t.device))
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 1000 + d)
    for module in (kv4, scoring):
        monkeypatch.setattr(module, "_raw_stream", lambda d: 1000 + d, raising=False)
        monkeypatch.setattr(module, "_current_device", lambda: now[0], raising=False)
    return seen


def cache(device=1, **other):
    parts = dict(pages=Tensor((2, 4, 2, 1, 1280), torch.uint8, device), table=ints(3, 2, device=device),
                 lens=ints(3, device=device))
    parts.update(other)
    return kv4.KV4Cache(**parts)


@pytest.mark.parametrize("device", [0, 1])
def test_calls_run_on_the_device_of_their_tensors(calls, device):
    c = cache(device)
    f, i = (lambda *s: floats(*s, device=device)), (lambda *s: ints(*s, device=device))
    c.append(0, f(4, 128), f(4, 128), i(4), i(4), q=f(4, 256), rope=f(64, 32, 2), values=True)
    c.attention(1, f(3, 256), lse=True)
    c.attention(1, f(5, 256), begin=i(4))
    c.fork(i(3), i(3))
    c.compact()
    scoring.token_scores(f(4, 50), i(4), 3)
    scoring.token_scores(f(4, 50))
    assert len(calls) == 7
    assert all(where == device and stream == 1000 + device for _, where, stream in calls)


def test_tensors_of_another_device_are_refused(calls):
    c = cache()
    f, i = floats, ints
    bad = [
        lambda: cache(pages=Tensor((2, 4, 2, 1, 1280), torch.uint8, -1)),  # of the host
        lambda: cache(table=ints(3, 2, device=0)), lambda: cache(lens=ints(3, device=0)),
        lambda: c.append(0, f(4, 128, device=0), f(4, 128), i(4), i(4)),
        lambda: c.append(0, f(4, 128), f(4, 128, device=0), i(4), i(4)),
        lambda: c.append(0, f(4, 128), f(4, 128), i(4, device=0), i(4)),
        lambda: c.append(0, f(4, 128), f(4, 128), i(4), i(4, device=0)),
        lambda: c.append(0, f(4, 128), f(4, 128), i(4), i(4), q=f(4, 256, device=0)),
        lambda: c.append(0, f(4, 128), f(4, 128), i(4), i(4), rope=f(64, 32, 2, device=0)),
        lambda: c.attention(0, f(3, 256, device=0)), lambda: c.attention(0, f(3, 256, device=-1)),
        lambda: c.attention(0, f(3, 256), begin=i(4, device=0)),
        lambda: c.fork(i(3, device=0), i(3)), lambda: c.fork(i(3), i(3, device=0)),
        lambda: scoring.token_scores(f(4, 50), i(4, device=0)), lambda: scoring.token_scores(f(4, 50, device=-1), i(4)),
    ]
    for n, call in enumerate(bad):
        with pytest.raises(_lib.CudaError) as e:
            call()
        assert e.value.code == _lib.ERR_INVALID_ARG, n
    assert not calls


@pytest.mark.parametrize("shape", [(), (2,), (3, 1), (3, 7)])
def test_lengths_of_another_shape_are_refused(calls, shape):
    with pytest.raises(_lib.CudaError) as e:
        cache(lens=ints(*shape))
    assert e.value.code == _lib.ERR_INVALID_ARG
