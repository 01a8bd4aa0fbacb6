"""The Python checks of the operators on either side of the head: what they refuse never reaches the library."""
import ctypes

import pytest
import torch

import gsample
from gsample import runtime as rt


class NoLibrary:
    def __getattr__(self, name):
        raise AssertionError(f"{name} was called")


@pytest.fixture
def sampler():
    rt._torch_types()
    s = object.__new__(rt.Sampler)
    s.torch, s.vocab, s.device, s.ctx = torch, 128, torch.device("cpu"), None
    s.lib = NoLibrary()
    return s


def t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


BF, U8, I32 = torch.bfloat16, torch.uint8, torch.int32


@pytest.mark.parametrize("call,message", [
    (lambda s: s.rms_norm(t(2, 8, dtype=torch.float64), t(8)), "x must be float32 or bfloat16"),
    (lambda s: s.rms_norm(t(16), t(8)), "x must have shape"),
    (lambda s: s.rms_norm(t(2, 8), t(7)), "weight must have shape (8,)"),
    (lambda s: s.rms_norm(t(2, 8), t(8), residual=t(2, 8, dtype=BF)), "residual must be float32"),
    (lambda s: s.rms_norm(t(2, 8), t(8), residual=t(3, 8)), "residual must have shape"),
    (lambda s: s.rms_norm(t(8, 2).t(), t(8)), "rows must be contiguous"),
    (lambda s: s.rms_norm(t(1, 8).expand(4, 8), t(8)), "rows must be contiguous and not overlap"),
    (lambda s: s.rms_norm(t(2, 8), t(8), out=t(2, 16)[:, :8]), "out must be contiguous"),
    (lambda s: s.rms_norm(t(2, 32), t(32), codes=t(2, 32, dtype=U8)), "codes and scales go together"),
    (lambda s: s.rms_norm(t(2, 32), t(32), codes=t(2, 16, dtype=U8), scales=t(2, 1, dtype=U8)), "codes must have shape"),
    (lambda s: s.rms_norm_grad(t(2, 8, dtype=BF), t(2, 8), t(8)), "dy must be float32"),
    (lambda s: s.rms_norm_grad(t(2, 8), t(2, 8), t(8), dweight=t(8, dtype=BF)), "dweight must be float32"),
    (lambda s: s.mx_quantize(t(2, 32), "e5m2"), "format must be one of"),
    (lambda s: s.mx_quantize(t(2, 32, dtype=torch.float16), "e2m1"), "x must be float32 or bfloat16"),
    (lambda s: s.mx_quantize(t(2, 32), "e2m1", codes=t(2, 32, dtype=U8)), "codes must have shape (2, 16)"),
    (lambda s: s.mx_dequantize(t(2, 16, dtype=U8), t(2, 2, dtype=U8), "e2m1"), "scales must have shape (2, 1)"),
    (lambda s: s.mx_lmhead(t(3, 64, dtype=U8), t(3, 2, dtype=U8), t(127, 32, dtype=U8), t(128, 2, dtype=U8)),
     "weight must have shape (128, 32)"),
    (lambda s: s.mx_lmhead(t(3, 64, dtype=U8), t(3, 2, dtype=U8), t(128, 32, dtype=U8), t(128, 2, dtype=U8),
                           out=t(3, 128, dtype=BF)), "out must be float32"),
    (lambda s: s.lmhead_loss(t(3, 64), t(128, 64, dtype=BF), t(3, dtype=I32)), "hidden must be bfloat16"),
    (lambda s: s.lmhead_loss(t(3, 64, dtype=BF), t(100, 64, dtype=BF), t(3, dtype=I32)), "weight must have shape (128, 64)"),
    (lambda s: s.lmhead_loss(t(3, 64, dtype=BF), t(128, 64, dtype=BF), t(3, dtype=torch.int64)), "targets must be int32"),
    (lambda s: s.lmhead_loss(t(3, 64, dtype=BF), t(128, 64, dtype=BF), t(4, dtype=I32)), "targets must have shape (3,)"),
    (lambda s: s.lmhead_loss_grad(t(3, 64, dtype=BF), t(128, 64, dtype=BF), t(3, dtype=I32), t(3), t(3, dtype=BF)),
     "dloss must be float32"),
    (lambda s: s.lmhead_loss_grad(t(3, 64, dtype=BF), t(128, 64, dtype=BF), t(3, dtype=I32), t(3), t(3),
                                  dweight=t(128, 64)), "dweight must be bfloat16"),
])
def test_refused_before_the_library(sampler, call, message):
    with pytest.raises(gsample.GSampleError) as e:
        call(sampler)
    assert message in str(e.value), str(e.value)
    assert e.value.status == 1


@pytest.mark.parametrize("stream,waits", [(None, 1), (0, 1), (77, 0)])
def test_the_default_stream_is_waited_for(sampler, stream, waits):
    """0, the default stream's handle, stands for the context's own stream in the library."""
    from types import SimpleNamespace

    seen = []
    current = SimpleNamespace(synchronize=lambda: seen.append("inputs"), cuda_stream=77)
    sampler.torch = SimpleNamespace(cuda=SimpleNamespace(current_stream=lambda device: current), empty=torch.empty)
    sampler.synchronize = lambda: seen.append("results")
    assert sampler._begin(stream) == (stream or None)
    assert sampler._empty((2,), torch.float32, stream).shape == (2,)
    sampler._end(stream)
    assert seen == ["inputs", "results"][:2 * waits]


def test_other_devices_are_refused(sampler):
    sampler.device = torch.device("cuda", 0)
    with pytest.raises(gsample.GSampleError, match="sampler's device"):
        sampler.rms_norm(t(2, 8), t(8))


def test_the_library_refuses_a_null_context():
    lib = rt.library()
    n = ctypes.c_void_p()
    assert lib.gs_rms_norm(n, n, n, n, 0, 0, 1, 8, 8, 8, 1e-6, 0.0, n, n, n, n, n) == 1
    assert lib.gs_rms_norm_grad(n, n, n, n, n, 0, 0, 1, 8, 8, 8, 8, 1e-6, 0.0, n, n, n) == 1
    assert lib.gs_mx_quantize(n, n, 0, 0, 1, 32, 32, n, n, n) == 1
    assert lib.gs_mx_dequantize(n, n, n, 0, 1, 32, 0, n, n) == 1
    assert lib.gs_mx_lmhead(n, n, n, n, n, 1, 64, 0.0, n, n) == 1
    assert lib.gs_mx_lmhead_sample(n, n, n, n, n, 64, 0.0, n, None, n) == 1
    assert lib.gs_lmhead_loss(n, n, n, n, 1, 64, 0.0, n, n, n) == 1
    assert lib.gs_lmhead_loss_grad(n, n, n, n, n, n, 1, 64, 0.0, n, n, n) == 1
