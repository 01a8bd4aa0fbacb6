"""Results that a call on another stream than torch's current one allocates, and what the calls without a stream wait for."""
import contextlib
from types import SimpleNamespace

import pytest
import torch

import gsample
from gsample import runtime as rt

CURRENT, OTHER = 77, 78


class Torch:
    """torch's streams and allocator, noting what is asked of them in `seen`."""

    def __init__(self, capturing=()):
        self.seen, self.on = [], CURRENT
        self.cuda = self
        self.capturing = capturing
        self.uint8, self.int32, self.float32, self.bfloat16 = torch.uint8, torch.int32, torch.float32, torch.bfloat16

    def _stream(self, handle):
        return SimpleNamespace(cuda_stream=handle, synchronize=lambda: self.seen.append(f"{handle} drains"),
                               wait_stream=lambda s: self.seen.append(f"{handle} waits for {s.cuda_stream}"))

    def current_stream(self, device=None):
        return self._stream(self.on)

    def ExternalStream(self, handle, device=None):
        return self._stream(handle)

    @contextlib.contextmanager
    def stream(self, s):
        before, self.on = self.on, s.cuda_stream
        yield
        self.on = before

    def is_current_stream_capturing(self):
        return self.on in self.capturing

    def empty(self, shape, dtype, device):
        self.seen.append(f"memory of {self.on}")
        t = torch.zeros(shape, dtype=dtype)
        fake = SimpleNamespace(dtype=dtype, device=device, shape=t.shape, is_contiguous=lambda: True, data_ptr=t.data_ptr,
                               record_stream=lambda s: self.seen.append(f"kept for {s.cuda_stream}"))
        return fake


class Library:
    def __init__(self, seen):
        self.seen = seen

    def __getattr__(self, name):
        return lambda *args: self.seen.append(name) or 0


def sampler(capturing=()):
    rt._torch_types()
    s = object.__new__(rt.Sampler)
    s.torch, s.vocab, s.device, s.ctx = Torch(capturing), 128, torch.device("cpu"), None
    s.lib = Library(s.torch.seen)
    s._check = lambda status: None
    s.synchronize = lambda: s.torch.seen.append("results")
    return s


def t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


BF, U8, I32 = torch.bfloat16, torch.uint8, torch.int32
CALLS = [
    ("gs_rms_norm", 1, lambda s, **k: s.rms_norm(t(2, 32), t(32), **k)),
    ("gs_rms_norm_grad", 2, lambda s, **k: s.rms_norm_grad(t(2, 32), t(2, 32), t(32), **k)),
    ("gs_mx_quantize", 2, lambda s, **k: s.mx_quantize(t(2, 32), "e4m3", **k)),
    ("gs_mx_dequantize", 1, lambda s, **k: s.mx_dequantize(t(2, 32, dtype=U8), t(2, 1, dtype=U8), "e4m3", **k)),
    ("gs_mx_lmhead", 1, lambda s, **k: s.mx_lmhead(t(2, 64, dtype=U8), t(2, 2, dtype=U8), t(128, 32, dtype=U8),
                                                   t(128, 2, dtype=U8), **k)),
    ("gs_lmhead_loss", 2, lambda s, **k: s.lmhead_loss(t(2, 64, dtype=BF), t(128, 64, dtype=BF), t(2, dtype=I32), **k)),
    ("gs_lmhead_loss_grad", 2, lambda s, **k: s.lmhead_loss_grad(t(2, 64, dtype=BF), t(128, 64, dtype=BF), t(2, dtype=I32),
                                                                 t(2), t(2), **k)),
]


@pytest.mark.parametrize("name,results,call", CALLS, ids=[c[0] for c in CALLS])
def test_another_stream_waits_for_what_still_uses_the_memory(name, results, call):
    """The allocator hands out memory that torch's current stream may still be reading or writing."""
    s = sampler()
    call(s, stream=OTHER)
    seen = s.torch.seen
    assert seen.count(f"memory of {CURRENT}") == results and seen.count(f"kept for {OTHER}") == results
    last = max(i for i, what in enumerate(seen) if what == f"memory of {CURRENT}")
    wait = f"{OTHER} waits for {CURRENT}"
    assert wait in seen[last:] and len(seen) - 1 - seen[::-1].index(wait) < seen.index(name), seen
    assert seen[-1] == name  # (and nothing waits for the call itself)


@pytest.mark.parametrize("name,results,call", CALLS, ids=[c[0] for c in CALLS])
@pytest.mark.parametrize("stream", [None, CURRENT])
def test_torch_s_own_stream_needs_no_further_wait(name, results, call, stream):
    s = sampler()
    call(s, stream=stream)
    assert [w for w in s.torch.seen if not w.startswith("memory")] == (
        [name] if stream else [f"{CURRENT} drains", name, "results"])


@pytest.mark.parametrize("name,results,call", CALLS, ids=[c[0] for c in CALLS])
@pytest.mark.parametrize("capturing", [CURRENT, OTHER])
def test_no_memory_across_a_capture(name, results, call, capturing):
    """Such a wait would reach into or out of the graph: the results' memory has to be given."""
    s = sampler((capturing,))
    with pytest.raises(gsample.GSampleError, match="under capture") as e:
        call(s, stream=OTHER)
    assert e.value.status == 1 and name not in s.torch.seen
    assert not any("waits" in w for w in s.torch.seen)


@pytest.mark.parametrize("stream", [None, 0, OTHER])
def test_head_and_sampler_without_a_stream_wait_for_the_results(stream):
    """What the call reads may be dropped once it returns."""
    s = sampler()
    batch = rt.Batch()
    batch.rows = 2
    s.mx_lmhead_sample_launch(t(2, 64, dtype=U8), t(2, 2, dtype=U8), t(128, 32, dtype=U8), t(128, 2, dtype=U8), 0.0, t(2, 128),
                              batch, stream=stream)
    assert s.torch.seen == (["gs_mx_lmhead_sample"] if stream else [f"{CURRENT} drains", "gs_mx_lmhead_sample", "results"])
