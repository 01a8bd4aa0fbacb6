"""The operators on either side of the head on another stream than torch's current one."""
import numpy as np
import pytest
import torch

import head_ops as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sampler():
    import gsample

    s = gsample.Sampler(vocab_size=512, max_rows=4)
    yield s
    s.close()


def test_a_result_s_memory_is_not_written_while_the_current_stream_uses_it(sampler):
    """A tensor that the current stream has yet to copy is dropped, and the result of a call on another stream takes
    its memory."""
    torch.cuda.empty_cache()
    rng = np.random.default_rng(41)
    rows, width = 1500, 8000  # a size of its own, so that the allocator hands the same block out again
    x = torch.from_numpy(rng.normal(0, 1, (rows, width)).astype(np.float32)).cuda()
    w = torch.ones(width).cuda()
    want, _ = ref.norm(x.cpu(), w.cpu())
    a, b = torch.randn(4096, 4096, device="cuda"), torch.empty(4096, 4096, device="cuda")
    side = torch.cuda.Stream()
    taken = 0
    for k in range(3):
        block, kept = torch.full_like(x, 3.0 + k), torch.empty_like(x)
        torch.cuda.synchronize()
        for _ in range(30):  # the copy below is some way off
            torch.mm(a, a, out=b)
        kept.copy_(block)
        at = block.data_ptr()
        del block
        y = sampler.rms_norm(x, w, stream=side.cuda_stream)
        taken += y.data_ptr() == at
        torch.cuda.synchronize()
        assert (kept == 3.0 + k).all()
        assert ((y.double().cpu() - want).abs() <= 2.0 ** -17 * want.abs() + 1e-37).all()
        del y, kept
    assert taken  # (the case that this is about)


def test_results_left_out_under_a_capture_are_refused(sampler):
    import gsample

    x, w = torch.ones(4, 64).cuda(), torch.ones(64).cuda()
    y = torch.zeros_like(x)
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    graph, refused = torch.cuda.CUDAGraph(), []
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        try:
            sampler.rms_norm(x, w, stream=other.cuda_stream)
        except gsample.GSampleError as e:
            refused.append(str(e))
        own = sampler.rms_norm(x, w, stream=side.cuda_stream)  # the graph's own memory
        sampler.rms_norm(own, w, out=y, stream=side.cuda_stream)
    assert refused and "under capture" in refused[0]
    for k in range(3):
        x.fill_(2.0 + k)
        y.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.allclose(y, torch.ones_like(y), atol=1e-5)
