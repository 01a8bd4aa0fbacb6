"""rms_norm and its gradients against the plain form in 64 bits."""
import numpy as np
import pytest
import torch

import head_ops as ref

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def sampler():
    import gsample

    s = gsample.Sampler(vocab_size=512, max_rows=1)
    yield s
    s.close()


def rows_of(rng, rows, width, dtype, scale=1.0):
    x = rng.normal(0, 1, (rows, width)) * np.exp(rng.normal(0, 0.5, (rows, 1))) * scale
    return torch.from_numpy(x.astype(np.float32)).to(dtype)


# y is one rounding of binary32 products whose r carries the sum of squares'
# roundings (at most width / 8 + 16 of them in a row, halved by the root): 2^-17
# covers widths up to 16384
def close(got, want, dtype, more=0.0):
    half = ref.U16 if dtype == torch.bfloat16 else ref.U32
    bound = (half + 2.0 ** -17) * want.abs() + more + 1e-37
    bad = (got.double().cpu() - want).abs() > bound
    assert not bad.any(), (int(bad.sum()), float(((got.double().cpu() - want).abs() / bound).max()))


SIZES = [(1, 1), (1, 32), (3, 7), (5, 64), (1, 2048), (2, 577), (7, 704), (4, 2049), (3, 4096), (2, 8191), (2, 16384),
         (2050, 96), (2051, 2048), (2049, 513), (4099, 33)]


@pytest.mark.parametrize("rows,width", SIZES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_norm_and_gradient_match_the_formulas(sampler, rows, width, dtype):
    rng = np.random.default_rng(rows * 31 + width)
    t = DTYPES[dtype]
    x, res, dy, ds = (rows_of(rng, rows, width, t) for _ in range(4))
    w = torch.from_numpy(rng.normal(1, 0.3, width).astype(np.float32)).to(t)
    want, h = ref.norm(x, w, res, 1e-6)
    summed = torch.empty_like(x, device="cuda")
    y = sampler.rms_norm(x.cuda(), w.cuda(), residual=res.cuda(), summed=summed)
    assert torch.equal(summed.cpu(), h)
    close(y, want, t)
    dx, dw = sampler.rms_norm_grad(dy.cuda(), summed, w.cuda(), dsummed=ds.cuda())
    want_dx, want_dw, size = ref.norm_grad(dy, h, w, ds, 1e-6)
    # dx subtracts two terms: their own roundings stay where the difference is small
    hd = h.double()
    r = 1 / torch.sqrt((hd * hd).mean(1, keepdim=True) + 1e-6)
    g = dy.double() * w.double()
    parts = r * (g.abs() + hd.abs() * r * r * (g * hd).abs().mean(1, keepdim=True)) + ds.double().abs()
    close(dx, want_dx, t, 2.0 ** -17 * parts)
    bad = (dw.double().cpu() - want_dw).abs() > ((rows + 64) * ref.U32 + 2.0 ** -17) * size + 1e-37
    assert not bad.any(), int(bad.sum())


@pytest.mark.parametrize("offset", [0.0, 1.0])
@pytest.mark.parametrize("weight_dtype", ["f32", "bf16"])
def test_without_residual_with_offset_and_a_weight_of_its_own_type(sampler, offset, weight_dtype):
    rng = np.random.default_rng(5)
    x = rows_of(rng, 9, 1536, torch.bfloat16)
    dy = rows_of(rng, 9, 1536, torch.bfloat16)
    w = torch.from_numpy(rng.normal(0, 0.3, 1536).astype(np.float32)).to(DTYPES[weight_dtype])
    want, _ = ref.norm(x, w, None, 1e-5, offset)
    y = sampler.rms_norm(x.cuda(), w.cuda(), eps=1e-5, weight_offset=offset)
    close(y, want, torch.bfloat16)
    dx, dw = sampler.rms_norm_grad(dy.cuda(), x.cuda(), w.cuda(), eps=1e-5, weight_offset=offset)
    want_dx, want_dw, size = ref.norm_grad(dy, x, w, None, 1e-5, offset)
    close(dx, want_dx, torch.bfloat16, 2.0 ** -15 * want_dx.abs().max())
    assert ((dw.double().cpu() - want_dw).abs() <= 2.0 ** -15 * size).all()


def test_strided_rows_odd_offsets_and_results_in_place(sampler):
    rng = np.random.default_rng(6)
    for t in (torch.float32, torch.bfloat16):
        base = rows_of(rng, 11, 1009, t).cuda()
        x, res = base[:, 3:3 + 417], rows_of(rng, 11, 500, t).cuda()[:, 1:418]
        w = torch.from_numpy(rng.normal(1, 0.1, 417).astype(np.float32)).to(t)
        want, h = ref.norm(x.cpu(), w, res.cpu())
        keep = base.clone()
        close(sampler.rms_norm(x, w.cuda(), residual=res), want, t)
        assert torch.equal(base, keep)
        xc, rc = x.contiguous(), res.contiguous()
        y = sampler.rms_norm(xc, w.cuda(), residual=rc, summed=rc, out=xc)
        assert y.data_ptr() == xc.data_ptr() and torch.equal(rc.cpu(), h)
        close(y, want, t)
        dy = rows_of(rng, 11, 417, t).cuda()
        want_dx, _, _ = ref.norm_grad(dy.cpu(), h, w)
        dx, _ = sampler.rms_norm_grad(dy, rc, w.cuda(), dx=dy)
        close(dx, want_dx, t, 2.0 ** -15 * want_dx.abs().max())


def test_blocks_are_those_of_the_quantiser(sampler):
    """The e4m3 output is mx_quantize of the unrounded y: rows whose f32 y is exact in both."""
    rng = np.random.default_rng(7)
    for rows, width in ((1, 32), (5, 96), (3, 2048), (2050, 64), (2, 8224)):
        x = rows_of(rng, rows, width, torch.float32).cuda()
        w = torch.ones(width).cuda()
        y = sampler.rms_norm(x, w)
        codes, scales = torch.empty(rows, width, dtype=torch.uint8).cuda(), torch.empty(rows, width // 32, dtype=torch.uint8).cuda()
        out = torch.empty_like(x)
        sampler.rms_norm(x, w, out=out, codes=codes, scales=scales)
        assert torch.equal(out, y)
        c, s = sampler.mx_quantize(y, "e4m3")
        assert torch.equal(c, codes) and torch.equal(s, scales)


def test_zero_rows_tiny_rows_and_values_that_are_not_finite(sampler):
    w = torch.ones(64).cuda()
    x = torch.zeros(4, 64)
    x[1] = 1e-30
    x[2, 5] = float("inf")
    x[3, 9] = float("nan")
    y = sampler.rms_norm(x.cuda(), w, eps=1e-6).cpu()
    want, _ = ref.norm(x, w.cpu())
    assert torch.equal(y[0], torch.zeros(64)) and torch.allclose(y[1].double(), want[1], rtol=1e-6, atol=0)
    assert y[2, 5].isnan() and (y[2, :5] == 0).all() and y[3].isnan().all()
    codes, scales = torch.empty(4, 64, dtype=torch.uint8).cuda(), torch.empty(4, 2, dtype=torch.uint8).cuda()
    sampler.rms_norm(x.cuda(), w, codes=codes, scales=scales)
    v = sampler.mx_dequantize(codes, scales, "e4m3", dtype=torch.float32).cpu()
    assert (v[0] == 0).all() and scales[0].tolist() == [0, 0]
    assert v[2, :32].isnan().all() and (v[2, 32:] == 0).all() and v[3].isnan().all()


def test_no_rows(sampler):
    x = torch.empty(0, 40).cuda()
    w = torch.ones(40).cuda()
    assert sampler.rms_norm(x, w).shape == (0, 40)
    dx, dw = sampler.rms_norm_grad(x, x, w, dweight=torch.full((40,), 7.0).cuda())
    assert dx.shape == (0, 40) and (dw == 0).all()


def test_gradient_against_differences(sampler):
    rng = np.random.default_rng(8)
    x, dy = rows_of(rng, 6, 257, torch.float32), rows_of(rng, 6, 257, torch.float32)
    w = torch.from_numpy(rng.normal(1, 0.3, 257).astype(np.float32))
    dx, dw = sampler.rms_norm_grad(dy.cuda(), x.cuda(), w.cuda())
    dirx, dirw = torch.from_numpy(rng.normal(0, 1, (6, 257))), torch.from_numpy(rng.normal(0, 1, 257))
    f = lambda a, b: float((ref.norm(a, b)[0] * dy.double()).sum())  # noqa: E731
    e = 1e-5
    by_x = (f(x.double() + e * dirx, w) - f(x.double() - e * dirx, w)) / (2 * e)
    by_w = (f(x, w.double() + e * dirw) - f(x, w.double() - e * dirw)) / (2 * e)
    assert abs(float((dx.double().cpu() * dirx).sum()) - by_x) <= 1e-4 * abs(by_x) + 1e-4
    assert abs(float((dw.double().cpu() * dirw).sum()) - by_w) <= 1e-4 * abs(by_w) + 1e-4


def test_same_bits_every_time_on_another_stream_and_in_a_graph(sampler):
    rng = np.random.default_rng(9)
    x, res, dy = (rows_of(rng, 600, 1000, torch.bfloat16).cuda() for _ in range(3))
    w = torch.from_numpy(rng.normal(1, 0.3, 1000).astype(np.float32)).cuda()
    h = torch.empty_like(x)
    y = sampler.rms_norm(x, w, residual=res, summed=h)
    dx, dw = sampler.rms_norm_grad(dy, h, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y2 = sampler.rms_norm(x, w, residual=res, stream=side.cuda_stream)
        dx2, dw2 = sampler.rms_norm_grad(dy, h, w, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(y, y2) and torch.equal(dx, dx2) and torch.equal(dw, dw2)
    graph = torch.cuda.CUDAGraph()
    y3, h3, dx3, dw3 = (torch.empty_like(v) for v in (y, h, dx, dw))
    with torch.cuda.graph(graph, stream=side):
        sampler.rms_norm(x, w, residual=res, out=y3, summed=h3, stream=side.cuda_stream)
        sampler.rms_norm_grad(dy, h3, w, dx=dx3, dweight=dw3, stream=side.cuda_stream)
    for k in range(3):
        for v in (y3, h3, dx3, dw3):
            v.zero_()
        x.copy_(torch.roll(x, 1, 0))
        want = sampler.rms_norm(x, w, residual=res, summed=h)
        want_dx, want_dw = sampler.rms_norm_grad(dy, h, w)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y3, want) and torch.equal(dx3, want_dx) and torch.equal(dw3, want_dw)


def test_refusals(sampler):
    import gsample

    x = torch.zeros(2, 48).cuda()
    w = torch.ones(48).cuda()
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8).cuda()  # noqa: E731
    for call in (
        lambda: sampler.rms_norm(x.half(), w),
        lambda: sampler.rms_norm(x, w, eps=-1.0),
        lambda: sampler.rms_norm(x, w, weight_offset=float("nan")),
        lambda: sampler.rms_norm(x, w, codes=u8(2, 48), scales=u8(2, 1)),  # 48 holds no whole number of blocks
        lambda: sampler.rms_norm(torch.zeros(1, 16385).cuda(), torch.ones(16385).cuda()),
    ):
        with pytest.raises(gsample.GSampleError):
            call()
