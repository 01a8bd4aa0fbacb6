"""Microscaled quantisation, and the 4-bit head, against the plain forms."""
import numpy as np
import pytest
import torch

import head_ops as ref

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def samplers():
    import gsample

    made = {}

    def get(vocab, rows=1):
        if (vocab, rows) not in made:
            made[vocab, rows] = gsample.Sampler(vocab_size=vocab, max_rows=rows)
        return made[vocab, rows]

    yield get
    for s in made.values():
        s.close()


def blocks(rng, rows, width):
    """Rows with blocks of every kind: ordinary, zero, one value alone, ties, at the range's ends, subnormal."""
    x = rng.normal(0, 1, (rows, width)) * np.exp(rng.normal(0, 3, (rows, width // 32)).repeat(32, 1))
    x = x.astype(np.float32).reshape(-1, 32)
    kinds = [np.zeros(32), np.r_[np.zeros(31), 1e-20], np.arange(32) / 4.0, np.arange(32) / 8.0 - 2.0,
             np.r_[3.0e38, np.arange(31) * 1e37], np.full(32, 1e-41), np.r_[2.0 ** -126, np.full(31, -2.0 ** -130)],
             np.r_[7.0, -7.0, 6.5, 5.0, -5.0, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25, -0.25, -0.0, np.zeros(19)],
             np.r_[np.full(4, 447.0), np.full(4, 449.0), np.full(8, 479.9), np.linspace(0, 500, 16)],
             np.r_[511.0, np.arange(31) * 2.0 ** -9], np.r_[1.0 - 2.0 ** -24, np.linspace(-1, 1, 31)]]
    for i in range(len(x)):
        if i % 3 == 1:
            x[i] = kinds[(i // 3) % len(kinds)]
    return x.reshape(rows, width)


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,width", [(1, 32), (1, 64), (3, 96), (37, 160), (2, 2048), (129, 32)])
def test_codes_and_scales_are_the_definition_s(samplers, fmt, dtype, rows, width):
    s = samplers(512)
    rng = np.random.default_rng(rows + width)
    x = torch.from_numpy(blocks(rng, rows, width)).to(DTYPES[dtype])
    want_codes, want_scales = ref.mx_quantize(x.double().numpy(), fmt)
    codes, scales = s.mx_quantize(x.cuda(), fmt)
    assert np.array_equal(scales.cpu().numpy(), want_scales)
    assert np.array_equal(codes.cpu().numpy(), ref.mx_pack(want_codes, fmt))
    values = ref.mx_dequantize(want_codes, want_scales, fmt)
    assert np.array_equal(s.mx_dequantize(codes, scales, fmt, dtype=torch.float32).cpu().double().numpy(), values)
    half = s.mx_dequantize(codes, scales, fmt)
    assert torch.equal(half.cpu(), torch.from_numpy(values).to(torch.bfloat16))


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
def test_special_blocks_read_back_as_nan(samplers, fmt):
    s = samplers(512)
    x = np.ones((4, 96), np.float32)
    x[0, 5], x[1, 40], x[2, 95] = np.nan, np.inf, -np.inf
    codes, scales = s.mx_quantize(torch.from_numpy(x).cuda(), fmt)
    v = s.mx_dequantize(codes, scales, fmt).float().cpu().numpy()
    bad = np.zeros((4, 96), bool)
    bad[0, :32] = bad[1, 32:64] = bad[2, 64:] = True
    assert np.array_equal(np.isnan(v), bad) and (v[~bad] == 1).all()


def test_every_code_reads_back(samplers):
    s = samplers(512)
    for fmt in ("e2m1", "e4m3"):
        n = 16 if fmt == "e2m1" else 256
        codes = np.tile(np.arange(n, dtype=np.uint8), (256, 32 * 8 // n * 2))[:, :512]
        scales = np.repeat(np.arange(256, dtype=np.uint8)[:, None], codes.shape[1] // 32, 1)
        want = ref.mx_dequantize(codes, scales, fmt)
        got = s.mx_dequantize(torch.from_numpy(ref.mx_pack(codes, fmt).copy()).cuda(), torch.from_numpy(scales).cuda(), fmt,
                              dtype=torch.float32).cpu().numpy()
        with np.errstate(over="ignore"):
            assert np.array_equal(got, want.astype(np.float32), equal_nan=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
def test_many_blocks_read_back_as_in_slices(samplers, fmt, dtype):
    gen = torch.Generator(device="cuda:0").manual_seed(3)
    rows, width = 349526, 96  # over 2^22 groups of 8, and no multiple of a workgroup's
    x = torch.randn(rows, width, device="cuda:0", generator=gen)
    s = samplers(1000)
    codes, scales = s.mx_quantize(x, fmt)
    whole = torch.full((rows + 1, width), 7.0, dtype=dtype).cuda()
    s.mx_dequantize(codes, scales, fmt, out=whole[:rows])
    for a, b in ((0, 100), (100, 4000), (rows - 3000, rows)):
        some = s.mx_quantize(x[a:b], fmt)
        assert torch.equal(some[0], codes[a:b]) and torch.equal(some[1], scales[a:b])
        assert torch.equal(s.mx_dequantize(*some, fmt, dtype=dtype), whole[a:b])
    # The scale puts a block's largest magnitude m at 4 to 8 (e2m1) or 256 to 512 (e4m3). Past 6 or 448 it becomes
    # that: off by less than m - 6 <= m 2/8, or m - 448 <= m 64/512. Anything else is off by at most half a step of the
    # top binade, 1 <= m/4, or 16 <= m/16. bf16 holds every one of these values (and the subtraction below rounds).
    off = (whole[:rows].float() - x).abs().view(rows, -1, 32)
    most = x.abs().view(rows, -1, 32).amax(2) * (2.0 ** -2 if fmt == "e2m1" else 2.0 ** -3) * (1 + 2.0 ** -20)
    assert (off.amax(2) <= most).all()
    assert (whole[rows] == 7.0).all()


def test_strided_rows_and_no_rows(samplers):
    s = samplers(512)
    rng = np.random.default_rng(3)
    for t in (torch.float32, torch.bfloat16):
        base = torch.from_numpy(rng.normal(0, 1, (9, 201)).astype(np.float32)).to(t).cuda()
        x = base[:, 5:5 + 160]
        a, b = s.mx_quantize(x, "e2m1"), s.mx_quantize(x.contiguous(), "e2m1")
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    codes, scales = s.mx_quantize(torch.empty(0, 64).cuda(), "e4m3")
    assert codes.shape == (0, 64) and s.mx_dequantize(codes, scales, "e4m3").shape == (0, 64)


def head_operands(rng, m, width, vocab, special=False):
    h = rng.normal(0, 1, (m, width)) * np.exp(rng.normal(0, 0.5, (m, 1)))
    w = rng.normal(0, 0.05, (vocab, width)) * np.exp(rng.normal(0, 0.5, (vocab, 1)))
    hc, hs = quick_quantize(h, "e4m3")
    wc, ws = quick_quantize(w, "e2m1")
    if special:
        ws[min(5, vocab - 1), -1] = 255
    hv, wv = ref.mx_dequantize(hc, hs, "e4m3"), ref.mx_dequantize(wc, ws, "e2m1")
    cuda = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    return (cuda(hc), cuda(hs), cuda(ref.mx_pack(wc, "e2m1")), cuda(ws)), torch.from_numpy(hv), torch.from_numpy(wv)


def quick_quantize(x, fmt):
    """Codes near x's (any codes serve as the head's operands)."""
    emax, _, _, top = ref.FORMATS[fmt]
    values = ref.mx_values(fmt)
    half = values[:len(values) // 2]
    half = half[np.isfinite(half)]
    b = x.reshape(x.shape[0], -1, 32)
    scales = np.clip(np.floor(np.log2(np.abs(b).max(2))) - emax + 127, 0, 254).astype(np.uint8)
    v = np.minimum(np.abs(b) / 2.0 ** (scales.astype(np.float64) - 127)[:, :, None], top)
    codes = np.minimum(np.searchsorted(half, v), len(half) - 1) + np.where(b < 0, len(values) // 2, 0)
    return codes.astype(np.uint8).reshape(x.shape), scales


# The scaled matrix instruction adds 8 neighbouring products in fixed point: a
# product is cut off 13 bits below the group's largest product exponent (checked
# lane by lane: beside a product of 1, one of 2^-13 is kept, one of 2^-14 is
# not, and from the next group of 8 on the sums are binary32). 2^exponent is at
# most the product, so a group is off by at most 8 x 2^-13 of its largest
# product. The groups' sums are added in binary32, at most width / 8 of them and
# each off by at most a whole step. The cap adds a few roundings of the result.
def check_logits(got, hv, wv, cap):
    z = hv @ wv.T
    m, width = hv.shape
    cut = torch.zeros_like(z)
    for k in range(0, width, 8):
        cut += (hv[:, None, k:k + 8] * wv[None, :, k:k + 8]).abs().amax(2)
    bound = 8 * 2.0 ** -13 * cut + width / 4 * ref.U32 * (hv.abs() @ wv.abs().T) + 1e-30
    want = ref.capped(z, cap)
    bound = bound + 8 * ref.U32 * want.abs()
    ok = ((got.double().cpu() - want).abs() <= bound) | (want.isnan() & got.cpu().isnan())
    assert ok.all(), (int((~ok).sum()), torch.nonzero(~ok)[:5].tolist())
    # and over all logits together (measured 2e-6 to 7e-6 of their norm)
    fine = ~want.isnan()
    assert (got.double().cpu() - want)[fine].norm() <= 2.0 ** -14 * want[fine].norm() + 1e-30


@pytest.mark.parametrize("m", [1, 2, 17, 32, 33, 64, 65, 128, 129, 300])
@pytest.mark.parametrize("width,vocab,cap", [(64, 1, 0.0), (128, 257, 30.0), (576, 1000, 0.0), (1536, 515, 2.0), (320, 256, 0.0)])
def test_head_matches_the_dequantised_product(samplers, m, width, vocab, cap):
    rng = np.random.default_rng(m * 7 + width)
    ops, hv, wv = head_operands(rng, m, width, vocab)
    s = samplers(vocab)
    out = torch.full((m + 1, vocab), 77.0).cuda()
    s.mx_lmhead(*ops, softcap_value=cap, out=out[:m])
    check_logits(out[:m], hv, wv, cap)
    assert (out[m] == 77.0).all()  # rows behind the last stay as they were


def test_head_of_a_large_vocabulary_and_wide_rows(samplers):
    rng = np.random.default_rng(11)
    for m, width, vocab in ((3, 5376, 3001), (70, 2048, 8192)):
        ops, hv, wv = head_operands(rng, m, width, vocab)
        check_logits(samplers(vocab).mx_lmhead(*ops), hv, wv, 0.0)


@pytest.mark.parametrize("m,width,vocab,cap,shift", [
    (100, 64, 66001, 0.0, 0),   # tiles of 128 hidden rows, more tiles than compute units
    (330, 192, 33000, 30.0, 0),
    (160, 64, 33001, 30.0, 0),  # tiles of 256
    (256, 128, 32772, 2.0, 0),
    (250, 128, 32772, 0.0, 1),  # (logits and scales that allow no wide accesses)
    (900, 192, 8450, 0.0, 0),
    (600, 128, 33001, 0.5, 0),  # and more of them than compute units
])
def test_head_of_many_tiles(samplers, m, width, vocab, cap, shift):
    rng = np.random.default_rng(m + width)
    (hc, hs, wc, ws), hv, wv = head_operands(rng, m, width, vocab)
    s = samplers(vocab)
    out = torch.full(((m + 1) * vocab + shift,), 77.0).cuda()[shift:].view(m + 1, vocab)
    if shift:
        hs, ws = (torch.cat([torch.zeros(2, dtype=torch.uint8).cuda(), t.flatten()])[2:].view(t.shape) for t in (hs, ws))
    s.mx_lmhead(hc, hs, wc, ws, softcap_value=cap, out=out[:m])
    some = torch.from_numpy(np.unique(np.concatenate([rng.integers(0, vocab, 500), np.arange(vocab - 300, vocab)])))
    check_logits(out[:m][:, some.cuda()], hv, wv[some], cap)
    assert (out[m] == 77.0).all()
    # the rest: the same sums, whatever rows a call has
    for r in range(0, m, 120):
        n = min(120, m - r)
        few = s.mx_lmhead(hc[r:r + n], hs[r:r + n].contiguous(), wc, ws, softcap_value=cap)
        if n > 64:
            assert torch.equal(out[r:r + n], few)
        else:
            assert ((out[r:r + n] - few).abs() <= 1e-3 * (1 + few.abs())).all()


@pytest.mark.parametrize("m", [3, 100, 256])
def test_head_of_the_largest_vocabulary(samplers, m):
    """Tiles of the logits whose byte offsets reach 2^31 (256 rows)."""
    vocab, width = 2097152, 64
    gen = torch.Generator(device="cuda:0").manual_seed(m)
    code = lambda *shape, lo=0, hi=256: torch.randint(lo, hi, shape, dtype=torch.uint8, device="cuda:0", generator=gen)  # noqa: E731
    hc, hs, wc, ws = code(m, width, hi=0x7f), code(m, 2, lo=124, hi=130), code(vocab, width // 2), code(vocab, 2, lo=118, hi=128)
    out = samplers(vocab).mx_lmhead(hc, hs, wc, ws, softcap_value=0.0)
    some = np.unique(np.concatenate([np.random.default_rng(m).integers(0, vocab, 400), np.arange(260), np.arange(vocab - 260, vocab)]))
    at = torch.from_numpy(some).cuda()
    w = wc[at].cpu().numpy()
    wv = ref.mx_dequantize(np.stack([w & 15, w >> 4], -1).reshape(len(some), width), ws[at].cpu().numpy(), "e2m1")
    hv = ref.mx_dequantize(hc.cpu().numpy(), hs.cpu().numpy(), "e4m3")
    check_logits(out[:, at], torch.from_numpy(hv), torch.from_numpy(wv), 0.0)


def test_a_special_block_stays_in_its_own_logit(samplers):
    rng = np.random.default_rng(12)
    for width in (64, 320, 512):
        ops, hv, wv = head_operands(rng, 40, width, 300, special=True)
        out = samplers(300).mx_lmhead(*ops)
        check_logits(out, hv, wv, 0.0)
        assert out[:, 5].isnan().all() and int(out.isnan().sum()) == 40


def test_norm_head_and_sampler_run_together(samplers):
    """A decode step: the residual's sum, the norm in e4m3, the 4-bit head and the draw."""
    import gsample
    from gsample import runtime as rt

    rng = np.random.default_rng(13)
    m, width, vocab = 6, 256, 4096
    s = samplers(vocab, 8)
    x, res = (torch.from_numpy(rng.normal(0, 1, (m, width)).astype(np.float32)).to(torch.bfloat16).cuda() for _ in range(2))
    w = torch.ones(width, dtype=torch.bfloat16).cuda()
    wc, ws = s.mx_quantize(torch.from_numpy(rng.normal(0, 0.1, (vocab, width)).astype(np.float32)).cuda(), "e2m1")
    codes, scales = torch.empty(m, width, dtype=torch.uint8).cuda(), torch.empty(m, width // 32, dtype=torch.uint8).cuda()
    s.rms_norm(x, w, residual=res, summed=res, codes=codes, scales=scales)
    scratch = torch.empty(m, vocab).cuda()
    cfg = gsample.DecodingConfig(temperature=0.8, topK=40, topP=0.95, repetitionWindow=0)
    conf = np.stack([rt.row_config(cfg, seed=r) for r in range(m)])
    out = s.mx_lmhead_sample(codes, scales, wc, ws, 30.0, scratch, conf)
    logits = s.mx_lmhead(codes, scales, wc, ws, softcap_value=30.0)
    assert torch.equal(logits, scratch)
    again = s.sample(logits, conf)
    assert np.array_equal(out.tokens, again.tokens) and np.array_equal(out.probabilities, again.probabilities)


def test_same_bits_on_another_stream_and_in_a_graph(samplers):
    rng = np.random.default_rng(14)
    ops, _, _ = head_operands(rng, 20, 512, 1000)
    s = samplers(1000)
    want = s.mx_lmhead(*ops, softcap_value=5.0)
    x = torch.from_numpy(rng.normal(0, 1, (20, 512)).astype(np.float32)).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = s.mx_lmhead(*ops, softcap_value=5.0, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    codes, scales = torch.empty(20, 512, dtype=torch.uint8).cuda(), torch.empty(20, 16, dtype=torch.uint8).cuda()
    out = torch.empty_like(want)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        s.mx_quantize(x, "e4m3", codes=codes, scales=scales, stream=side.cuda_stream)
        s.mx_lmhead(codes, scales, *ops[2:], softcap_value=5.0, out=out, stream=side.cuda_stream)
    for _ in range(3):
        x.mul_(1.25)
        out.zero_()
        eager = s.mx_lmhead(*s.mx_quantize(x, "e4m3"), *ops[2:], softcap_value=5.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_refusals(samplers):
    import gsample

    s = samplers(512)
    x = torch.zeros(2, 96).cuda()
    codes, scales = s.mx_quantize(x, "e4m3")
    wc, ws = torch.zeros(512, 48, dtype=torch.uint8).cuda(), torch.zeros(512, 3, dtype=torch.uint8).cuda()
    for call in (
        lambda: s.mx_quantize(torch.zeros(2, 40).cuda(), "e4m3"),
        lambda: s.mx_quantize(x, "e3m2"),
        lambda: s.mx_lmhead(codes, scales, wc, ws),  # 96 is no multiple of 64
        lambda: s.mx_lmhead(codes, scales, wc[:500], ws),
        lambda: s.mx_dequantize(codes, scales[:, :2], "e4m3"),
    ):
        with pytest.raises(gsample.GSampleError):
            call()


@pytest.mark.parametrize("cap", [float("nan"), float("inf"), -float("inf")])
def test_a_cap_that_is_not_finite_is_refused(samplers, cap):
    import gsample

    z = lambda *shape: torch.zeros(*shape, dtype=torch.uint8).cuda()  # noqa: E731
    with pytest.raises(gsample.GSampleError, match="softcap must be finite"):
        samplers(512).mx_lmhead(z(3, 64), z(3, 2), z(512, 32), z(512, 2), softcap_value=cap)
