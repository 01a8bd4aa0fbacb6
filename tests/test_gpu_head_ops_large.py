"""The operators on either side of the head at the ends of their sizes: offsets past 2^31, more rows than a launch has
workgroups, the widest rows, 2^20 rows and 2^30 hidden values. The formulas in 64 bits on the GPU, over some rows."""
import pytest
import torch

import head_ops as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def samplers():
    import gsample

    made = {}

    def get(vocab):
        if vocab not in made:
            made[vocab] = gsample.Sampler(vocab_size=vocab, max_rows=1)
        return made[vocab]

    yield get
    for s in made.values():
        s.close()
    made.clear()
    torch.cuda.empty_cache()


def randn(seed, *shape, dtype=torch.bfloat16):
    gen = torch.Generator(device="cuda:0").manual_seed(seed)
    return torch.randn(*shape, device="cuda:0", generator=gen, dtype=dtype)


def some_rows(rows, n=200):
    """The first rows, the last ones, and n others."""
    gen = torch.Generator().manual_seed(rows)
    at = torch.cat([torch.arange(min(rows, 70)), torch.arange(max(0, rows - 70), rows), torch.randint(0, rows, (n,), generator=gen)])
    return at.unique().cuda()


@pytest.mark.parametrize("rows,width,dtype", [
    (4300001, 5, torch.float32),      # past 2^20 workgroups of four rows
    (1100003, 2048, torch.bfloat16),  # past 2^20 of one; 2.25e9 values
])
def test_norm_and_gradient_of_very_many_rows(samplers, rows, width, dtype):
    s = samplers(512)
    x, dy, w = randn(1, rows, width, dtype=dtype), randn(2, rows, width, dtype=dtype), randn(3, width, dtype=torch.float32)
    y = s.rms_norm(x, w, eps=1e-6)
    dx, dw = s.rms_norm_grad(dy, x, w, eps=1e-6)
    half = ref.U16 if dtype == torch.bfloat16 else ref.U32
    at = some_rows(rows)
    hd, gd = x[at].double(), dy[at].double() * w.double()
    r = 1 / torch.sqrt((hd * hd).mean(1, keepdim=True) + 1e-6)
    want = hd * r * w.double()
    assert ((y[at].double() - want).abs() <= (half + 2.0 ** -17) * want.abs() + 1e-37).all()
    want = r * (gd - hd * r * r * (gd * hd).mean(1, keepdim=True))
    parts = r * (gd.abs() + hd.abs() * r * r * (gd * hd).abs().mean(1, keepdim=True))
    assert ((dx[at].double() - want).abs() <= (half + 2.0 ** -17) * want.abs() + 2.0 ** -17 * parts + 1e-37).all()
    want, size = torch.zeros(width, device="cuda:0", dtype=torch.float64), torch.zeros(width, device="cuda:0", dtype=torch.float64)
    for a in range(0, rows, 50000):
        hd, gd = x[a:a + 50000].double(), dy[a:a + 50000].double()
        terms = gd * hd / torch.sqrt((hd * hd).mean(1, keepdim=True) + 1e-6)
        want += terms.sum(0)
        size += terms.abs().sum(0)
    # a share sums up to rows / 768 + 1 rows one after another (four waves' of them joined), the join 24 shares a slice
    # and 32 slices: the roundings in a row, and each term's own 2^-17
    chain = rows // 768 + 4 + 32 + 32
    assert ((dw.double() - want).abs() <= (chain * ref.U32 + 2.0 ** -17) * size + 1e-37).all()


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
def test_blocks_past_2_31_values(samplers, fmt):
    s = samplers(512)
    rows, width = 1100003, 2048
    x = randn(4, rows, width)
    codes, scales = s.mx_quantize(x, fmt)
    values = s.mx_dequantize(codes, scales, fmt)
    for a in (0, 524288, 1048576 - 40, rows - 1000):
        some = s.mx_quantize(x[a:a + 1000].clone(), fmt)
        assert torch.equal(some[0], codes[a:a + 1000]) and torch.equal(some[1], scales[a:a + 1000])
        assert torch.equal(s.mx_dequantize(*some, fmt), values[a:a + 1000])


def test_head_of_more_than_2_31_logits(samplers):
    m, width, vocab = 1100, 64, 2097152
    s = samplers(vocab)
    hc, hs = s.mx_quantize(randn(5, m, width), "e4m3")
    wc, ws = s.mx_quantize(randn(6, vocab, width), "e2m1")
    out = s.mx_lmhead(hc, hs, wc, ws)
    at, of = some_rows(vocab, 2000), some_rows(m, 30)
    h = s.mx_dequantize(hc, hs, "e4m3", dtype=torch.float32)[of].double()
    w = s.mx_dequantize(wc[at], ws[at], "e2m1", dtype=torch.float32).double()
    want = h @ w.T
    # groups of 8 products cut 13 bits below their largest, their sums in binary32
    cut = sum((h[:, None, k:k + 8] * w[None, :, k:k + 8]).abs().amax(2) for k in range(0, width, 8))
    bound = 8 * 2.0 ** -13 * cut + width / 4 * ref.U32 * (h.abs() @ w.abs().T) + 1e-30
    assert ((out[of][:, at].double() - want).abs() <= bound).all()


@pytest.mark.parametrize("rows,width,vocab,cap", [
    (1048576, 64, 300, 0.0),   # the most rows
    (16383, 65536, 300, 30.0), # the widest ones, 2^30 hidden values but for one row
    (5, 65536, 16500, 0.0),    # pieces of the vocabulary because of W's bytes
])
def test_loss_and_gradients_at_the_largest_sizes(samplers, rows, width, vocab, cap):
    s = samplers(vocab)
    h, w = randn(7, rows, width), (2.0 * width ** -0.5 * randn(8, vocab, width)).bfloat16()
    gen = torch.Generator(device="cuda:0").manual_seed(9)
    t = torch.randint(-vocab // 8, vocab, (rows,), device="cuda:0", generator=gen, dtype=torch.int32)
    d = randn(10, rows, dtype=torch.float32)
    loss, lse = s.lmhead_loss(h, w, t, softcap_value=cap)
    dh, dw = s.lmhead_loss_grad(h, w, t, lse, d, softcap_value=cap)
    wd = w.double()
    wa = wd.abs()
    want_dw, dw_bound = torch.zeros_like(wd), torch.zeros_like(wd)
    step = max(1, min(65536, 2 ** 27 // width))
    for a in range(0, rows, step):
        rs = slice(a, a + step)
        hd, td, on = h[rs].double(), t[rs].clamp(min=0).long()[:, None], t[rs] >= 0
        z = ref.capped(hd @ wd.T, cap)
        want_lse = torch.logsumexp(z, 1)
        e = width * 2 * ref.U32 * (hd.abs() @ wa.T).amax(1) + (cap * 2.0 ** -21 if cap > 0 else 0.0)
        assert ((lse[rs].double() - want_lse).abs() <= e + 2.0 ** -20 * (1 + want_lse.abs())).all()
        want = torch.where(on, want_lse - z.gather(1, td)[:, 0], 0.0)
        assert ((loss[rs].double() - want).abs() <= 2 * e + 2.0 ** -19 * (1 + want_lse.abs() + want.abs())).all()
        dd = torch.where(on, d[rs].double(), 0.0)[:, None]
        p = (z - want_lse[:, None]).exp()
        hot = torch.zeros_like(p).scatter_(1, td, 1.0)
        g = (p - hot) * dd * (1 - (z / cap) ** 2 if cap > 0 else 1.0)
        ge = g.abs() * ref.U16 + p * dd.abs() * (2 * e + 2.0 ** -18)[:, None]
        if cap > 0:
            ge += 2.0 ** -20 * (p + hot) * dd.abs()
        want_dh = g @ wd
        bound = (ge + vocab * 2 * ref.U32 * g.abs()) @ wa + ref.U16 * want_dh.abs() + 1e-37
        off = (dh[rs].double() - want_dh).abs()
        assert (off <= bound).all(), float((off / bound).max())
        want_dw += g.T @ hd
        dw_bound += (ge + rows * 2 * ref.U32 * g.abs()).T @ hd.abs()
        print(f"rows from {a} compared", flush=True)
    off, bound = (dw.double() - want_dw).abs(), dw_bound + ref.U16 * want_dw.abs() + 1e-37
    assert (off <= bound).all(), float((off / bound).max())
