"""The operators on either side of the head at sizes whose loops take more than one turn."""
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

    def get(vocab):
        if vocab not in made:
            made[vocab] = gsample.Sampler(vocab_size=vocab, max_rows=1)
        return made[vocab]

    yield get
    for s in made.values():
        s.close()


# The bounds of a norm's gradient: one rounding of binary32 products whose sums over the row hold at most width / 8 + 16
# roundings in a row (2^-17 covers widths up to 16384), which stay where the two terms cancel; dweight sums the rows.
@pytest.mark.parametrize("rows,width,dtype", [
    (1153, 4100, "f32"),   # rows too wide to be fetched ahead, two or three of them for a workgroup
    (2311, 4104, "f32"),
    (1160, 8200, "bf16"),
    (1537, 8321, "bf16"),
    (1153, 16384, "f32"),
])
@pytest.mark.parametrize("residual", [True, False])
def test_norm_gradient_of_many_wide_rows(samplers, rows, width, dtype, residual):
    rng = np.random.default_rng(rows + width)
    t = DTYPES[dtype]
    of = lambda: torch.from_numpy(rng.standard_normal((rows, width), dtype=np.float32)).to(t)  # noqa: E731
    h, dy, ds = of(), of(), of() if residual else None
    w = torch.from_numpy(rng.normal(1, 0.3, width).astype(np.float32)).to(t)
    dx, dw = samplers(512).rms_norm_grad(dy.cuda(), h.cuda(), w.cuda(), dsummed=ds.cuda() if residual else None)
    want_dx, want_dw, size = ref.norm_grad(dy, h, w, ds, 1e-6)
    hd = h.double()
    r = 1 / torch.sqrt((hd * hd).mean(1, keepdim=True) + 1e-6)
    g = dy.double() * w.double()
    parts = r * (g.abs() + hd.abs() * r * r * (g * hd).abs().mean(1, keepdim=True))
    if residual:
        parts = parts + ds.double().abs()
    half = ref.U16 if t == torch.bfloat16 else ref.U32
    off = (dx.double().cpu() - want_dx).abs()
    assert (off <= (half + 2.0 ** -17) * want_dx.abs() + 2.0 ** -17 * parts).all(), float(off.max())
    assert ((dw.double().cpu() - want_dw).abs() <= ((rows + 64) * ref.U32 + 2.0 ** -17) * size).all()


@pytest.mark.parametrize("rows,width,vocab,cap", [
    (5000, 320, 30011, 30.0),   # two tiles of columns, pieces of 26624 vocabulary rows
    (9000, 576, 33001, 0.0),    # three of them, and of pieces too
])
def test_loss_gradients_in_pieces_of_the_vocabulary(samplers, rows, width, vocab, cap):
    """The formulas in 64 bits on the GPU (the logits have 150 to 300 million values)."""
    gen = torch.Generator(device="cuda:0").manual_seed(rows)
    randn = lambda *shape: torch.randn(*shape, device="cuda:0", generator=gen)  # noqa: E731
    h, w = randn(rows, width).bfloat16(), (2.0 * width ** -0.5 * randn(vocab, width)).bfloat16()
    t = torch.randint(0, vocab, (rows,), device="cuda:0", generator=gen, dtype=torch.int32)
    t[::5] = -100
    d = randn(rows)
    s = samplers(vocab)
    loss, lse = s.lmhead_loss(h, w, t, softcap_value=cap)
    dh, dw = s.lmhead_loss_grad(h, w, t, lse, d, softcap_value=cap)
    wd, scored = w.double(), t >= 0
    want_dw, dw_bound = torch.zeros_like(wd), torch.zeros_like(wd)
    for a in range(0, rows, 1000):
        rs = slice(a, a + 1000)
        hd, td, on = h[rs].double(), t[rs].clamp(min=0).long()[:, None], scored[rs]
        z = ref.capped(hd @ wd.T, cap)
        want_lse = torch.logsumexp(z, 1)
        # as for smaller vocabularies: a logit's error, that of lse and of the loss, of g, and of the products' sums
        e = width * 2 * ref.U32 * (hd.abs() @ wd.abs().T).amax(1) + (cap * 2.0 ** -21 if cap > 0 else 0.0)
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
        bound = (ge + vocab * 2 * ref.U32 * g.abs()) @ wd.abs() + ref.U16 * want_dh.abs() + 1e-37
        off = (dh[rs].double() - want_dh).abs()
        assert (off <= bound).all(), float((off / bound).max())
        want_dw += g.T @ hd
        dw_bound += (ge + rows * 2 * ref.U32 * g.abs()).T @ hd.abs()
    off, bound = (dw.double() - want_dw).abs(), dw_bound + ref.U16 * want_dw.abs() + 1e-37
    assert (off <= bound).all(), float((off / bound).max())


# The matrix instruction cuts a product 13 bits below the largest of its group of 8 neighbours; the groups' sums are
# added in binary32, a whole step each at most.
@pytest.mark.parametrize("width,vocab,cap", [(64, 300, 0.0), (704, 1000, 30.0), (2048, 515, 5.0)])
def test_a_row_s_logits_in_calls_of_any_size(samplers, width, vocab, cap):
    """Calls of up to 64 rows and of more sum in other orders: either is as near to the exact product."""
    rng = np.random.default_rng(width)
    s, rows = samplers(vocab), 200
    hc, hs = s.mx_quantize(torch.from_numpy(rng.standard_normal((rows, width), dtype=np.float32)).cuda(), "e4m3")
    wc, ws = s.mx_quantize(torch.from_numpy(rng.standard_normal((vocab, width), dtype=np.float32)).cuda() * width ** -0.5, "e2m1")
    h = s.mx_dequantize(hc, hs, "e4m3", dtype=torch.float32).double()
    w = s.mx_dequantize(wc, ws, "e2m1", dtype=torch.float32).double()
    want = ref.capped(h @ w.T, cap)
    cut = sum((h[:, None, k:k + 8] * w[None, :, k:k + 8]).abs().amax(2) for k in range(0, width, 8))
    bound = 8 * 2.0 ** -13 * cut + width / 4 * ref.U32 * (h.abs() @ w.abs().T) + 8 * ref.U32 * want.abs() + 1e-30
    for n in (1, 16, 64, 65, 130, 200):
        got = s.mx_lmhead(hc[:n], hs[:n].contiguous(), wc, ws, softcap_value=cap).double()
        assert ((got - want[:n]).abs() <= bound[:n]).all()
