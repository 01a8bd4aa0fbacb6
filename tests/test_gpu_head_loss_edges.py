"""The head's cross entropy at the ends of its arguments: softcaps far from the logits' size, gradients that are not
finite, certain targets, results in place of operands."""
import numpy as np
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


def operands(rng, rows, width, vocab, scale=1.0, shift=0.0):
    """hidden, weight and targets whose logits spread by `scale` about `shift`."""
    h = torch.from_numpy(rng.normal(0, 1, (rows, width)).astype(np.float32))
    w = torch.from_numpy(rng.normal(0, scale * width ** -0.5, (vocab, width)).astype(np.float32))
    h[:, 0], w[:, 0] = 1.0, shift
    t = torch.from_numpy(rng.integers(0, vocab, rows).astype(np.int32))
    return h.to(torch.bfloat16), w.to(torch.bfloat16), t


# A logit's error: `width` products in binary32, a whole step each where the matrix core truncates; then the cap, whose
# quotient, series and product are within a few steps of the capped value below 5/8 of the cap, and past it within
# 2e-7 of the cap, itself less than twice the value: 2^-20 of the value in either case (and of the cap, 2^-21, where
# the cap is small). The loss and lse carry the largest of the row, the exponentials' and the sum's roundings 2^-20.
def logit_error(h, w, z):
    return h.shape[1] * 2 * ref.U32 * (h.double().abs() @ w.double().abs().T).amax(1) + 2.0 ** -20 * z.abs().amax(1)


def check(s, h, w, t, cap):
    dev = [v.cuda() for v in (h, w, t)]
    loss, lse = s.lmhead_loss(*dev, softcap_value=cap)
    want_loss, want_lse, g, prob, scored = ref.loss(h, w, t, cap)
    e = logit_error(h, w, ref.capped(h.double() @ w.double().T, cap))
    assert ((lse.double().cpu() - want_lse).abs() <= e + 2.0 ** -20 * (1 + want_lse.abs())).all(), (lse, want_lse)
    assert ((loss.double().cpu() - want_loss).abs() <= 2 * e + 2.0 ** -19 * (1 + want_lse.abs() + want_loss.abs())).all()
    d = torch.from_numpy(np.random.default_rng(1).normal(0, 1, h.shape[0]).astype(np.float32))
    dh, dw = s.lmhead_loss_grad(*dev, lse, d.cuda(), softcap_value=cap)
    # g: the probability carries the logit's and lse's error, (1 - t^2) that of tanh, 2^-20 on |p - [target]|; then a
    # rounding to bf16 (and one of dloss over the largest of them, 2^-23, among the 2^-18)
    gd = g * d.double()[:, None]
    pd = prob * d.double().abs()[:, None]
    hot = torch.zeros_like(pd).scatter_(1, t.long()[:, None], d.double().abs()[:, None])
    ge = gd.abs() * ref.U16 + pd * (2 * e + 2.0 ** -18)[:, None] + 2.0 ** -20 * (pd + hot)
    for got, want, bound in (
            (dh, gd @ w.double(), ge @ w.double().abs() + w.shape[0] * 2 * ref.U32 * (gd.abs() @ w.double().abs())),
            (dw, gd.T @ h.double(), ge.T @ h.double().abs() + len(h) * 2 * ref.U32 * (gd.abs().T @ h.double().abs()))):
        off = (got.double().cpu() - want).abs()
        assert (off <= bound + ref.U16 * want.abs() + 1e-37).all(), float((off / (bound + ref.U16 * want.abs() + 1e-37)).max())


@pytest.mark.parametrize("rows", [3, 70, 200])
@pytest.mark.parametrize("cap", [1.5e3, 1e5, 1e8, 1e10, 1e20, 1e38])
@pytest.mark.parametrize("shift", [0.0, 100.0, -120.0])
def test_caps_far_above_the_logits(samplers, rows, cap, shift):
    rng = np.random.default_rng(rows)
    check(samplers(700), *operands(rng, rows, 128, 700, 3.0, shift), cap)


@pytest.mark.parametrize("rows", [3, 70, 200])
@pytest.mark.parametrize("cap", [2.0 ** -5, 1e-3, 1e-10, 1e-20, 1e-25, 1e-38, 1e-42, 3.4e38])
def test_caps_far_below_the_logits_and_at_the_end_of_the_range(samplers, rows, cap):
    """Below the logits most slopes are 0; a row of zeros has logits of 0, whose slope is 1 whatever the cap."""
    rng = np.random.default_rng(rows + 1)
    h, w, t = operands(rng, rows, 128, 700, 3.0)
    h[1] = 0.0
    check(samplers(700), h, w, t, cap)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_gradient_that_is_not_finite_stays_in_its_row(samplers, bad):
    rng = np.random.default_rng(31)
    s = samplers(700)
    h, w, t = (v.cuda() for v in operands(rng, 150, 128, 700, 2.0))
    t[7] = -1
    for cap in (0.0, 20.0):
        _, lse = s.lmhead_loss(h, w, t, softcap_value=cap)
        d = torch.from_numpy(rng.normal(0, 1, 150).astype(np.float32)).cuda()
        d[40], d[149] = 0.0, 0.0
        want, _ = s.lmhead_loss_grad(h, w, t, lse, d, softcap_value=cap)
        d[40], d[149], d[7] = bad, bad, bad
        got, dw = s.lmhead_loss_grad(h, w, t, lse, d, softcap_value=cap)
        alone, _ = s.lmhead_loss_grad(h, w, t, lse, d, softcap_value=cap, weight_grad=False)
        keep = [i for i in range(150) if i not in (40, 149)]
        for dh in (got, alone):
            assert torch.equal(dh[keep], want[keep])
            assert not dh[40].isfinite().any() and not dh[149].isfinite().any()
        assert not dw.isfinite().any()  # every vocabulary row takes its share of those rows
        d[:] = bad  # no row is finite
        dh, _ = s.lmhead_loss_grad(h, w, t, lse, d, softcap_value=cap)
        assert (dh[7] == 0).all() and not torch.cat([dh[:7], dh[8:]]).isfinite().any()


@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_a_certain_token_s_loss_is_never_below_zero(samplers, cap):
    """The target's logit alone makes up the sum of exponentials, so the loss is 0 but for roundings."""
    rng = np.random.default_rng(32)
    h, w, t = operands(rng, 400, 704, 700, 1.0)
    w *= 0.01
    for m in range(400):  # row m mod 100 of W points along hidden row m
        t[m] = m % 100
        h[m] = h[m % 100]
        w[m % 100] = h[m % 100] * (28.0 / 704 if cap == 0.0 else 1.0)
    loss, lse = samplers(700).lmhead_loss(*(v.cuda() for v in (h, w, t)), softcap_value=cap)
    want, _, _, _, _ = ref.loss(h, w, t, cap)
    e = logit_error(h, w, ref.capped(h.double() @ w.double().T, cap))
    assert (loss >= 0).all(), float(loss.min())
    assert ((loss.double().cpu() - want).abs() <= 2 * e + 2.0 ** -19 * (1 + lse.double().cpu().abs())).all()


@pytest.mark.parametrize("rows,width,vocab", [(60, 128, 700), (5000, 64, 30011)])  # (the second in pieces of the vocabulary)
def test_gradients_in_place_of_their_operands(samplers, rows, width, vocab):
    rng = np.random.default_rng(33)
    s = samplers(vocab)
    h, w, t = (v.cuda() for v in operands(rng, rows, width, vocab, 2.0))
    t[::7] = -1
    d = torch.from_numpy(rng.normal(0, 1, rows).astype(np.float32)).cuda()
    _, lse = s.lmhead_loss(h, w, t, softcap_value=20.0)
    want = s.lmhead_loss_grad(h, w, t, lse, d, softcap_value=20.0)
    got = s.lmhead_loss_grad(h, w, t, lse, d, softcap_value=20.0, dhidden=h, dweight=w)
    assert got[0].data_ptr() == h.data_ptr() and got[1].data_ptr() == w.data_ptr()
    assert torch.equal(h, want[0]) and torch.equal(w, want[1])


@pytest.mark.parametrize("rows,width", [(2500, 64), (2500, 4200), (5, 577)])
def test_norm_gradients_in_place_of_their_inputs(samplers, rows, width):
    rng = np.random.default_rng(34)
    s = samplers(700)
    for dtype in (torch.float32, torch.bfloat16):
        of = lambda: torch.from_numpy(rng.standard_normal((rows, width), dtype=np.float32)).to(dtype).cuda()  # noqa: E731
        h, dy, ds, w = of(), of(), of(), torch.from_numpy(rng.normal(1, 0.2, width).astype(np.float32)).cuda()
        want, want_dw = s.rms_norm_grad(dy, h, w, dsummed=ds)
        for place in range(3):
            ops = [v.clone() for v in (dy, h, ds)]
            v = w.clone()
            s.rms_norm_grad(ops[0], ops[1], v, dsummed=ops[2], dx=ops[place], dweight=v)
            assert torch.equal(ops[place], want) and torch.equal(v, want_dw)
