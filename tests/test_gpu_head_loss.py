"""The head's cross entropy and its gradients against the plain form in 64 bits."""
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


def operands(rng, rows, width, vocab, scale=1.0):
    h = torch.from_numpy(rng.normal(0, 1, (rows, width)).astype(np.float32)).to(torch.bfloat16)
    w = torch.from_numpy((rng.normal(0, scale * width ** -0.5, (vocab, width))).astype(np.float32)).to(torch.bfloat16)
    t = rng.integers(0, vocab, rows).astype(np.int32)
    if rows > 2:
        t[rng.integers(0, rows, rows // 4 + 1)] = -100
        t[0], t[-1] = vocab - 1, vocab
    return h, w, torch.from_numpy(t)


# A logit's error: `width` products in binary32, a whole step each where the
# matrix core truncates, and 2^-21 of the cap for the tanh. The loss and lse
# carry the largest of the row, the exponentials' and the sum's (2^-20 covers
# an exponent's argument of up to 128 and a thousand terms a lane in pairs).
def logit_error(h, w, cap):
    e = h.shape[1] * 2 * ref.U32 * (h.double().abs() @ w.double().abs().T).amax(1)
    return e + (cap * 2.0 ** -21 if cap > 0 else 0.0)


def check(s, h, w, t, cap, dloss=None, rows=None):
    dev = [v.cuda() for v in (h, w, t)]
    loss, lse = s.lmhead_loss(*dev, softcap_value=cap)
    want_loss, want_lse, g, prob, scored = ref.loss(h, w, t, cap)
    e = logit_error(h, w, cap)
    assert ((lse.double().cpu() - want_lse).abs() <= e + 2.0 ** -20 * (1 + want_lse.abs())).all()
    assert ((loss.double().cpu() - want_loss).abs() <= 2 * e + 2.0 ** -19 * (1 + want_lse.abs() + want_loss.abs())).all()
    assert (loss.cpu()[~scored] == 0).all()
    d = torch.from_numpy(np.random.default_rng(1).normal(0, 1, h.shape[0]).astype(np.float32)) if dloss is None else dloss
    dh, dw = s.lmhead_loss_grad(*dev, lse, d.cuda(), softcap_value=cap)
    gd = torch.where(scored[:, None], g * d.double()[:, None], 0.0)
    # g: the probability carries the logit's and lse's error; (1 - t^2) that of tanh, 2^-20, on |p - [target]| <= 1;
    # then one rounding to bf16
    pd = prob * d.double().abs()[:, None]
    ge = gd.abs() * ref.U16 + pd * (2 * e + 2.0 ** -18)[:, None]
    if cap > 0:
        hot = torch.zeros_like(pd).scatter_(1, torch.where(scored, t.long(), 0)[:, None], d.double().abs()[:, None])
        ge = ge + 2.0 ** -20 * (pd + hot)
    ge = torch.where(scored[:, None], ge, 0.0)
    n = h.shape[0]
    for got, want, bound in ((dh, gd @ w.double(), ge @ w.double().abs() + w.shape[0] * 2 * ref.U32 * (gd.abs() @ w.double().abs())),
                             (dw, gd.T @ h.double(), ge.T @ h.double().abs() + n * 2 * ref.U32 * (gd.abs().T @ h.double().abs()))):
        bound = bound + ref.U16 * want.abs() + 1e-37
        off = (got.double().cpu() - want).abs()
        assert (off <= bound).all(), (int((off > bound).sum()), float((off / bound).max()), torch.nonzero(off > bound)[:4].tolist())
    return loss, lse, dh, dw


@pytest.mark.parametrize("rows", [1, 2, 33, 64, 65, 100, 128, 129, 257, 300])
@pytest.mark.parametrize("width,vocab,cap", [(64, 1, 0.0), (64, 300, 30.0), (192, 513, 0.0), (704, 1000, 3.0), (320, 256, 0.0)])
def test_loss_and_gradients_match_the_formulas(samplers, rows, width, vocab, cap):
    rng = np.random.default_rng(rows + width)
    check(samplers(vocab), *operands(rng, rows, width, vocab, 2.0), cap)


def test_a_large_vocabulary_in_pieces(samplers):
    """More rows than a piece's gradients have room for at this vocabulary: several pieces, the last one short."""
    rng = np.random.default_rng(21)
    rows, width, vocab = 5000, 64, 30011  # 5000 x 30208 bf16 gradients are 302 MB
    h, w, t = operands(rng, rows, width, vocab, 2.0)
    check(samplers(vocab), h, w, t, 30.0)


@pytest.mark.parametrize("rows,width,vocab,cap", [
    (3, 64, 66000, 0.0),     # more tiles of 256 than compute units: smaller ones, the last one ragged or not
    (70, 64, 66001, 30.0),
    (128, 128, 90112, 3.0),
    (100, 64, 151643, 0.0),
    (130, 64, 66016, 0.0),
])
def test_a_vocabulary_of_more_tiles_than_compute_units(samplers, rows, width, vocab, cap):
    rng = np.random.default_rng(rows + vocab)
    h, w, t = operands(rng, rows, width, vocab, 2.0)
    h[0] *= -4.0  # a row whose logits are large on both sides
    dev = [v.cuda() for v in (h, w, t)]
    loss, lse = samplers(vocab).lmhead_loss(*dev, softcap_value=cap)
    z = ref.capped(h.double() @ w.double().T, cap)
    want = torch.logsumexp(z, 1)
    e = logit_error(h, w, cap)
    assert ((lse.double().cpu() - want).abs() <= e + 2.0 ** -20 * (1 + want.abs())).all()
    scored = (t >= 0) & (t < vocab)
    want_loss = torch.where(scored, want - z[torch.arange(rows), torch.where(scored, t.long(), 0)], 0.0)
    assert ((loss.double().cpu() - want_loss).abs() <= 2 * e + 2.0 ** -19 * (1 + want.abs() + want_loss.abs())).all()


def test_the_largest_vocabulary(samplers):
    check(samplers(2097152), *operands(np.random.default_rng(27), 3, 64, 2097152, 2.0), 30.0)


def test_confident_rows_and_far_logits(samplers):
    """Targets whose probability is near one, and logits of +-100 without a cap."""
    rng = np.random.default_rng(22)
    vocab, width = 700, 128
    h, w, t = operands(rng, 90, width, vocab, 12.0)
    t = torch.from_numpy((h.double() @ w.double().T).argmax(1).numpy().astype(np.int32))
    check(samplers(vocab), h, w, t, 0.0)
    check(samplers(vocab), h, w, t, 15.0)


def test_rows_not_scored_add_nothing_even_when_not_finite(samplers):
    rng = np.random.default_rng(23)
    vocab, width = 520, 128
    s = samplers(vocab)
    h, w, t = operands(rng, 70, width, vocab)
    t[:] = torch.from_numpy(rng.integers(0, vocab, 70).astype(np.int32))
    t[10:20], t[69] = -1, 2 ** 31 - 1
    d = torch.ones(70)
    clean = check(s, h, w, t, 0.0, d)
    h[10:20] = float("nan")
    h[69] = float("inf")
    d[10:20] = float("nan")
    dev = [v.cuda() for v in (h, w, t)]
    loss, lse = s.lmhead_loss(*dev)
    dh, dw = s.lmhead_loss_grad(*dev, lse, d.cuda())
    keep = [i for i in range(70) if not (10 <= i < 20 or i == 69)]
    assert torch.equal(loss[keep], clean[0][keep]) and (loss[10:20] == 0).all() and loss[69] == 0
    assert torch.equal(dh[keep], clean[2][keep]) and (dh[10:20] == 0).all() and torch.equal(dw, clean[3])
    t[:] = -100  # nothing is scored
    dh, dw = s.lmhead_loss_grad(h.cuda(), w.cuda(), t.cuda(), lse, d.cuda())
    assert (dh == 0).all() and (dw == 0).all()


def test_one_gradient_alone_and_no_rows(samplers):
    rng = np.random.default_rng(24)
    s = samplers(600)
    h, w, t = (v.cuda() for v in operands(rng, 40, 128, 600))
    loss, lse = s.lmhead_loss(h, w, t)
    d = torch.ones(40).cuda()
    dh, dw = s.lmhead_loss_grad(h, w, t, lse, d)
    a = s.lmhead_loss_grad(h, w, t, lse, d, weight_grad=False)
    b = s.lmhead_loss_grad(h, w, t, lse, d, hidden_grad=False)
    assert a[1] is None and b[0] is None and torch.equal(a[0], dh) and torch.equal(b[1], dw)
    e = h[:0]
    loss, lse = s.lmhead_loss(e, w, t[:0])
    dh, dw = s.lmhead_loss_grad(e, w, t[:0], lse, d[:0], dweight=torch.ones_like(w))
    assert loss.shape == (0,) and dh.shape == (0, 128) and (dw == 0).all()


def test_gradient_against_differences(samplers):
    rng = np.random.default_rng(25)
    h, w, t = operands(rng, 20, 64, 300, 2.0)
    s = samplers(300)
    dev = [v.cuda() for v in (h, w, t)]
    _, lse = s.lmhead_loss(*dev, softcap_value=4.0)
    d = torch.from_numpy(rng.normal(0, 1, 20).astype(np.float32))
    dh, dw = s.lmhead_loss_grad(*dev, lse, d.cuda(), softcap_value=4.0)
    f = lambda a, b: float((ref.loss(a, b, t, 4.0)[0] * d.double()).sum())  # noqa: E731
    e = 1e-5
    dir_h, dir_w = (torch.from_numpy(rng.normal(0, 1, v.shape)) for v in (h, w))
    for got, along, by in (
            (dh, dir_h, (f(h.double() + e * dir_h, w) - f(h.double() - e * dir_h, w)) / (2 * e)),
            (dw, dir_w, (f(h, w.double() + e * dir_w) - f(h, w.double() - e * dir_w)) / (2 * e))):
        # every value off by at most 2^-7 of what it sums: far less than this in sum
        assert abs(float((got.double().cpu() * along).sum()) - by) <= 2.0 ** -7 * float((got.double().cpu() * along).abs().sum())


def test_loss_is_what_the_head_and_token_log_probability_give(samplers):
    """The framework's own path over the same operands: the lm_head's logits, then tokenLogProbability."""
    rng = np.random.default_rng(26)
    vocab, width = 5000, 256
    s = samplers(vocab)
    h, w, t = operands(rng, 12, width, vocab, 3.0)
    t = torch.from_numpy(rng.integers(0, vocab, 12).astype(np.int32))
    dev = [v.cuda() for v in (h, w, t)]
    loss, _ = s.lmhead_loss(*dev, softcap_value=30.0)
    logits = s.lmhead(dev[0], dev[1], 30.0)
    by_logits = -s.token_log_probability(logits, t.numpy())
    e = 4 * logit_error(h, w, 30.0).numpy() + 2.0 ** -18 * (1 + by_logits)
    assert (np.abs(loss.cpu().numpy() - by_logits) <= e).all()


def test_norm_loss_and_gradients_run_together(samplers):
    """A training step's end: sum and norm, the loss, its gradients, the norm's."""
    rng = np.random.default_rng(27)
    vocab, width, rows = 900, 192, 75
    s = samplers(vocab)
    x, res = (torch.from_numpy(rng.normal(0, 1, (rows, width)).astype(np.float32)).to(torch.bfloat16) for _ in range(2))
    nw = torch.from_numpy(rng.normal(1, 0.1, width).astype(np.float32))
    _, w, t = operands(rng, rows, width, vocab, 2.0)
    h = torch.empty(rows, width, dtype=torch.bfloat16).cuda()
    y = s.rms_norm(x.cuda(), nw.cuda(), residual=res.cuda(), summed=h)
    loss, lse, dy, dw = check(s, y.cpu(), w, t, 20.0, torch.full((rows,), 1.0 / rows))
    dx, dnw = s.rms_norm_grad(dy, h, nw.cuda())
    want_dx, want_dnw, size = ref.norm_grad(dy.cpu(), h.cpu(), nw)
    assert ((dx.double().cpu() - want_dx).abs() <= ref.U16 * want_dx.abs() + 2.0 ** -15 * want_dx.abs().amax()).all()
    assert ((dnw.double().cpu() - want_dnw).abs() <= 2.0 ** -15 * size).all()


def test_same_bits_every_time_on_another_stream_and_in_a_graph(samplers):
    rng = np.random.default_rng(28)
    s = samplers(1500)
    h, w, t = (v.cuda() for v in operands(rng, 150, 256, 1500))
    d = torch.full((150,), 0.01).cuda()
    loss, lse = s.lmhead_loss(h, w, t, softcap_value=30.0)
    dh, dw = s.lmhead_loss_grad(h, w, t, lse, d, softcap_value=30.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    loss2, lse2 = s.lmhead_loss(h, w, t, softcap_value=30.0, stream=side.cuda_stream)
    dh2, dw2 = s.lmhead_loss_grad(h, w, t, lse2, d, softcap_value=30.0, stream=side.cuda_stream)
    side.synchronize()
    for a, b in ((loss, loss2), (lse, lse2), (dh, dh2), (dw, dw2)):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    outs = [torch.empty_like(v) for v in (loss, lse, dh, dw)]
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        s.lmhead_loss(h, w, t, softcap_value=30.0, loss=outs[0], lse=outs[1], stream=side.cuda_stream)
        s.lmhead_loss_grad(h, w, t, outs[1], d, softcap_value=30.0, dhidden=outs[2], dweight=outs[3],
                           stream=side.cuda_stream)
    for _ in range(3):
        h.copy_(torch.roll(h, 1, 0))
        for v in outs:
            v.zero_()
        loss, lse = s.lmhead_loss(h, w, t, softcap_value=30.0)
        dh, dw = s.lmhead_loss_grad(h, w, t, lse, d, softcap_value=30.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, (loss, lse, dh, dw)):
            assert torch.equal(a, b)


def test_work_memory_is_not_grown_under_capture(samplers):
    import gsample

    s = gsample.Sampler(vocab_size=300, max_rows=1)
    try:
        rng = np.random.default_rng(29)
        h, w, t = (v.cuda() for v in operands(rng, 10, 64, 300))
        out = [torch.empty(10).cuda() for _ in range(2)]
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        seen = []
        with torch.cuda.graph(graph, stream=side):
            out[0].zero_()
            try:
                s.lmhead_loss(h, w, t, loss=out[0], lse=out[1], stream=side.cuda_stream)
            except gsample.GSampleError as e:
                seen.append(str(e))
        assert seen and "capture" in seen[0]
        s.lmhead_loss(h, w, t, loss=out[0], lse=out[1])  # and the context still works
        assert torch.isfinite(out[0]).all()
    finally:
        s.close()


def test_refusals(samplers):
    import gsample

    s = samplers(300)
    h = torch.zeros(4, 96, dtype=torch.bfloat16).cuda()
    w = torch.zeros(300, 96, dtype=torch.bfloat16).cuda()
    t = torch.zeros(4, dtype=torch.int32).cuda()
    f = torch.zeros(4).cuda()
    for call in (
        lambda: s.lmhead_loss(h, w, t),  # 96 is no multiple of 64
        lambda: s.lmhead_loss(h[:, :64].contiguous(), w[:200, :64].contiguous(), t),
        lambda: s.lmhead_loss(h[:, :64].contiguous(), w[:, :64].contiguous(), t.long()),
        lambda: s.lmhead_loss_grad(h[:, :64].contiguous(), w[:, :64].contiguous(), t, f, f, hidden_grad=False, weight_grad=False),
    ):
        with pytest.raises(gsample.GSampleError):
            call()


@pytest.mark.parametrize("cap", [float("nan"), float("inf"), -float("inf")])
def test_a_cap_that_is_not_finite_is_refused(samplers, cap):
    import gsample

    h, w = torch.zeros(4, 64, dtype=torch.bfloat16).cuda(), torch.zeros(300, 64, dtype=torch.bfloat16).cuda()
    t, f = torch.zeros(4, dtype=torch.int32).cuda(), torch.zeros(4).cuda()
    with pytest.raises(gsample.GSampleError, match="softcap must be finite"):
        samplers(300).lmhead_loss(h, w, t, softcap_value=cap)
    with pytest.raises(gsample.GSampleError, match="softcap must be finite"):
        samplers(300).lmhead_loss_grad(h, w, t, f, f, softcap_value=cap)
