"""The operators on either side of the lm_head whose speed is measured.

A decode step adds the last block's output to the residual stream, takes the
final norm and multiplies by the head; a training or scoring step does the
same and ends in the cross entropy of the next tokens. `listed()` holds the
calls of both, `draw()` gives others of the same ranges.

  family "norm"       rms_norm with the residual's addition; its output in the
                      input's type, or in e4m3 with a scale for 32 values
  family "norm_grad"  its gradients
  family "mx"         mx_quantize, and the values read back (mx_dequantize)
  family "mx_head"    mx_lmhead: e4m3 hidden states by an e2m1 head
  family "score"      lmhead_loss: the cross entropy of each row's token
  family "train"      lmhead_loss and lmhead_loss_grad

With `own` false `run` computes them from elementary torch operations in 32
bits; with `own` true it makes the framework's calls.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

V = 262144
EPS = 1e-6
IGNORED = -100  # the target of a row that is not scored (a prompt's position, padding)

# element formats of the microscaled types: largest exponent, least normal exponent, mantissa bits, largest value
E2M1 = {"name": "e2m1", "emax": 2, "emin": 0, "bits": 1, "max": 6.0}
E4M3 = {"name": "e4m3", "emax": 8, "emin": -6, "bits": 3, "max": 448.0}
FORMATS = {"e2m1": E2M1, "e4m3": E4M3}
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # the final norm of one decoded token, written as the 4-bit head reads it: a few kilobytes, all latency
        {"name": "norm_token", "family": "norm", "rows": 1, "width": 2048, "dtype": "bf16", "residual": True,
         "out": "mx"},
        # the norm of a training step's positions, the sum kept for the gradient
        {"name": "norm_train", "family": "norm", "rows": 8192, "width": 2048, "dtype": "bf16", "residual": True,
         "out": "same"},
        # its gradient, with the residual stream's own gradient to add, at a ragged number of positions
        {"name": "norm_grad", "family": "norm_grad", "rows": 4099, "width": 3840, "dtype": "bf16", "residual": True},
        # the gradient of a small f32 norm of odd width (a fine-tuning step of a small model)
        {"name": "norm_grad_odd", "family": "norm_grad", "rows": 333, "width": 577, "dtype": "f32",
         "residual": False},
        # a head's weights laid out in 4 bits once at load time, and read back to check them
        {"name": "mx_weights", "family": "mx", "rows": V, "width": 2048, "dtype": "bf16", "format": "e2m1"},
        # a decode batch's hidden states in 8 bits
        {"name": "mx_hidden", "family": "mx", "rows": 37, "width": 1536, "dtype": "f32", "format": "e4m3"},
        # one decoded token through the 4-bit head
        {"name": "mx_head_token", "family": "mx_head", "rows": 1, "width": 1536, "vocab": V, "softcap": 0.0},
        # a server's decode batch through the 4-bit head, with the final softcap
        {"name": "mx_head_batch", "family": "mx_head", "rows": 64, "width": 2048, "vocab": V, "softcap": 30.0},
        # the positions of a prompt (scoring it, checking drafted tokens)
        {"name": "mx_head_prompt", "family": "mx_head", "rows": 512, "width": 2048, "vocab": V, "softcap": 30.0},
        # a scored answer: the loss alone, on a vocabulary that no tile divides
        {"name": "score_answer", "family": "score", "rows": 100, "width": 2048, "vocab": 151643, "softcap": 0.0},
        # a small fine-tuning step of a narrow head, part of its rows not scored
        {"name": "train_small", "family": "train", "rows": 300, "width": 704, "vocab": 50257, "softcap": 0.0},
        # a training step of the whole head: loss and both gradients
        {"name": "train_step", "family": "train", "rows": 4096, "width": 2048, "vocab": V, "softcap": 30.0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _vocab(rng):
    return V if rng.random() < 0.5 else rng.randrange(32001, V)


def draw(rng):
    family = rng.choice(["norm", "norm_grad", "mx", "mx_head", "score", "train"])
    if family in ("norm", "norm_grad"):
        mx = family == "norm" and rng.random() < 0.5
        width = 32 * rng.randrange(2, 257) if mx or rng.random() < 0.6 else rng.randrange(33, 8192)
        case = {"family": family, "rows": _log_int(rng, 1, 16384), "width": width,
                "dtype": rng.choice(["bf16", "bf16", "f32"]), "residual": rng.random() < 0.7}
        return dict(case, out="mx" if mx else "same") if family == "norm" else case
    if family == "mx":
        return {"family": family, "rows": _log_int(rng, 1, 65536), "width": 32 * rng.randrange(2, 129),
                "dtype": rng.choice(["bf16", "f32"]), "format": rng.choice(["e2m1", "e4m3"])}
    softcap = rng.choice([0.0, 30.0])
    rows = _log_int(rng, 1, {"mx_head": 512, "score": 2048, "train": 2048}[family])
    width = 64 * rng.randrange(8, 41) if rows <= 512 else 64 * rng.randrange(8, 33)
    return {"family": family, "rows": rows, "width": width, "vocab": _vocab(rng), "softcap": softcap}


# ---------------------------------------------------------------- inputs

def _randn(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda:0", dtype=dtype)


def _zipf_ids(seed, n, vocab):
    """Zipf(1.1) ids: the ids a text repeats most are the lowest."""
    cdf = np.cumsum(np.arange(1, vocab + 1, dtype=np.float64) ** -1.1)
    ids = np.searchsorted(cdf / cdf[-1], np.random.default_rng(seed).random(n), side="right")
    return np.minimum(ids, vocab - 1).astype(np.int32)


def _stream_like(gen, rows, width, dtype):
    """A residual stream: positions of unequal size, and a few channels far larger than the others."""
    x = _randn(gen, rows, width)
    x *= torch.exp(0.5 * _randn(gen, rows, 1))
    x[:, ::61] *= 12.0
    return x.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda:0").manual_seed(seed)
    family, rows, width = case["family"], case["rows"], case["width"]
    empty = lambda *shape, dtype: torch.empty(*shape, dtype=dtype, device="cuda:0")  # noqa: E731
    s = {"case": case}
    if family in ("norm", "norm_grad"):
        dtype = DTYPES[case["dtype"]]
        s["weight"] = (1.0 + 0.2 * _randn(gen, width)).to(dtype)
        s["x"] = _stream_like(gen, rows, width, dtype)
        s["residual"] = _stream_like(gen, rows, width, dtype) if case["residual"] else None
        # what such a program keeps between steps: the results' memory and the gradient's partial sums
        s["out"] = empty(rows, width, dtype=dtype)
        s["summed"] = empty(rows, width, dtype=dtype)
        if family == "norm_grad":
            s["dy"] = (1e-3 * _randn(gen, rows, width)).to(dtype)
            s["dweight"] = empty(width, dtype=torch.float32)
        elif case["out"] == "mx":
            s["codes"] = empty(rows, width, dtype=torch.uint8)
            s["scales"] = empty(rows, width // 32, dtype=torch.uint8)
            s["values"] = empty(rows, width, dtype=torch.bfloat16)
        return s
    if family == "mx":
        # weights and states whose blocks differ in size
        x = _randn(gen, rows, width)
        x *= 0.02 * torch.exp(0.5 * _randn(gen, rows, 1))
        s["x"] = x.to(DTYPES[case["dtype"]])
        s["codes"] = empty(rows, width // 2 if case["format"] == "e2m1" else width, dtype=torch.uint8)
        s["scales"] = empty(rows, width // 32, dtype=torch.uint8)
        s["values"] = empty(rows, width, dtype=torch.bfloat16)
        return s
    vocab = case["vocab"]
    if family == "mx_head":
        x = _randn(gen, rows, width)
        s["hidden"], s["hidden_scales"] = _quantized(x, E4M3)
        parts = []
        for at in range(0, vocab, 32768):
            w = _randn(gen, min(32768, vocab - at), width)
            parts.append(_quantized(w.mul_(0.03), E2M1))
        s["weight"] = torch.cat([p[0] for p in parts])
        s["weight_scales"] = torch.cat([p[1] for p in parts])
        s["out"] = empty(rows, vocab, dtype=torch.float32)
        return s
    s["hidden"] = _randn(gen, rows, width).to(torch.bfloat16)
    weight = empty(vocab, width, dtype=torch.bfloat16)
    for at in range(0, vocab, 32768):
        weight[at:at + 32768] = _randn(gen, min(32768, vocab - at), width).mul_(0.04)
    s["weight"] = weight
    targets = _zipf_ids(seed, rows, vocab)
    if rows > 8:  # the first positions are a prompt, the last ones padding
        targets[:rows // 8] = IGNORED
        targets[rows - rows // 16:] = IGNORED
    s["targets"] = torch.from_numpy(targets).to("cuda:0")
    s["loss"] = empty(rows, dtype=torch.float32)
    s["lse"] = empty(rows, dtype=torch.float32)
    if family == "train":
        s["dloss"] = torch.full((rows,), 1.0 / max(1, int((targets >= 0).sum())), device="cuda:0")
        s["dhidden"] = torch.empty_like(s["hidden"])
        s["dweight"] = torch.empty_like(weight)
    return s


# ---------------------------------------------------------------- plain forms

def _to_grid(v, f):
    """v rounded to the element format's values, ties to the even mantissa, the largest value kept."""
    e = torch.frexp(v.abs())[1] - 1  # floor(log2 |v|)
    step = torch.ldexp(torch.ones_like(v), torch.clamp(e, min=f["emin"]) - f["bits"])
    return torch.clamp(torch.round(v / step) * step, -f["max"], f["max"])


def _shared_exponent(blocks, f):
    """floor(log2 of the block's largest magnitude) less the format's largest exponent."""
    amax = blocks.abs().amax(-1, keepdim=True)
    return torch.where(amax > 0, torch.clamp(torch.frexp(amax)[1] - 1 - f["emax"], -127, 127), -127)


def _block_values(x, f):
    """x (f32) as the values that its microscaled blocks of 32 stand for."""
    b = x.reshape(x.shape[0], -1, 32)
    e = _shared_exponent(b, f)
    return torch.ldexp(_to_grid(torch.ldexp(b, -e), f), e).reshape(x.shape)


def _quantized(x, f):
    """Codes and scales of x (f32): the inputs of the head's cases."""
    b = x.reshape(x.shape[0], -1, 32)
    e = _shared_exponent(b, f)
    q = _to_grid(torch.ldexp(b, -e), f).reshape(x.shape)
    scales = (e + 127).to(torch.uint8).reshape(x.shape[0], -1)
    if f is E4M3:
        return q.to(torch.float8_e4m3fn).view(torch.uint8), scales
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=x.device)
    code = torch.searchsorted(grid, q.abs().contiguous()).to(torch.uint8) | ((q < 0).to(torch.uint8) << 3)
    return code[:, 0::2] | (code[:, 1::2] << 4), scales


def _values(codes, scales, f, dtype=torch.float32):
    """What codes and scales stand for, in `dtype`."""
    if f is E4M3:
        v = codes.view(torch.float8_e4m3fn).to(dtype)
    else:
        half = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device, dtype=dtype)
        table = torch.cat([half, -half])
        v = torch.stack([table[(codes & 15).long()], table[(codes >> 4).long()]], -1).reshape(codes.shape[0], -1)
    scale = torch.ldexp(torch.ones((), device=codes.device, dtype=dtype), scales.int() - 127)
    return (v.reshape(v.shape[0], -1, 32) * scale[:, :, None]).reshape(v.shape)


def _capped(z, cap):
    return cap * torch.tanh(z / cap) if cap > 0 else z


def _norm_plain(s):
    x, w = s["x"], s["weight"].float()
    # the sum is rounded to its type first: it is what the next block, and the gradient, read
    h = (x.float() + s["residual"].float()).to(x.dtype) if s["residual"] is not None else x
    hf = h.float()
    y = hf * torch.rsqrt(hf.square().mean(-1, keepdim=True) + EPS) * w
    y = _block_values(y, E4M3).to(torch.bfloat16) if s["case"]["out"] == "mx" else y.to(x.dtype)
    return [y, h] if s["residual"] is not None else [y]


def _norm_grad_plain(s):
    h, dy, w = s["x"].float(), s["dy"].float(), s["weight"].float()
    r = torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
    g = dy * w
    dh = r * (g - h * r * r * (g * h).mean(-1, keepdim=True))
    if s["residual"] is not None:
        dh = dh + s["residual"].float()
    return [dh.to(s["x"].dtype), (dy * h * r).sum(0)]


def _loss_plain(s, grads):
    hidden, weight, cap = s["hidden"].float(), s["weight"].float(), s["case"]["softcap"]
    target = s["targets"].long()
    scored = target >= 0
    at = target.clamp(min=0)[:, None]
    z = _capped(hidden @ weight.T, cap)
    top = z.amax(-1, keepdim=True)
    lse = top + (z - top).exp().sum(-1, keepdim=True).log()
    loss = torch.where(scored, (lse - z.gather(1, at))[:, 0], 0.0)
    if not grads:
        return [loss, lse[:, 0]]
    g = (z - lse).exp()
    g.scatter_add_(1, at, torch.full_like(lse, -1.0))
    if cap > 0:
        g *= 1.0 - (z / cap).square()
    g *= torch.where(scored, s["dloss"], 0.0)[:, None]
    return [loss, lse[:, 0], (g @ weight).to(torch.bfloat16), (g.T @ hidden).to(torch.bfloat16)]


def _run_plain(s):
    case = s["case"]
    family = case["family"]
    if family == "norm":
        return _norm_plain(s)
    if family == "norm_grad":
        return _norm_grad_plain(s)
    if family == "mx":
        return [_block_values(s["x"].float(), FORMATS[case["format"]]).to(torch.bfloat16)]
    if family == "mx_head":
        z = _values(s["hidden"], s["hidden_scales"], E4M3) @ _values(s["weight"], s["weight_scales"], E2M1).T
        return [_capped(z, case["softcap"])]
    return _loss_plain(s, family == "train")


# ---------------------------------------------------------------- the framework's calls

_ENGINES = {}


def _engine(vocab):
    """The context of a vocabulary and the one stream that the program works on (not torch's default
    stream, whose null handle the library reads as "the context's own")."""
    if vocab not in _ENGINES:
        path = os.path.join(os.getcwd(), "gemma-webgpu-engine_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import gsample

        if "stream" not in _ENGINES:
            _ENGINES["stream"] = torch.cuda.Stream()
        _ENGINES[vocab] = gsample.Sampler(vocab_size=vocab, max_rows=1)
    return _ENGINES[vocab], _ENGINES["stream"].cuda_stream


def _run_own(s):
    case = s["case"]
    family = case["family"]
    engine, stream = _engine(case.get("vocab", V))
    if family == "norm":
        mx = case["out"] == "mx"
        summed = s["summed"] if case["residual"] else None
        engine.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=EPS, out=None if mx else s["out"],
                        summed=summed, codes=s.get("codes"), scales=s.get("scales"), stream=stream)
        y = s["out"]
        if mx:
            y = engine.mx_dequantize(s["codes"], s["scales"], "e4m3", out=s["values"], stream=stream)
        return [y, summed] if case["residual"] else [y]
    if family == "norm_grad":
        return list(engine.rms_norm_grad(s["dy"], s["x"], s["weight"], dsummed=s["residual"], eps=EPS, dx=s["out"],
                                         dweight=s["dweight"], stream=stream))
    if family == "mx":
        engine.mx_quantize(s["x"], case["format"], codes=s["codes"], scales=s["scales"], stream=stream)
        return [engine.mx_dequantize(s["codes"], s["scales"], case["format"], out=s["values"], stream=stream)]
    if family == "mx_head":
        return [engine.mx_lmhead(s["hidden"], s["hidden_scales"], s["weight"], s["weight_scales"],
                                 softcap_value=case["softcap"], out=s["out"], stream=stream)]
    loss, lse = engine.lmhead_loss(s["hidden"], s["weight"], s["targets"], softcap_value=case["softcap"],
                                   loss=s["loss"], lse=s["lse"], stream=stream)
    if family == "score":
        return [loss, lse]
    dhidden, dweight = engine.lmhead_loss_grad(s["hidden"], s["weight"], s["targets"], lse, s["dloss"],
                                               softcap_value=case["softcap"], dhidden=s["dhidden"],
                                               dweight=s["dweight"], stream=stream)
    return [loss, lse, dhidden, dweight]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    family, rows, width = case["family"], case["rows"], case["width"]
    size = 4 if case.get("dtype") == "f32" else 2
    if family == "norm":
        one = rows * width
        written = one * (1 + 1 / 32) + 2 * one + one * (1 + 1 / 32) if case["out"] == "mx" else one * size
        return {"bytes": one * size * (3 if case["residual"] else 1) + width * size + written, "flops": 4 * one}
    if family == "norm_grad":
        one = rows * width
        return {"bytes": one * size * (4 if case["residual"] else 3) + width * (size + 4), "flops": 12 * one}
    if family == "mx":
        one = rows * width
        coded = one * ((0.5 if case["format"] == "e2m1" else 1.0) + 1 / 32)
        return {"bytes": one * size + 2 * coded + 2 * one, "flops": 4 * one}
    vocab = case["vocab"]
    if family == "mx_head":
        return {"bytes": vocab * width * (0.5 + 1 / 32) + rows * width * (1 + 1 / 32) + 4 * rows * vocab,
                "flops": 2 * rows * width * vocab}
    operands = 2 * (vocab + rows) * width
    if family == "score":
        return {"bytes": operands + 12 * rows, "flops": 2 * rows * width * vocab}
    return {"bytes": 2 * operands + 16 * rows, "flops": 6 * rows * width * vocab}


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_blocks(y, fmt):
    """Each block's values by counting: the nearest of all values of the format, at the block's scale."""
    if fmt == "e2m1":
        grid = [m * 2.0 ** e for e in (0, 1, 2) for m in (1.0, 1.5)] + [0.5, 0.0]
        top = 2
    else:
        grid = [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1] + [m * 2.0 ** -9 for m in range(8)]
        top = 8
    grid = torch.tensor(sorted(set(grid)), dtype=torch.float64, device=y.device)
    middle = (grid[1:] + grid[:-1]) / 2
    b = y.reshape(-1, 32)
    a = b.abs().amax(1)
    e = torch.floor(torch.log2(a.clamp(min=1e-300)))
    e = torch.where(torch.exp2(e) > a, e - 1, e)  # log2 rounded up to a whole number
    e = torch.where(torch.exp2(e + 1) <= a, e + 1, e)
    scale = torch.exp2((e - top).clamp(-127, 127))[:, None]
    v = (b / scale).abs()
    low = torch.searchsorted(middle, v)  # middles below v; one that v equals belongs to the even index
    tie = (low < len(middle)) & (middle[low.clamp(max=len(middle) - 1)] == v)
    index = torch.where(tie & (low % 2 == 1), low + 1, low)
    return (torch.sign(b) * grid[index] * scale).reshape(y.shape)


def exact(case, seed):
    s = prepare(case, seed)
    family = case["family"]
    if family == "norm":
        x, w = s["x"].double(), s["weight"].double()
        h = x
        if s["residual"] is not None:
            h = (x + s["residual"].double()).to(s["x"].dtype).double()
        y = h / torch.sqrt((h ** 2).mean(1, keepdim=True) + EPS) * w
        if case["out"] == "mx":
            y = _exact_blocks(y, "e4m3")
        return [y, h] if s["residual"] is not None else [y]
    if family == "norm_grad":
        h, dy, w = s["x"].double(), s["dy"].double(), s["weight"].double()
        n = h.shape[1]
        rms = torch.sqrt((h ** 2).sum(1, keepdim=True) / n + EPS)
        unit = h / rms
        dh = (dy * w - unit * ((dy * w * unit).sum(1, keepdim=True) / n)) / rms
        if s["residual"] is not None:
            dh = dh + s["residual"].double()
        return [dh, torch.einsum("rc,rc->c", dy, unit)]
    if family == "mx":
        parts = [_exact_blocks(p.double(), case["format"]).to(torch.bfloat16) for p in s["x"].split(16384)]
        return [torch.cat(parts)]  # every value of a block fits 16 bits
    cap = case["softcap"]
    if family == "mx_head":
        hidden = _values(s["hidden"], s["hidden_scales"], E4M3, torch.float64)
        z = hidden @ _values(s["weight"], s["weight_scales"], E2M1, torch.float64).t()
        return [cap * torch.tanh(z / cap) if cap > 0 else z]
    hidden, weight, targets = s["hidden"].double(), s["weight"].double(), s["targets"].long()
    loss, lse, dhidden, dweight = [], [], [], torch.zeros_like(weight) if family == "train" else None
    for h, t, d in zip(hidden.split(1024), targets.split(1024),
                       s["dloss"].double().split(1024) if family == "train" else [None] * 2 ** 20):
        u = h @ weight.t()
        z = cap * torch.tanh(u / cap) if cap > 0 else u
        total = torch.logsumexp(z, 1)
        rows = torch.nonzero(t >= 0)[:, 0]
        one = torch.zeros_like(total)
        one[rows] = total[rows] - z[rows, t[rows]]
        loss.append(one)
        lse.append(total)
        if family == "train":
            p = torch.exp(z - total[:, None])
            p[rows, t[rows]] -= 1.0
            if cap > 0:
                p /= torch.cosh(u / cap) ** 2
            factor = torch.zeros_like(total)
            factor[rows] = d[rows]
            p *= factor[:, None]
            dhidden.append(p @ weight)
            dweight += p.t() @ h
    if family == "score":
        return [torch.cat(loss), torch.cat(lse)]
    return [torch.cat(loss), torch.cat(lse), torch.cat(dhidden), dweight]
