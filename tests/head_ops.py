"""Plain 64-bit forms of the operators on either side of the head, on the CPU, for the tests of them."""
import numpy as np
import torch

U32, U16 = 2.0 ** -24, 2.0 ** -8  # half a step of binary32 and of bf16, relative to the value
FORMATS = {"e2m1": (2, 0, 1, 6.0), "e4m3": (8, -6, 3, 448.0)}  # emax, least normal exponent, mantissa bits, largest


def norm(x, weight, residual=None, eps=1e-6, offset=0.0):
    """(y, h): h rounded to x's type, y in 64 bits."""
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    hd = h.double()
    r = 1.0 / torch.sqrt((hd * hd).mean(1, keepdim=True) + eps)
    return hd * r * (offset + weight.double()), h


def norm_grad(dy, h, weight, dsummed=None, eps=1e-6, offset=0.0):
    """(dx, dweight, the sum of the magnitudes that dweight adds)."""
    hd, g = h.double(), dy.double() * (offset + weight.double())
    r = 1.0 / torch.sqrt((hd * hd).mean(1, keepdim=True) + eps)
    dx = r * (g - hd * r * r * (g * hd).mean(1, keepdim=True))
    if dsummed is not None:
        dx = dx + dsummed.double()
    terms = dy.double() * hd * r
    return dx, terms.sum(0), terms.abs().sum(0)


def mx_values(fmt):
    """Every value of an element format, by code."""
    emax, emin, bits, top = FORMATS[fmt]
    bias, n = 1 - emin, 16 if fmt == "e2m1" else 256
    out = []
    for c in range(n):
        sign, e, m = c // (n // 2), (c % (n // 2)) >> bits, c % (1 << bits)
        v = (m / (1 << bits)) * 2.0 ** emin if e == 0 else (1 + m / (1 << bits)) * 2.0 ** (e - bias)
        if fmt == "e4m3" and c % 128 == 127:
            v = np.nan
        out.append(-v if sign else v)
    return np.array(out)


def mx_quantize(x, fmt):
    """(codes one a byte, scales) by looking for the nearest value, ties to the even code."""
    emax, _, _, top = FORMATS[fmt]
    values = mx_values(fmt)
    half = values[:len(values) // 2]
    half = half[np.isfinite(half)]
    b = np.asarray(x, dtype=np.float64).reshape(-1, 32)
    amax = np.abs(b).max(1)
    special = ~np.isfinite(amax)
    scales = np.zeros(len(b), dtype=np.int64)
    codes = np.zeros(b.shape, dtype=np.int64)
    for i in range(len(b)):
        if special[i]:
            scales[i] = 255
            codes[i] = 0x7F if fmt == "e4m3" else 0
            continue
        e = int(np.floor(np.log2(amax[i]))) if amax[i] > 0 else -1000
        scales[i] = max(0, e - emax + 127)
        v = np.minimum(np.abs(b[i]) * 2.0 ** (127 - scales[i]), top)
        d = np.abs(v[:, None] - half[None, :])
        near = d.argmin(1)
        nxt = np.minimum(near + 1, len(half) - 1)
        tie = d[np.arange(32), near] == d[np.arange(32), nxt]
        near = np.where(tie & (near % 2 == 1), nxt, near)
        codes[i] = near + np.where(np.signbit(b[i]), len(values) // 2, 0)
    shape = np.asarray(x).shape
    return codes.reshape(shape).astype(np.uint8), scales.reshape(shape[0], -1).astype(np.uint8)


def mx_pack(codes, fmt):
    return codes[:, 0::2] | (codes[:, 1::2] << 4) if fmt == "e2m1" else codes


def mx_dequantize(codes, scales, fmt):
    """codes one a byte; 64-bit values."""
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return (mx_values(fmt)[codes].reshape(codes.shape[0], -1, 32) * s[:, :, None]).reshape(codes.shape)


def capped(z, cap):
    return cap * torch.tanh(z / cap) if cap > 0 else z


def loss(hidden, weight, targets, cap):
    """(loss, lse, g without dloss, the probabilities, which rows are scored) in 64 bits; rows not scored have
    loss 0 and g 0."""
    h, w = hidden.double(), weight.double()
    z = capped(h @ w.T, cap)
    lse = torch.logsumexp(z, 1)
    t = targets.long()
    scored = (t >= 0) & (t < w.shape[0])
    at = torch.where(scored, t, 0)[:, None]
    out = torch.where(scored, lse - z.gather(1, at)[:, 0], 0.0)
    p = torch.exp(z - lse[:, None])
    g = p.scatter_add(1, at, torch.full((h.shape[0], 1), -1.0, dtype=torch.float64))
    if cap > 0:
        g = g * (1 - (z / cap) ** 2)
    g = torch.where(scored[:, None], g, 0.0)
    return out, lse, g, p, scored
