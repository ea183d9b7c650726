"""Oracle of MXFP4 (test infrastructure, never product): blocks, values and products in 64 bits.

A block of 32 values along the last axis shares 2^e, e = floor(log2(max |x|)) - 2, at least -127; a value becomes the
nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times 2^e, ties to the even code, beyond 6 to 6.  A block with an infinity or
NaN has the byte 255.  Pinned by tests/test_mx4.py.
"""

import torch

BLOCK = 32
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def pow2(e):
    """2^e in float64 for whole e (from the bits: a device's pow may be an ulp off)."""
    return ((e + 1023) << 52).view(torch.float64)


def quantize(x):
    """(codes [..., K / 2], bytes [..., K / 32]) of x [..., K]; codes of a NaN block are not defined."""
    b = x.double().reshape(x.shape[:-1] + (x.shape[-1] // BLOCK, BLOCK))
    top = b.abs().amax(-1)
    finite = torch.isfinite(b).all(-1)
    safe = torch.where(finite & (top > 0), top, torch.ones_like(top))
    e = (torch.frexp(safe).exponent.long() - 1 - 2).clamp(min=-127)
    e = torch.where(top > 0, e, torch.full_like(e, -127))
    a = torch.where(finite[..., None], b, torch.zeros_like(b)).abs() * pow2(-e)[..., None]
    code = torch.zeros(a.shape, dtype=torch.uint8, device=x.device)
    for c in range(1, 8):
        mid = 0.5 * (VALUES[c - 1] + VALUES[c])
        code += ((a >= mid) if c % 2 == 0 else (a > mid)).to(torch.uint8)
    code |= torch.signbit(b).to(torch.uint8) << 3
    code = code.reshape(x.shape)
    scales = torch.where(finite, e + 127, torch.full_like(e, 255)).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scales


def values(codes, scales):
    """[..., K] in float64."""
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), dtype=torch.float64, device=codes.device)
    c = torch.stack((codes & 15, codes >> 4), -1).reshape(scales.shape + (BLOCK,))
    e = scales.long() - 127
    unit = torch.where(scales == 255, torch.full(e.shape, float("nan"), dtype=torch.float64, device=codes.device), pow2(e))
    return (table[c.long()] * unit[..., None]).reshape(codes.shape[:-1] + (2 * codes.shape[-1],))


def quantized(x):
    return values(*quantize(x))


def product(xq, wv, bias=None, weight=None):
    """Sums of xq [M, K] by wv [N, K] (values in float64), and a bound of the error of fp32 sums: every product of two
    values and two scales is exact, and K additions in fp32, truncating at worst, lose 2^-23 of the magnitudes' sum
    each.  ``weight`` [M, 1] multiplies the sums, ``bias`` is added to them: one more rounding of each."""
    K = xq.shape[1]
    y, mag = xq @ wv.t(), xq.abs() @ wv.abs().t()
    err = (K + 8) * 2.0 ** -23 * mag
    if weight is not None:
        y, err = y * weight, err * weight.abs()
        err = err + 2.0 ** -23 * y.abs()
    if bias is not None:
        y = y + bias.double()
        err = err + 2.0 ** -23 * (y.abs() + err)
    return y, err


def gated(y, err, act):
    """act(gate) * up of the halves of y, and the error that the sums' errors and fp32 leave."""
    h = y.shape[-1] // 2
    g, u, eg, eu = y[..., :h], y[..., h:], err[..., :h], err[..., h:]
    f = torch.nn.functional.silu(g) if act == "silu" else torch.nn.functional.gelu(g)
    # Slopes of silu and gelu stay below 1.13; exp, erf, reciprocal and products within 2^-17 of the factors.
    return f * u, 1.13 * eg * (u.abs() + eu) + f.abs() * eu + 2.0 ** -17 * ((f * u).abs() + (g * u).abs() * 2.0 ** -3)
