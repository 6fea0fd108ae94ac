"""Plain float64 implementation of the 8-bit block format and of the operators on it (any device), for the tests."""
import math

import torch

# name: (torch type, mantissa bits, exponent of the smallest normal value, exponent of the largest value 1.75 * 2^top)
FORMATS = {"e4m3": (torch.float8_e4m3fn, 3, -6, 8), "e5m2": (torch.float8_e5m2, 2, -14, 15)}


def two_to(e):
    """2^e in float64, exact (by its bits), e an integer tensor in the normal range."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def split(x, fmt, keep_positive=False):
    """(codes' values in float64 [rows, cols], blocks' exponents [rows, blocks])."""
    _, bits, low, top = FORMATS[fmt]
    x = x.double()
    rows, cols = x.shape
    codes, exps = torch.zeros_like(x), []
    for at in range(0, cols, 128):
        b = x[:, at:at + 128]
        m = torch.where(b.isfinite(), b.abs(), 0.0).amax(1)
        f, q = torch.frexp(m)                                         # m = f 2^q, 0.5 <= f < 1
        e = torch.where(m > 0, q - 1 - top + (f > 0.875).int(), -126).clamp(min=-126)
        v = b * two_to(-e)[:, None]
        fin = torch.where(v.isfinite(), v, 0.0)
        _, q = torch.frexp(fin)
        step = two_to(torch.where(fin != 0, q - 1, low).clamp(min=low) - bits)
        r = torch.round(fin / step) * step
        if keep_positive:
            r = torch.where((r == 0) & (v > 0), 2.0 ** (low - bits), r)
        r = torch.where(v.isfinite(), r, v if fmt == "e5m2" else torch.full_like(v, math.nan))
        codes[:, at:at + 128] = r
        exps.append(e)
    return codes, torch.stack(exps, 1)


def values(x, fmt="e4m3", keep_positive=False):
    codes, e = split(x, fmt, keep_positive)
    return codes * two_to(e).repeat_interleave(128, 1)[:, :x.shape[1]]


def of(q):
    """The values of a Block8, from its codes and scales by torch's own conversions."""
    s = q.scales.view(torch.uint8).int() - 127
    return q.codes.float().double() * two_to(s).repeat_interleave(128, 1)[:, :q.codes.shape[1]]
