"""E4M3 codes and their rows' scales in 64 bits, and when a kernel's codes and
scales agree with them."""
from __future__ import annotations

import torch

MAX = 448.0
U32 = 2.0 ** -24                 # half a step of fp32, relative
CODE = 2.0 ** -4                 # half a step of a normal E4M3 value, relative
CODE_SUB = 2.0 ** -10            # half a step of a subnormal one


def rounded(x: torch.Tensor) -> torch.Tensor:
    """The E4M3 value nearest to x (float64), ties to even, saturated to +-448: from the format, without a
    conversion of torch."""
    a = x.abs().clamp(max=MAX)
    e = torch.floor(torch.log2(a.clamp(min=2.0 ** -6))).clamp(min=-6)
    e = torch.where(torch.pow(2.0, e) > a.clamp(min=2.0 ** -6), e - 1, e)    # log2 next to a power of two
    e = torch.where(torch.pow(2.0, e + 1) <= a, e + 1, e)
    step = torch.pow(2.0, e - 3)
    return torch.sign(x) * (torch.round(a / step) * step).clamp(max=MAX)


def values(codes: torch.Tensor) -> torch.Tensor:
    """What uint8 codes stand for (their scales aside), in float64."""
    return codes.view(torch.float8_e4m3fn).to(torch.float32).double()


def check(codes, scales, rows, off, what=""):
    """codes [..., n] and scales [...] hold the rows (float64 [..., n], known to the relative error `off`): the scale is
    max|row| / 448 and each code the rounding of some value within that error of row / scale."""
    codes, scales, rows = codes.cpu(), scales.cpu().double(), rows.cpu().double()
    top = rows.abs().amax(-1)
    want = top / MAX
    # the row's error, the division's rounding
    assert ((scales - want).abs() <= (off + 2 * U32) * want).all(), \
        (what, ((scales - want).abs() / want.clamp(min=1e-300)).max())
    got = values(codes)
    # the row's error on both sides of the quotient, the reciprocal's and the product's rounding
    rel = 2 * off + 4 * U32
    q = rows / torch.where(want > 0, want, torch.ones_like(want)).unsqueeze(-1)
    lo, hi = rounded(q - q.abs() * rel), rounded(q + q.abs() * rel)
    bad = ~((got >= lo) & (got <= hi))
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4], q[bad][:4])
    # and so the value is within half a step of the row, plus the row's error
    err = (got * scales.unsqueeze(-1) - rows).abs()
    room = (CODE + 2 * rel) * rows.abs() + CODE_SUB * scales.unsqueeze(-1) * (1 + rel)
    assert (err <= room).all(), (what, (err - room).max())
