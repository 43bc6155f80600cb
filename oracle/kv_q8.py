"""8-bit KV-cache oracle (torch on CPU, 64 bits). Test infrastructure only.

Restates the formula of lk_store_kv_q8 (no counterpart in the reference): for
a row x with M = 127 (int8) or 448 (e4m3), a = max(max|x|, 2^-100),
scale = RN32(a / M), r = RN32(M / a), q = rint(x r) or RN_e4m3(RN32(x r)); a row
with an infinity or NaN is q = 0, scale = NaN.
"""

from __future__ import annotations

import numpy as np
import torch

M_OF = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def nearest_e4m3(y: torch.Tensor) -> torch.Tensor:
    """The e4m3 value nearest to y (fp64), ties to even: four bits of
    significand from 2^-6 on, steps of 2^-9 below, at most 448."""
    _, e = torch.frexp(y)                       # |y| in [2^(e-1), 2^e)
    step = torch.exp2((e.double() - 4).clamp_min(-9.0))
    return ((y / step).round() * step).clamp(-448.0, 448.0)


def quantise(x: torch.Tensor, dtype: torch.dtype):
    """x [..., D] -> (q [..., D] fp64 values, scale [...] fp32)."""
    m = M_OF[dtype]
    x = x.double()
    a = x.abs().amax(-1).clamp_min(2.0 ** -100)
    fine = torch.isfinite(x).all(-1)
    a = torch.where(fine, a, torch.ones_like(a)).numpy().astype(np.float32)  # exact: 16-bit values
    scale = torch.from_numpy(a / np.float32(m))
    r = torch.from_numpy(np.float32(m) / a).double()
    y = x * r[..., None]
    q = y.round() if dtype == torch.int8 else nearest_e4m3(y.float().double())
    q = torch.where(fine[..., None], q, torch.zeros_like(q))
    return q, torch.where(fine, scale, torch.full_like(scale, float("nan")))


def rows(data: torch.Tensor, scale, table: torch.Tensor, n: int) -> torch.Tensor:
    """Positions 0..n-1 of one sequence, [n, H_kv, D] fp64: scale * q (scale
    None: a 16-bit cache). data [nb, bs, H_kv, D], scale [nb, H_kv, bs]."""
    bs = data.shape[1]
    pos = torch.arange(n)
    blk, off = table.long()[pos // bs], pos % bs
    x = data[blk, off].to(torch.float32).double()
    return x if scale is None else x * scale[blk, :, off].double()[..., None]
