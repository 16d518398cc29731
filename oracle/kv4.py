"""The 4-bit key/value cache in float64, written from the format's definition
(include/forgeml_b200.h), one group at a time.

stands_for(x): what rows x [..., D] read back as, before the rounding to x's
dtype.  attention(): q [B,T,QH,D] over rows 0..start+t of those numbers.
"""

from __future__ import annotations

import math

import torch


def stands_for(x: torch.Tensor) -> torch.Tensor:
    x = x.detach().cpu()
    out = torch.empty(x.shape, dtype=torch.float64)
    for c0 in range(0, x.shape[-1], 32):
        g = x[..., c0:c0 + 32].double()
        z, top = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
        s = ((top - z) / 15).to(x.dtype).double()
        code = ((g - z) / s.masked_fill(s == 0, 1.0)).round().clamp(0, 15)
        code = code.masked_fill(s == 0, 0.0)
        val = z + code * s
        finite = g.isfinite().all(-1, keepdim=True)
        out[..., c0:c0 + 32] = torch.where(finite, val, torch.full_like(val, math.nan))
    return out


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, starts) -> torch.Tensor:
    """k, v [B,n,H,D] float64 rows in position order; float64 [B,T,QH*D]."""
    q = q.detach().cpu().double()
    b, t, qh, d = q.shape
    group = qh // k.shape[2]
    out = torch.empty(b, t, qh, d, dtype=torch.float64)
    for i in range(b):
        n = int(starts[i]) + t
        late = torch.arange(n)[None, :] > int(starts[i]) + torch.arange(t)[:, None]
        for h in range(qh):
            kh, vh = k[i, :n, h // group], v[i, :n, h // group]
            w = torch.softmax((q[i, :, h] @ kh.T / math.sqrt(d)).masked_fill(late, -math.inf), 1)
            # a row that is not attended does not count, whatever it holds
            nan = (~late).double() @ vh.isnan().double() > 0
            out[i, :, h] = (w @ vh.nan_to_num(0.0)).masked_fill(nan, math.nan)
    return out.reshape(b, t, qh * d)
