"""Drafted-tree attention oracle (torch on CPU, 64 bits). Test infrastructure only.

No counterpart in the reference: Attention._decode_fast
(litevllm/layers/attention.py:91-139) for several query tokens per sequence,
the last of its context, with a visibility bit for each pair of them.
"""

from __future__ import annotations

import torch

from .kv_q8 import rows


def attend(q, k, v, seen, scale):
    """q [n, H, D], k / v [S, H_kv, D], seen bool [n, S] -> (out, mean|v|),
    both [n, H, D] fp64. A key that a token does not see takes no part at
    all, whatever its values; no key seen: NaN."""
    n, H, D = q.shape
    S, H_kv = k.shape[0], k.shape[1]
    qg = q.double().view(n, H_kv, H // H_kv, D)
    x = torch.einsum("nhgd,shd->nhgs", qg, k) * scale
    hide = ~seen[:, None, None, :]
    x = x.masked_fill(hide, -float("inf"))
    top = x.amax(-1, keepdim=True) if S else torch.zeros((n, H_kv, H // H_kv, 1))
    p = torch.exp(x - torch.where(torch.isinf(top) & (top < 0), torch.zeros_like(top), top))
    p = p.masked_fill(hide, 0.0) / p.masked_fill(hide, 0.0).sum(-1, keepdim=True)
    special = ~torch.isfinite(v).all(-1).all(-1)  # keys whose values need care: 0 * inf
    vz = torch.where(special[:, None, None], torch.zeros_like(v), v)
    out = torch.einsum("nhgs,shd->nhgd", p, vz)
    size = torch.einsum("nhgs,shd->nhgd", p, vz.abs())
    for s in special.nonzero().flatten().tolist():
        add = p[..., s, None] * v[s][None, :, None, :]
        out = torch.where(seen[:, s][:, None, None, None], out + add, out)
    none = ~seen.any(-1)  # also where there is no key at all
    out[none] = float("nan")
    return out.reshape(n, H, D), size.reshape(n, H, D)


def visible(n: int, ctx: int, mask=None) -> torch.Tensor:
    """bool [n, ctx]: mask is a list of n integers (bit d: drafted token d), or
    None for a chain."""
    prior = max(ctx - n, 0)
    seen = torch.zeros((n, ctx), dtype=torch.bool)
    seen[:, :prior] = True
    for i in range(n):
        bits = (1 << (i + 1)) - 1 if mask is None else mask[i]
        for d in range(ctx - prior):
            seen[i, prior + d] = bool(bits >> d & 1)
    return seen


def tree(query, kd, ks, vd, vs, tables, ctx, counts, masks, scale):
    """Rows of every sequence in turn: (out, mean|v|) [T, H, D] fp64. masks[b] as
    in visible()."""
    outs, sizes, at = [], [], 0
    for b, (c, n) in enumerate(zip(ctx, counts)):
        k, v = rows(kd, ks, tables[b], c), rows(vd, vs, tables[b], c)
        o, s = attend(query[at:at + n], k, v, visible(n, c, masks[b]), scale)
        outs.append(o)
        sizes.append(s)
        at += n
    return torch.cat(outs), torch.cat(sizes)


def decode(query, kd, ks, vd, vs, tables, ctx, scale):
    outs, sizes = [], []
    for b, c in enumerate(ctx):
        k, v = rows(kd, ks, tables[b], c), rows(vd, vs, tables[b], c)
        o, s = attend(query[b:b + 1], k, v, torch.ones((1, c), dtype=torch.bool), scale)
        outs.append(o)
        sizes.append(s)
    return torch.cat(outs), torch.cat(sizes)
