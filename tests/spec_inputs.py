"""Inputs shared by the tests of the 8-bit cache and of drafted-tree attention,
built on the CPU, and the error bound of the attention kernels."""

import random

import torch

from litevllm_b200 import ops
from oracle import kv_q8

EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative


def randn(seed, *shape, dtype=torch.float32, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype)


def tables_for(ctx, bs, seed, extra=2):
    """(tables int32 [B, max], pool blocks): shuffled blocks, zero padded."""
    need = [-(-c // bs) for c in ctx]
    pool = sum(need) + extra
    order = list(range(pool))
    random.Random(seed).shuffle(order)
    tables = torch.zeros((len(ctx), max(need + [1])), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return tables, pool


def cache_for(kind, pool, bs, H_kv, D, seed, dtype):
    """(data, scale or None) on the CPU; kind: a 16-bit dtype or an 8-bit one.
    Rows of very different size, so that scales matter."""
    size = torch.exp(randn(seed + 1, pool, bs, H_kv, 1))
    x = (randn(seed, pool, bs, H_kv, D) * size).to(dtype)
    if kind not in kv_q8.M_OF:
        return x, None
    q, s = kv_q8.quantise(x, kind)
    return q.float().to(kind), s.transpose(1, 2).contiguous()


def on(dev, data, scale):
    if scale is None:
        return data.to(dev)
    return ops.QuantizedCache(data.to(dev), scale.to(dev))


def random_tree(rng, n):
    parents = [-1] + [rng.randrange(-1, i) for i in range(1, n)]
    return parents[:n]


def bits_of(parents):
    sees = []
    for i, p in enumerate(parents):
        sees.append((sees[p] if p >= 0 else 0) | 1 << i)
    return sees


def row_bounds(kd, ks, vd, vs):
    """(largest |k| of a row, largest |v| element) of finite rows of a cache pair."""
    k, v = (d.double() if s is None else d.double() * s.double().transpose(1, 2)[..., None]
            for d, s in ((kd.float(), ks), (vd.float(), vs)))
    k, v = (torch.where(torch.isfinite(x), x, 0.0) for x in (k, v))
    return k.norm(dim=-1).max().item(), v.abs().max().item()


def assert_attention(got, want, size, q, bounds, scale, keys, weight_eps):
    """|got - want| within the roundings of the kernel, element by element.

    got is rounded to its type once: half a step of |want|. A weight is rounded
    to 16 bits (weight_eps relative) and carries the score's error: D products
    and sums in fp32, each at most 2^-23 of sum |q k| <= |q| |k|, plus three further
    roundings of the scaled score and 2^-21 for the exponential. Sums over `keys`
    terms in fp32 add 2^-23 each to numerator and denominator. A change of weights
    by a relative e moves the average by at most 2 e times the average of |v| (size).

    Small weights: f16 is subnormal below 2^-14, so a weight w_j is off by up to
    2^-25 there, whatever its size. Weights are taken relative to a running
    maximum that some key's weight has reached (w >= 1 for that key t). Over a
    16-bit cache w_j = p_j / p_t up to the same factor, the average is
    sum w_j v_j / sum w_j with sum w_j >= 1, and the error at most
    sum_j 2^-25 |v_j| <= keys 2^-25 max|v|. Over an 8-bit cache w_j = p_j s_j / (p_t s_t)
    weighs the integers q_j, |q_j| <= M, and the average is
    (p_t s_t / sum p) sum w_j q_j: its error is at most
    s_t keys 2^-25 M <= keys 2^-25 max|v|, since a row's largest |v| is M s.
    """
    got, want, size = got.detach().double().cpu(), want.double(), size.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN pattern differs"
    same = torch.isinf(want)
    assert torch.equal(got[same], want[same])
    D = q.shape[-1]
    kmax, vmax = bounds
    dot = q.double().norm(dim=-1, keepdim=True) * kmax * abs(scale) * 1.4427
    e = weight_eps + (D + 4) * 2.0 ** -23 * dot + 2.0 ** -21 + keys * 2.0 ** -23
    bound = EPS[q.dtype] * want.abs() + 2 * e * size + keys * 2.0 ** -25 * vmax
    ok = torch.isfinite(want)
    err = (got - want).abs()
    assert (err[ok] <= bound[ok]).all(), (
        f"max error {err[ok].max().item():.3e}, worst ratio to its bound "
        f"{(err[ok] / bound[ok]).max().item():.2f}")
