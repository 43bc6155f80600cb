"""Logits-processing oracle (numpy, 64 bits). Test infrastructure only.

The repetition step is _apply_repetition_penalty
(litevllm/layers/sampler.py:190-201); frequency and presence penalties, biases
and the allowed mask have no counterpart in the reference.
"""

from __future__ import annotations

import numpy as np


def process(x, prompt=None, output=None, repetition=None, presence=None, frequency=None, bias=None,
            allowed=None):
    """x [B, V]; prompt / output: lists of B id lists; repetition, presence,
    frequency: [B]; bias: list of B lists of (id, value); allowed: bool [B, V].
    Ids outside [0, V) are ignored."""
    x = np.array(x, dtype=np.float64)
    B, V = x.shape
    inside = lambda ids: [i for i in ids if 0 <= i < V]  # noqa: E731
    for b in range(B):
        out = inside(output[b]) if output is not None else []
        past = sorted(set(out) | set(inside(prompt[b]) if prompt is not None else []))
        if repetition is not None and past:
            r = float(repetition[b])
            x[b, past] = np.where(x[b, past] > 0, x[b, past] / r, x[b, past] * r)
        for i in set(out):
            c = out.count(i)
            x[b, i] -= (float(frequency[b]) * c if frequency is not None else 0.0) + (
                float(presence[b]) if presence is not None else 0.0)
        if bias is not None:
            for i, v in bias[b]:
                if 0 <= i < V:
                    x[b, i] += v
        if allowed is not None:
            x[b, ~allowed[b]] = -np.inf
    return x
