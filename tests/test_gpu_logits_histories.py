"""Logits processing with long histories: more distinct tokens in one part of the
vocabulary than its list holds (all marks are then looked at), and more output tokens
than 16-bit counts hold, with biases, masks and rows at odd addresses."""

import random

import pytest
import torch

from litevllm_b200 import ops
from tests.test_gpu_process_logits import args, check, make

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def long_case(dtype, V, n_prompt, n_output, n_bias, grammar, seed, lo, hi):
    """Histories of tokens lo .. hi - 1, drawn evenly, and all of their entries counted."""
    c = make(2, V, dtype, 1, 1, n_bias, grammar, seed)
    rng = random.Random(seed + 1)
    c["prompt"] = [[rng.randrange(lo, hi) for _ in range(n_prompt)] for _ in range(2)]
    c["output"] = [[rng.randrange(lo, hi) for _ in range(n_output)] for _ in range(2)]
    c["plen"], c["olen"] = [n_prompt, n_prompt - 7], [n_output, n_output - 5]
    c["rep"], c["pres"], c["freq"] = [1.3, 0.8], [0.7, -0.4], [0.3, 0.01]
    if n_bias:  # some on tokens of the history
        c["bias"] = [r[: n_bias // 2] + [(rng.randrange(lo, hi), 1.5) for _ in range(n_bias - n_bias // 2)]
                     for r in c["bias"]]
    return c


def run_all_ways(c, cuda):
    kw, x = args(c, cuda), c["x"].to(cuda)
    B, V = x.shape
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    got = ops.process_logits(x, status=status, **kw)
    check(got, c)
    assert status.item() == 0 and torch.equal(x.cpu(), c["x"])
    wide = torch.full((B, V + 3), 3.0, dtype=x.dtype, device=cuda)
    assert torch.equal(ops.process_logits(x, out=wide[:, 2:2 + V], **kw), got)
    wide[:, 1:1 + V] = x
    assert torch.equal(ops.process_logits(wide[:, 1:1 + V], out=wide[:, 1:1 + V], **kw), got)
    assert (wide[:, 0] == 3).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n_bias,grammar", [(0, False), (12, True)])
@pytest.mark.parametrize("V,lo,hi", [(20011, 100, 4060), (9001, 4200, 8160), (4096, 0, 4096)])
def test_more_distinct_tokens_than_a_part_lists(cuda, dtype, n_bias, grammar, V, lo, hi):
    c = long_case(dtype, V, 4000, 3000, n_bias, grammar, seed=V, lo=lo, hi=hi)
    assert all(len(set(c["prompt"][b] + c["output"][b])) > 2500 for b in range(2))
    run_all_ways(c, cuda)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hi", [40, 4000])
def test_outputs_past_16_bit_counts(cuda, dtype, hi):
    """17000 output tokens; of few ids each more than 255 times, or of thousands."""
    c = long_case(dtype, 5003, 500, 17000, 20, True, seed=hi, lo=3, hi=hi)
    run_all_ways(c, cuda)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [16383, 16384])
def test_one_token_over_and_over(cuda, dtype, n):
    """The largest count of 16 bits, and the first of 32."""
    x = torch.zeros((1, 50), dtype=dtype, device=cuda)
    ids = torch.full((1, n), 7, device=cuda)
    got = ops.process_logits(x, output_ids=ids, frequency=torch.full((1,), 0.25, device=cuda),
                             bias_ids=torch.tensor([[7, 8]], device=cuda), bias=torch.ones((1, 2), device=cuda))
    want = x.float()
    want[0, 7], want[0, 8] = 1.0 - 0.25 * n, 1.0
    assert torch.equal(got, want.to(dtype))
