"""Prefill over an 8-bit cache on the GPU: the contexts are read back into 16-bit
blocks, rounded once more, and attended by the prefill kernel."""

import pytest
import torch

from litevllm_b200 import ops
from litevllm_b200.attention import Attention
from tests.spec_inputs import cache_for, on

pytestmark = pytest.mark.gpu

INT8, E4M3 = torch.int8, torch.float8_e4m3fn
BF16, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("kind", [BF16, INT8])
@pytest.mark.parametrize("seqs", [0, 1, 3])
def test_no_new_tokens_under_a_table_without_columns(cuda, kind, seqs):
    """As over a 16-bit cache: nothing to attend, an empty result."""
    kd, ks = cache_for(kind, 2, 16, 2, 128, 1, BF16)
    c = on(cuda, kd, ks)
    none = torch.zeros((0, 8, 128), dtype=BF16, device=cuda)
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=cuda)  # noqa: E731
    got = Attention(8, 128, 2).forward(none, None, None, c, c, i32(seqs, 0), None, i32(seqs),
                                       is_prefill=True, cu_seqlens_q=i32(seqs + 1), max_q_len=1)
    assert got.shape == (0, 8, 128)
