"""Outputs that overlap an input, or each other, other than as documented are refused;
those that lie beside or between each other's rows are not."""

import pytest
import torch

from litevllm_b200 import ops
from tests.test_gpu_tree import case, run

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def test_process_logits(cuda):
    V = 100
    x = torch.randn((6, V), device=cuda)
    freq, ids = torch.ones(4, device=cuda), torch.tensor([[3, 3, 7]] * 4, device=cuda)
    call = lambda a, b: ops.process_logits(a, output_ids=ids, frequency=freq, out=b)  # noqa: E731
    flat = x.flatten()
    wide = torch.randn((4, 3 * V), device=cuda)
    before, wide_before = x.clone(), wide.clone()
    for a, b in ((x[:4], x[2:]), (x[1:5], x[:4]), (flat[:4 * V].view(4, V), flat[1:4 * V + 1].view(4, V)),
                 (wide[:, :V], wide[:, V - 1:2 * V - 1]), (wide[:, V:2 * V], wide[:, :V + 1][:, 1:]),
                 (wide[:, :V], wide.flatten()[:4 * V].view(4, V)),
                 (wide.flatten()[:4 * V].view(4, V), wide[:, :V])):
        with pytest.raises(ValueError, match="overlap"):
            call(a, b)
    torch.cuda.synchronize()
    assert torch.equal(x, before) and torch.equal(wide, wide_before)
    # beside, between and in place
    for a, b in ((wide[:, :V], wide[:, V:2 * V]), (wide[:, 2 * V:], wide[:, :V]), (wide[::1, V:2 * V], wide[:, 2 * V:])):
        want = call(a.clone(), None)
        assert torch.equal(call(a, b), want)
    even, odd = torch.randn((8, V), device=cuda).view(4, 2, V).unbind(1)
    want = call(even.clone(), None)
    assert torch.equal(call(even, odd), want) and torch.equal(call(even, even), want)


def test_load(cuda):
    k, v = (ops.new_quantized_cache(2, 16, 2, 64, device=cuda) for _ in range(2))
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    call = lambda a, b: ops.load_kvcache_q8(k, v, i32([0, 1]), i32(20), i32(0, 20), 20, key_out=a, value_out=b)  # noqa: E731
    both = torch.full((40, 2, 64), 3.0, dtype=BF16, device=cuda)
    for lo in (0, 1, 19):
        for a, b in ((both[lo:lo + 20], both[:20]), (both[:20], both[lo:lo + 20])):
            with pytest.raises(ValueError, match="overlap"):
                call(a, b)
    torch.cuda.synchronize()
    assert (both == 3).all()
    call(both[20:], both[:20])
    assert (both == 0).all()
    none = both[:0]
    ops.load_kvcache_q8(k, v, i32([0, 1]), i32(20), i32(0, 0), 0, key_out=none, value_out=none)


@pytest.mark.parametrize("kind", [BF16, torch.int8])
@pytest.mark.parametrize("width", [12, 512], ids=["few rows", "many rows"])
def test_tree_attention(cuda, kind, width):
    """In place over the query's own rows, whether contexts are split or not."""
    c = case(kind, BF16, 32, 8, 64, 16, [150, 40, 190, 77], [9, 13, 11, 13], seed=2)
    c["tables"] = torch.cat([c["tables"], torch.zeros((4, width - c["tables"].shape[1]), dtype=torch.int32)], 1)
    want = run(c, cuda)
    n = c["q"].shape[0]
    wide = torch.zeros((n + 2, 32 * 64 + 64), dtype=BF16, device=cuda)
    q = wide[:n, :32 * 64].view(n, 32, 64)
    q.copy_(c["q"])
    before = wide.clone()
    c["q"] = q
    for out in (wide[1:n + 1, :32 * 64], wide[:n, 64:], wide.flatten()[:n * 32 * 64]):
        with pytest.raises(ValueError, match="overlap"):
            run(c, cuda, out=out.view(n, 32, 64))
    torch.cuda.synchronize()
    assert torch.equal(wide, before)
    assert run(c, cuda, out=q) is q and torch.equal(q, want)


def test_decode(cuda):
    k, v = (ops.new_quantized_cache(8, 16, 2, 64, device=cuda) for _ in range(2))
    ops.store_kvcache_q8(*(torch.randn((128, 2, 64), device=cuda).bfloat16() for _ in range(2)), k, v,
                         torch.arange(128, device=cuda))
    table = torch.arange(8, dtype=torch.int32, device=cuda).expand(3, 8)
    lens = torch.tensor([100, 7, 128], dtype=torch.int32, device=cuda)
    q = torch.randn((4, 4, 64), device=cuda).bfloat16()
    want = ops.paged_decode_q8(q[:3].clone(), k, v, table, lens, 0.125)
    with pytest.raises(ValueError, match="overlap"):
        ops.paged_decode_q8(q[:3], k, v, table, lens, 0.125, out=q[1:])
    assert torch.equal(ops.paged_decode_q8(q[:3], k, v, table, lens, 0.125, out=q[:3]), want)
