"""What the 8-bit cache, drafted-tree and logits functions refuse with tensors on
the GPU: each call differs from a valid one in one argument, raises before
anything is launched and leaves its outputs as they were."""

import pytest
import torch

from litevllm_b200 import _lib, ops

pytestmark = pytest.mark.gpu

BF16, F16, I32, I64 = torch.bfloat16, torch.float16, torch.int32, torch.int64


def refused(error, match, f, args, **changed):
    with pytest.raises(error, match=match):
        f(**{**args, **changed})


def caches(cuda, D=64, kind=torch.int8):
    return [ops.new_quantized_cache(4, 16, 2, D, kind, device=cuda) for _ in range(2)]


def test_store(cuda):
    k, v = caches(cuda)
    x = torch.ones(3, 2, 64, dtype=BF16, device=cuda)
    args = dict(key=x, value=x, key_cache=k, value_cache=v, slot_mapping=torch.arange(3, device=cuda))
    f = ops.store_kvcache_q8
    refused(ValueError, "equal shapes", f, args, value=x[:2])
    refused(ValueError, "num_blocks", f, args, key=x[:, :1], value=x[:, :1])
    refused(ValueError, "d-stride", f, args, key=x.transpose(1, 2).contiguous().transpose(1, 2))
    refused(TypeError, "dtype", f, args, key=x.float(), value=x.float())
    refused(TypeError, "share a dtype", f, args, value=x.half())
    refused(TypeError, "int64", f, args, slot_mapping=torch.arange(3, device=cuda, dtype=I32))
    refused(TypeError, "int64", f, args, slot_mapping=torch.arange(4, device=cuda))
    refused(TypeError, "status", f, args, status=torch.zeros(1, dtype=I64, device=cuda))
    refused(TypeError, "Tensor", f, args, slot_mapping=[0, 1, 2])
    refused(RuntimeError, "CUDA", f, args, slot_mapping=torch.arange(3))
    wide = caches(cuda, D=96)
    y = torch.ones(3, 2, 96, dtype=BF16, device=cuda)
    refused(_lib.LiteKernError, "unsupported", f, args, key=y, value=y, key_cache=wide[0], value_cache=wide[1])
    assert not k.data.any() and not v.scale.any()


def test_load(cuda):
    k, v = caches(cuda)
    i32 = lambda *x: torch.tensor(x, dtype=I32, device=cuda)  # noqa: E731
    args = dict(key_cache=k, value_cache=v, block_tables=i32([0, 1]), context_lens=i32(20),
                cu_rows=i32(0, 20), num_rows=20)
    f = ops.load_kvcache_q8
    out = torch.full((20, 2, 64), 3.0, dtype=BF16, device=cuda)
    refused(TypeError, "block_tables", f, args, block_tables=torch.zeros(1, 2, dtype=I64, device=cuda))
    refused(TypeError, "context_lens", f, args, context_lens=i32(20, 1))
    refused(TypeError, "cu_rows", f, args, cu_rows=i32(0, 10, 20))
    refused(ValueError, "num_rows", f, args, num_rows=-1)
    refused(TypeError, "dtype", f, args, dtype=torch.float64)
    refused(TypeError, "dtype", f, args, dtype="bf16")
    refused(ValueError, "key_out", f, args, key_out=out[:19])
    refused(ValueError, "key_out", f, args, value_out=out.half())
    refused(ValueError, "different", f, args, key_out=out, value_out=out)
    assert (out == 3).all()


def test_attention(cuda):
    k, v = caches(cuda)
    i32 = lambda *x: torch.tensor(x, dtype=I32, device=cuda)  # noqa: E731
    q = torch.ones(3, 4, 64, dtype=BF16, device=cuda)
    mask = torch.ones(3, 1, dtype=I64, device=cuda)
    args = dict(query=q, key_cache=k, value_cache=v, block_tables=i32([0, 1]), context_lens=i32(20),
                cu_seqlens_q=i32(0, 3), max_q_len=3, scale=0.1, tree_mask=mask)
    f = ops.paged_tree_attention
    out = torch.full_like(q, 3.0)
    refused(ValueError, r"\[T, H, D\]", f, args, query=q[0])
    refused(ValueError, "shape", f, args, query=torch.ones(3, 4, 128, dtype=BF16, device=cuda))
    refused(TypeError, "dtype", f, args, query=q.float())
    refused(TypeError, "cu_seqlens_q", f, args, cu_seqlens_q=i32(0, 1, 3))
    refused(TypeError, "Tensor", f, args, cu_seqlens_q=None)
    refused(ValueError, "max_q_len", f, args, max_q_len=-1)
    refused(TypeError, "max_q_len", f, args, max_q_len=None)
    refused(TypeError, "tree_mask", f, args, tree_mask=mask.int())
    refused(TypeError, "tree_mask", f, args, tree_mask=mask[:2])
    refused(ValueError, "tree_mask", f, args, max_q_len=65)
    refused(ValueError, "out", f, args, out=out.half())
    refused(ValueError, "out", f, args, out=out[:1].expand(3, 4, 64))
    refused(_lib.LiteKernError, "invalid", f, args, query=q[:, :3].contiguous())      # H no multiple of H_kv
    x16 = [torch.zeros(4, 16, 2, 64, dtype=F16, device=cuda) for _ in range(2)]
    refused(TypeError, "match", f, args, key_cache=x16[0], value_cache=x16[1])
    refused(TypeError, "both", f, args, key_cache=x16[0])
    dec = dict(query=q, key_cache=k, value_cache=v, block_tables=i32([0], [1], [2]),
               context_lens=i32(3, 4, 5), scale=0.1)
    refused(ValueError, "one query per row", ops.paged_decode_q8, dec, query=q[:2])
    refused(TypeError, "both", ops.paged_decode_q8, dec, key_cache=x16[0], value_cache=x16[1])
    refused(ValueError, "workspace", ops.paged_decode_q8, dec, block_tables=i32(*[[0] * 4096] * 3),
            workspace=torch.zeros(16, dtype=torch.uint8, device=cuda))
    assert (out == 3).all()


def test_logits(cuda):
    x = torch.ones(2, 100, dtype=BF16, device=cuda)
    f = ops.process_logits
    args = dict(logits=x)
    i64 = torch.zeros(2, 3, dtype=I64, device=cuda)
    refused(ValueError, r"\[B, V\]", f, args, logits=x[:, :0])
    refused(TypeError, "dtype", f, args, logits=x.double())
    refused(TypeError, "prompt_ids", f, args, prompt_ids=i64.int())
    refused(TypeError, "output_ids", f, args, output_ids=i64[:1])
    refused(TypeError, "prompt_lens", f, args, prompt_ids=i64, prompt_lens=torch.ones(3, dtype=I32, device=cuda))
    refused(TypeError, "presence", f, args, presence=torch.ones(2, dtype=BF16, device=cuda))
    refused(ValueError, "together", f, args, bias_ids=i64)
    refused(TypeError, "bias", f, args, bias_ids=i64, bias=torch.zeros(2, 2, device=cuda))
    refused(TypeError, "allowed", f, args, allowed=torch.zeros(2, 3, dtype=I32, device=cuda))
    refused(ValueError, "out", f, args, out=x.half())
    refused(ValueError, "out", f, args, out=x[:1].expand(2, 100))
    cols = torch.ones(100, 2, dtype=BF16, device=cuda).t()
    refused(ValueError, "in place", f, args, logits=cols, out=cols)
    many = torch.zeros(2, 1025, dtype=I64, device=cuda)
    refused(_lib.LiteKernError, "unsupported", f, args, bias_ids=many, bias=many.float())
    assert (x == 1).all()
