"""What the read-back of whole blocks of an 8-bit cache refuses, without a GPU."""

import pytest
import torch

from litevllm_b200 import _lib, ops

P = 1 << 20  # aligned stand-in pointer: nothing is launched on these paths


def test_load_q8_blocks_rejects_bad_arguments():
    f = _lib.lib().lk_load_kv_q8_blocks
    #      ko vo ot kd ks vd vs bt stride ctx S H  D  nb  bs max dt fmt st stream
    args = [P, P, P, P, P, P, P, P, 4, P, 2, 8, 128, 10, 16, 4, 2, 1, None, None]

    def rc(**at):
        a = list(args)
        for k, v in at.items():
            a[int(k[1:])] = v
        return f(*a)

    assert rc(_10=0) == 0 and rc(_15=0) == 0                # no sequences, no columns
    for i in (0, 1, 2, 3, 4, 5, 6, 7, 9):
        assert rc(**{f"_{i}": None}) == -1
    for i in (10, 11, 13, 15):
        assert rc(**{f"_{i}": -1}) == -1
    assert rc(_14=0) == -1
    assert rc(_12=80) == -2                                 # head dim
    assert rc(_16=7) == -2 and rc(_17=0) == -2              # type, format
    assert rc(_13=1 << 31) == -2
    assert rc(_10=1 << 20, _15=1 << 10) == -1               # rows past 32 bits
    assert rc(_0=P + 2) == -3 and rc(_5=P + 8) == -3


def test_ops_refuse_cpu_tensors():
    k, v = (ops.new_quantized_cache(4, 16, 2, 64, device="cpu") for _ in range(2))
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.load_kvcache_q8_blocks(k, v, i32(1, 2), i32(1))
    with pytest.raises(TypeError, match="both be QuantizedCache"):
        ops.load_kvcache_q8_blocks(k, v.data, i32(1, 2), i32(1))
