"""Refusals of the 8-bit cache, drafted-tree attention and logits processing,
which need no GPU, and the oracle's own properties."""

import pytest
import torch

from litevllm_b200 import _lib, ops
from oracle import kv_q8, tree_attention

P = 1 << 20  # aligned stand-in pointer: nothing is launched on these paths


def replaced(args, **at):
    a = list(args)
    for k, v in at.items():
        a[int(k[1:])] = v
    return a


def test_store_q8_rejects_bad_arguments():
    f = _lib.lib().lk_store_kv_q8
    #      key val kd ks vd vs slots T  H  D    strides     nb  bs  dt fmt st stream
    args = [P, P, P, P, P, P, P, 4, 8, 128, 1024, 1024, 10, 16, 2, 1, None, None]
    assert f(*replaced(args, _7=0)) == 0                    # no tokens: nothing to do
    assert f(*replaced(args, _7=-1)) == -1
    assert f(*replaced(args, _8=0)) == -1
    for i in range(7):
        assert f(*replaced(args, **{f"_{i}": None})) == -1
    assert f(*replaced(args, _9=96)) == -2                  # head dim
    assert f(*replaced(args, _14=0)) == -2                  # fp32 rows
    assert f(*replaced(args, _15=0)) == -2                  # not an 8-bit format
    assert f(*replaced(args, _15=3)) == -2
    assert f(*replaced(args, _12=1 << 31)) == -2            # slots past 32 bits
    assert f(*replaced(args, _2=P + 8)) == -3               # cache not 16-byte aligned
    assert f(*replaced(args, _13=0)) == -1


def test_load_q8_rejects_bad_arguments():
    f = _lib.lib().lk_load_kv_q8
    #      ko vo kd ks vd vs bt stride ctx cu S rows H D nb bs max dt fmt st stream
    args = [P, P, P, P, P, P, P, 4, P, P, 2, 100, 8, 128, 10, 16, 4, 2, 1, None, None]
    assert f(*replaced(args, _10=0)) == 0
    assert f(*replaced(args, _11=0)) == 0
    for i in (0, 1, 2, 3, 4, 5, 6, 8, 9):
        assert f(*replaced(args, **{f"_{i}": None})) == -1
    assert f(*replaced(args, _11=-1)) == -1
    assert f(*replaced(args, _13=80)) == -2
    assert f(*replaced(args, _17=7)) == -2
    assert f(*replaced(args, _18=0)) == -2
    assert f(*replaced(args, _0=P + 2)) == -3


def test_tree_rejects_bad_arguments():
    f = _lib.lib().lk_paged_tree_attention
    #       out  s   q   s   k  ks v  vs nb  bt s  cu ctx m  ms mw T  B  mq H   Hk D   bs mb sc  dt fmt ws bytes st stream
    args = [P, 4096, P, 4096, P, P, P, P, 10, P, 4, P, P, P, 1, 1, 8, 2, 4, 32, 8, 128, 16, 4, 0.1, 2, 1, P, 1 << 30,
            None, None]
    for i in (16, 17, 18):
        assert f(*replaced(args, **{f"_{i}": 0})) == 0      # nothing to do
        assert f(*replaced(args, **{f"_{i}": -1})) == -1
    for i in (0, 2, 4, 5, 6, 7, 9, 12):
        assert f(*replaced(args, **{f"_{i}": None})) == -1
    assert f(*replaced(args, _19=12)) == -1                 # H not a multiple of H_kv
    assert f(*replaced(args, _15=0)) == -1                  # a mask without words
    assert f(*replaced(args, _18=65)) == -1                 # more tokens than mask bits
    assert f(*replaced(args, _11=None)) == -1               # decode form with a mask, several tokens
    assert f(*replaced(args, _11=None, _13=None, _18=1)) == -1   # ... with T != B
    assert f(*replaced(args, _21=256)) == -2
    assert f(*replaced(args, _25=0)) == -2
    assert f(*replaced(args, _26=5)) == -2
    assert f(*replaced(args, _8=1 << 31)) == -2
    assert f(*replaced(args, _23=1 << 30)) == -2            # table capacity past 32 bits
    assert f(*replaced(args, _4=P + 4)) == -3
    # a table that is split wants its workspace
    wide = replaced(args, _23=4096)
    need = _lib.lib().lk_paged_tree_workspace_bytes(8, 2, 4, 32, 8, 128, 16, 4096, 1)
    assert need > 0
    assert f(*replaced(wide, _27=None, _28=0)) == -4
    assert f(*replaced(wide, _28=need - 1)) == -4
    assert f(*replaced(wide, _27=P + 8)) == -4
    d = _lib.lib().lk_paged_decode_q8
    #       out s    q  s     kd ks vd vs nb bt s ctx B  H   Hk D   bs mb sc  dt fmt ws bytes st stream
    dargs = [P, 4096, P, 4096, P, P, P, P, 10, P, 4, P, 2, 32, 8, 128, 16, 4, 0.1, 2, 1, P, 1 << 30, None, None]
    assert d(*replaced(dargs, _12=0)) == 0
    assert d(*replaced(dargs, _20=0)) == -2                 # 16-bit caches: lk_paged_decode
    assert d(*replaced(dargs, _15=80)) == -2
    assert d(*replaced(dargs, _5=None)) == -1


def test_tree_workspace_sizes():
    f = _lib.lib().lk_paged_tree_workspace_bytes
    assert f(8, 8, 1, 32, 8, 128, 16, 8, 1) == 0               # 128 keys: no split
    assert f(0, 8, 1, 32, 8, 128, 16, 8, 1) == 0
    assert f(8, 8, 1, 32, 7, 128, 16, 8, 1) == 0
    one = f(1, 1, 1, 32, 8, 128, 16, 8192, 1)
    assert one % (32 * (128 + 4) * 4) == 0 and one > 0


def test_process_logits_rejects_bad_arguments():
    f = _lib.lib().lk_process_logits
    #       out ld   x  B  V    ld   p  pld pl pm o  old ol om rep pr fr bi b  nb al ald dt st stream
    args = [P, 100, P, 2, 100, 100, P, 4, P, 4, P, 4, P, 4, P, P, P, P, P, 3, P, 4, 2, None, None]
    assert f(*replaced(args, _3=0)) == 0
    for at, v in ((0, None), (2, None), (6, None), (10, None), (17, None), (18, None), (4, 0), (3, -1),
                  (5, 99), (1, 99), (7, 3), (11, 3), (21, 3), (9, -1), (13, -1), (19, -1)):
        assert f(*replaced(args, **{f"_{at}": v})) == -1, at
    assert f(*replaced(args, _1=101)) == -1                 # in place with another row stride
    assert f(*replaced(args, _19=1025)) == -2
    assert f(*replaced(args, _3=65536)) == -2
    assert f(*replaced(args, _22=9)) == -2


def caches(kind=torch.int8, nb=4, bs=16, H=2, D=64):
    return tuple(ops.new_quantized_cache(nb, bs, H, D, kind, device="cpu") for _ in range(2))


def test_ops_refuse_cpu_tensors_and_mismatched_caches():
    k, v = caches()
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    slots = torch.zeros(3, dtype=torch.int64)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.store_kvcache_q8(x, x, k, v, slots)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.load_kvcache_q8(k, v, i32(1, 2), i32(1), i32(2), 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_decode_q8(x, k, v, i32(3, 1), i32(3), 0.1)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_tree_attention(x, k, v, i32(1, 1), i32(1), i32(2), 3, 0.1)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.process_logits(torch.zeros(2, 10))
    with pytest.raises(TypeError, match="both be QuantizedCache"):
        ops.paged_decode_q8(x, k.data, v.data, i32(3, 1), i32(3), 0.1)
    with pytest.raises(TypeError, match="both be QuantizedCache"):
        ops.paged_tree_attention(x, k, v.data, i32(1, 1), i32(1), i32(2), 3, 0.1)
    other = caches(torch.float8_e4m3fn)[1]
    with pytest.raises(TypeError, match="both"):
        ops.store_kvcache_q8(x, x, k, other, slots)
    with pytest.raises(TypeError, match="fp32"):
        ops.store_kvcache_q8(x, x, k._replace(scale=k.scale.double()), v, slots)
    with pytest.raises(ValueError, match="scales"):
        ops.store_kvcache_q8(x, x, k._replace(scale=k.scale.transpose(1, 2).contiguous()), v, slots)
    with pytest.raises(ValueError, match="contiguous"):
        ops.store_kvcache_q8(x, x, k._replace(data=k.data.transpose(0, 1).contiguous().transpose(0, 1)), v, slots)
    with pytest.raises(TypeError, match="8-bit"):
        ops.new_quantized_cache(1, 16, 1, 64, torch.float16, device="cpu")


def test_tree_masks_from_parents():
    m = ops.tree_mask_from_parents([[-1, 0, 0, 2], [], [-1, -1]])
    assert m[:, 0].tolist() == [0b1, 0b11, 0b101, 0b1101, 0b1, 0b10]
    chain = ops.tree_mask_from_parents([[-1] + list(range(69))])
    assert chain.shape == (70, 2)
    assert chain[63].tolist() == [-1, 0] and chain[69].tolist() == [-1, 0b111111]
    assert chain[62, 0].item() == 2 ** 63 - 1
    for bad in ([0], [-1, 1], [-1, -2]):
        with pytest.raises(ValueError, match="parent"):
            ops.tree_mask_from_parents([bad])


def test_oracle_e4m3_rounding_is_torchs():
    """Every fp32 with 12 leading bits of significand in e4m3's range."""
    y = torch.cat([torch.arange(1, 4096).float() * 2.0 ** e for e in range(-22, -2)])
    y = y[y <= 448]
    assert torch.equal(kv_q8.nearest_e4m3(y.double()), y.to(torch.float8_e4m3fn).double())


def test_oracle_quantises_within_half_a_step():
    x = torch.randn(50, 3, 64, generator=torch.Generator().manual_seed(0)).bfloat16()
    for kind, m in kv_q8.M_OF.items():
        q, s = kv_q8.quantise(x, kind)
        assert q.abs().max() == m and torch.equal(q.float().to(kind).double(), q)
        err = (q * s.double()[..., None] - x.double()).abs()
        a = x.double().abs().amax(-1, keepdim=True)
        if kind is torch.int8:
            assert (err <= a / 127 * (0.5 + 1e-4)).all()
        else:
            assert (err <= torch.maximum(x.double().abs() * 2 ** -4, a / 448 * 2 ** -10) * (1 + 1e-5)).all()


def test_oracle_tree_equals_softmax_over_the_visible_keys():
    q, k, v = (torch.randn(n, 2, 8, dtype=torch.float64, generator=torch.Generator().manual_seed(n))
               for n in (3, 7, 7))
    v = v * 2
    seen = tree_attention.visible(3, 7, [0b1, 0b11, 0b101])
    o, _ = tree_attention.attend(q, k, v, seen, 0.5)
    for i in range(3):
        at = seen[i].nonzero().flatten()
        p = torch.softmax(torch.einsum("hd,shd->hs", q[i], k[at]) * 0.5, -1)
        assert torch.allclose(o[i], torch.einsum("hs,shd->hd", p, v[at]))
