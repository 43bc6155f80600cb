"""The 8-bit KV cache on the GPU against the 64-bit oracle: quantised rows are
equal bit for bit, rows read back are the oracle's values rounded once, and
decode attention is within its roundings."""

import random

import pytest
import torch

from litevllm_b200 import _lib, ops
from oracle import kv_q8, tree_attention
from tests.spec_inputs import assert_attention, cache_for, on, randn, row_bounds, tables_for

pytestmark = pytest.mark.gpu

INT8, E4M3 = torch.int8, torch.float8_e4m3fn
BF16, F16 = torch.bfloat16, torch.float16


def expected_cache(key, slots, kind, nb, bs):
    """(data, scale) after the store of rows into zeroed caches."""
    T, H_kv, D = key.shape
    q, s = kv_q8.quantise(key, kind)
    data = torch.zeros((nb * bs, H_kv, D), dtype=torch.float64)
    scale = torch.zeros((nb * bs, H_kv))
    for t, slot in enumerate(slots):
        if 0 <= slot < nb * bs:
            data[slot], scale[slot] = q[t], s[t]
    return data.view(nb, bs, H_kv, D), scale.view(nb, bs, H_kv).transpose(1, 2)


def assert_same(got: ops.QuantizedCache, data, scale):
    assert torch.equal(got.data.float().cpu().double(), data)
    s = got.scale.cpu()
    assert torch.equal(torch.isnan(s), torch.isnan(scale))
    assert torch.equal(s.nan_to_num(7.0), scale.nan_to_num(7.0))


@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,H_kv,D,bs", [(1, 1, 64, 16), (1, 8, 128, 16), (37, 3, 64, 8),
                                         (300, 8, 128, 24), (1025, 2, 128, 16)])
def test_store_matches_oracle(cuda, kind, dtype, T, H_kv, D, bs):
    nb = -(-T // bs) + 1
    # slices of a fused projection (16-byte loads), and an odd token stride
    for pad in (2 * H_kv * D, H_kv * D + 1):
        wide = randn(T + pad, T, pad + H_kv * D, dtype=dtype, std=3.0)
        key = wide[:, pad:].unflatten(1, (H_kv, D))
        value = wide[:, :H_kv * D].unflatten(1, (H_kv, D))
        slots = torch.tensor(random.Random(T).sample(range(nb * bs), T))
        slots[::5] = -1
        w = wide.cuda()
        kc, vc = (ops.new_quantized_cache(nb, bs, H_kv, D, kind) for _ in range(2))
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        ops.store_kvcache_q8(w[:, pad:].unflatten(1, (H_kv, D)),
                             w[:, :H_kv * D].unflatten(1, (H_kv, D)), kc, vc, slots.cuda(), status)
        assert_same(kc, *expected_cache(key, slots.tolist(), kind, nb, bs))
        assert_same(vc, *expected_cache(value, slots.tolist(), kind, nb, bs))
        assert status.item() == 0


@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_store_special_rows(cuda, kind, dtype):
    """Zeros, one value, the smallest and largest values, ties, infinities, NaN."""
    D = 128
    big = torch.finfo(dtype).max
    x = torch.zeros((12, 1, D))
    x[1, 0, 5] = -2.5
    x[2] = big
    x[3, 0, ::2] = -big
    x[4, 0, 0] = float("inf")
    x[5, 0, 127] = -float("inf")
    x[6, 0, 64] = float("nan")
    x[7, 0, 3] = torch.finfo(dtype).smallest_normal
    x[8, 0, 9] = torch.finfo(dtype).smallest_normal / 64  # subnormal
    x[9, 0] = torch.arange(D) - 63.5    # with 127 below: halves, ties to even
    x[9, 0, 0] = 127.0
    x[10, 0] = torch.arange(D) * 448 / 128.0
    x[10, 0, 1] = 448.0
    x[11, 0, ::3] = 1e-3
    x = x.to(dtype)
    kc, vc = (ops.new_quantized_cache(1, 16, 1, D, kind) for _ in range(2))
    slots = torch.arange(12)
    ops.store_kvcache_q8(x.cuda(), x.cuda().flip(0), kc, vc, slots.cuda())
    assert_same(kc, *expected_cache(x, slots.tolist(), kind, 1, 16))
    assert_same(vc, *expected_cache(x.flip(0), slots.tolist(), kind, 1, 16))
    k, _ = ops.load_kvcache_q8(kc, vc, torch.zeros((1, 1), dtype=torch.int32, device=cuda),
                               torch.tensor([12], dtype=torch.int32, device=cuda),
                               torch.tensor([0, 12], dtype=torch.int32, device=cuda), 12,
                               dtype=torch.float32)
    assert torch.isnan(k[4:7]).all() and torch.isfinite(k[:4]).all() and torch.isfinite(k[7:]).all()


@pytest.mark.parametrize("kind", [INT8, E4M3])
def test_store_leaves_other_slots_and_flags_bad_ones(cuda, kind):
    kc, vc = (ops.new_quantized_cache(3, 16, 2, 64, kind) for _ in range(2))
    for c in (kc, vc):
        c.data.view(torch.uint8).fill_(17)
        c.scale.fill_(3.0)
    before = [t.clone() for c in (kc, vc) for t in (c.data.view(torch.uint8), c.scale)]
    x = randn(1, 5, 2, 64, dtype=BF16).cuda()
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    slots = torch.tensor([-1, 48, -7, 1 << 40, -1], device=cuda)
    ops.store_kvcache_q8(x, x, kc, vc, slots, status)
    after = [t for c in (kc, vc) for t in (c.data.view(torch.uint8), c.scale)]
    assert all(torch.equal(a, b) for a, b in zip(before, after))
    assert status.item() == _lib.LK_STATUS_SLOT_OOB
    ops.store_kvcache_q8(x[:0], x[:0], kc, vc, slots[:0])  # no tokens
    ops.store_kvcache_q8(x, x, kc, vc, torch.tensor([47, -1, 0, 16, 31], device=cuda))
    changed = (kc.scale != 3.0).any(1).view(-1).nonzero().flatten().tolist()
    assert changed == [0, 16, 31, 47]


@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [torch.float32, BF16, F16])
@pytest.mark.parametrize("H_kv,D,bs", [(1, 64, 16), (8, 128, 16), (3, 128, 24), (2, 64, 8)])
def test_load_matches_oracle(cuda, kind, dtype, H_kv, D, bs):
    ctx = [0, 1, bs, 3 * bs + 5, 77, 0, 130]
    tables, pool = tables_for(ctx, bs, 3)
    kd, ks = cache_for(kind, pool, bs, H_kv, D, 11, BF16)
    vd, vs = cache_for(kind, pool, bs, H_kv, D, 12, BF16)
    starts = [5]  # rows in front of the first sequence, and some past each context
    for i, c in enumerate(ctx):
        starts.append(starts[-1] + c + (i % 3))
    n = starts[-1] + 4
    outs = [torch.full((n, H_kv, D), 9.0, dtype=dtype, device=cuda) for _ in range(2)]
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    got = ops.load_kvcache_q8(on(cuda, kd, ks), on(cuda, vd, vs), tables.cuda(),
                              torch.tensor(ctx, dtype=torch.int32).cuda(),
                              torch.tensor(starts, dtype=torch.int32).cuda(), n, dtype=dtype,
                              key_out=outs[0], value_out=outs[1], status=status)
    assert got[0] is outs[0] and status.item() == 0
    for out, d, s in ((outs[0], kd, ks), (outs[1], vd, vs)):
        want = torch.full((n, H_kv, D), 9.0, dtype=torch.float64)
        want[starts[0]:starts[-1]] = 0.0
        for b, c in enumerate(ctx):
            # the product is rounded to fp32, then to the type
            want[starts[b]:starts[b] + c] = kv_q8.rows(d, s, tables[b], c).float().to(dtype).double()
        assert torch.equal(out.double().cpu(), want)


def test_load_bad_tables(cuda):
    kd, ks = cache_for(INT8, 2, 16, 1, 64, 1, BF16)
    c = on(cuda, kd, ks)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    k, v = ops.load_kvcache_q8(c, c, i32(1, 2).view(1, 2), i32(20), i32(0, 20), 20, status=status)
    assert status.item() == _lib.LK_STATUS_BLOCK_OOB
    assert (k[16:] == 0).all() and (k[:16] != 0).any()
    status.zero_()
    k, v = ops.load_kvcache_q8(c, c, i32(1).view(1, 1), i32(20), i32(0, 20), 20, status=status)
    assert status.item() == _lib.LK_STATUS_CTX_OOB
    assert (v[16:] == 0).all() and (v[:16] != 0).any()
    # no sequences, no rows, an empty table
    assert ops.load_kvcache_q8(c, c, i32().view(0, 1), i32(), i32(0), 0)[0].shape == (0, 1, 64)
    k, _ = ops.load_kvcache_q8(c, c, i32().view(1, 0), i32(0), i32(0, 3), 3)
    assert (k == 0).all()


DECODE = [  # (H, H_kv, D, bs, ctx)
    (1, 1, 64, 16, [1]),
    (32, 8, 128, 16, [0, 1, 15, 16, 17, 31, 32, 33, 127, 128, 129]),
    (32, 8, 128, 16, [777]),
    (8, 8, 128, 16, [255, 256, 257, 511, 512, 513]),          # G = 1
    (6, 2, 64, 24, [5, 1000, 300, 0]),                        # G = 3
    (16, 1, 128, 8, [700, 1, 64]),                            # G = 16
    (40, 1, 64, 32, [100, 513]),                              # G = 40
    (14, 2, 128, 48, [2500, 40]),                             # G = 7
    (5, 5, 64, 1, [66, 3]),                                   # one-slot blocks
    (80, 2, 128, 16, [4097, 0, 1, 2500, 64, 63, 3000]),       # G = 40, enough work for tcgen05
    (128, 1, 64, 32, [4097, 4096, 4000, 65, 4095]),           # G = 128, the same
]


@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("H,H_kv,D,bs,ctx", DECODE)
def test_decode_matches_oracle(cuda, kind, dtype, H, H_kv, D, bs, ctx):
    tables, pool = tables_for(ctx, bs, len(ctx))
    kd, ks = cache_for(kind, pool, bs, H_kv, D, 21, dtype)
    vd, vs = cache_for(kind, pool, bs, H_kv, D, 22, dtype)
    B = len(ctx)
    wide = randn(23, B, H * D + 8, dtype=dtype)      # a token stride wider than the heads
    q = wide[:, :H * D].unflatten(1, (H, D))
    scale = D ** -0.5
    want, size = tree_attention.decode(q, kd, ks, vd, vs, tables, ctx, scale)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    got = ops.paged_decode_q8(wide.cuda()[:, :H * D].unflatten(1, (H, D)), on(cuda, kd, ks),
                              on(cuda, vd, vs), tables.cuda(),
                              torch.tensor(ctx, dtype=torch.int32).cuda(), scale, status=status)
    assert status.item() == 0
    assert_attention(got, want, size, q, row_bounds(kd, ks, vd, vs), scale, max(ctx), 2.0 ** -11)


@pytest.mark.parametrize("kind", [INT8, E4M3])
def test_decode_long_context_with_wide_table(cuda, kind):
    """Many splits for one sequence, one for the other, most empty; the result of
    a repeated call is the same to the bit."""
    ctx = [9001, 40]
    bs = 16
    tables, pool = tables_for(ctx, bs, 5)
    tables = torch.cat([tables, torch.zeros((2, 900), dtype=torch.int32)], 1)
    kd, ks = cache_for(kind, pool, bs, 2, 128, 31, BF16)
    vd, vs = cache_for(kind, pool, bs, 2, 128, 32, BF16)
    q = randn(33, 2, 8, 128, dtype=BF16)
    want, size = tree_attention.decode(q, kd, ks, vd, vs, tables, ctx, 0.09)
    args = (q.cuda(), on(cuda, kd, ks), on(cuda, vd, vs), tables.cuda(),
            torch.tensor(ctx, dtype=torch.int32).cuda(), 0.09)
    got = ops.paged_decode_q8(*args)
    assert_attention(got, want, size, q, row_bounds(kd, ks, vd, vs), 0.09, max(ctx), 2.0 ** -11)
    assert all(torch.equal(got, ops.paged_decode_q8(*args)) for _ in range(5))


@pytest.mark.parametrize("kind", [INT8, E4M3])
def test_decode_rows_of_very_different_size(cuda, kind):
    """Values from 2^-60 to 2^60 in one context, huge and tiny queries: the
    weights are rounded relative to their own largest, so no term is lost."""
    bs, H_kv, D = 16, 1, 64
    ctx = [64, 64, 64]
    tables, pool = tables_for(ctx, bs, 1)
    x = randn(1, pool, bs, H_kv, D)
    v = (x * torch.exp2(torch.linspace(-60, 60, pool * bs)).view(pool, bs, 1, 1)).to(BF16)
    kd, ks = (lambda q, s: (q.float().to(kind), s.transpose(1, 2).contiguous()))(*kv_q8.quantise(x.to(BF16), kind))
    vd, vs = (lambda q, s: (q.float().to(kind), s.transpose(1, 2).contiguous()))(*kv_q8.quantise(v, kind))
    q = randn(2, 3, 2, D)
    q[1] *= 2.0 ** -100
    q[2] *= 2.0 ** 6
    q = q.to(BF16)
    want, size = tree_attention.decode(q, kd, ks, vd, vs, tables, ctx, 0.125)
    got = ops.paged_decode_q8(q.cuda(), on(cuda, kd, ks), on(cuda, vd, vs), tables.cuda(),
                              torch.tensor(ctx, dtype=torch.int32).cuda(), 0.125)
    assert_attention(got, want, size, q, row_bounds(kd, ks, vd, vs), 0.125, 64, 2.0 ** -11)


def test_decode_special_rows_stay_in_their_sequence(cuda):
    """A NaN K row or V row makes its own sequence NaN and no other; stale rows
    behind a context are not read."""
    bs, ctx = 16, [20, 20, 20]
    tables, pool = tables_for(ctx, bs, 2, extra=0)
    kd, ks = cache_for(INT8, pool, bs, 1, 64, 41, BF16)
    vd, vs = cache_for(INT8, pool, bs, 1, 64, 42, BF16)
    for b in range(3):  # stale slots of the last block
        for s in (ks, vs):
            s[tables[b, 1], :, 4:] = float("nan")
    ks[tables[0, 0], 0, 3] = float("nan")
    vs[tables[1, 1], 0, 2] = float("nan")
    q = randn(43, 3, 2, 64, dtype=BF16)
    got = ops.paged_decode_q8(q.cuda(), on(cuda, kd, ks), on(cuda, vd, vs), tables.cuda(),
                              torch.tensor(ctx, dtype=torch.int32).cuda(), 0.125)
    assert torch.isnan(got[:2]).all() and torch.isfinite(got[2]).all()


def test_decode_bad_tables_are_flagged(cuda):
    kd, ks = cache_for(INT8, 2, 16, 1, 64, 1, BF16)
    c = on(cuda, kd, ks)
    q = randn(3, 1, 2, 64, dtype=BF16).cuda()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    a = ops.paged_decode_q8(q, c, c, i32(1, 5).view(1, 2), i32(20), 0.1, status=status)
    assert status.item() == _lib.LK_STATUS_BLOCK_OOB and torch.isfinite(a).all()
    status.zero_()
    a = ops.paged_decode_q8(q, c, c, i32(1).view(1, 1), i32(20), 0.1, status=status)
    assert status.item() == _lib.LK_STATUS_CTX_OOB
    assert torch.equal(a, ops.paged_decode_q8(q, c, c, i32(1).view(1, 1), i32(16), 0.1))


def test_block_copies_move_data_and_scales(cuda):
    kd, ks = cache_for(E4M3, 4, 16, 2, 64, 1, BF16)
    vd, vs = cache_for(E4M3, 4, 16, 2, 64, 2, BF16)
    k, v = on(cuda, kd, ks), on(cuda, vd, vs)
    ops.copy_blocks([(k.data, v.data)], {1: 3})
    ops.copy_blocks([(k.scale, v.scale)], {1: 3})
    for c in (k, v):
        assert torch.equal(c.data[3].float(), c.data[1].float())
        assert torch.equal(c.scale[3], c.scale[1])


def test_round_trip_error_is_within_half_a_step(cuda):
    """Stored and read back: int8 within half of a / 127 (plus fp32 roundings of
    scale and product), e4m3 within 2^-4 of the value or half its smallest step."""
    x = randn(9, 64, 4, 128, dtype=BF16, std=2.0)
    for kind in (INT8, E4M3):
        kc, vc = (ops.new_quantized_cache(4, 16, 4, 128, kind) for _ in range(2))
        ops.store_kvcache_q8(x.cuda(), x.cuda(), kc, vc, torch.arange(64, device=cuda))
        got, _ = ops.load_kvcache_q8(kc, vc, torch.arange(4, dtype=torch.int32, device=cuda).view(1, 4),
                                     torch.tensor([64], dtype=torch.int32, device=cuda),
                                     torch.tensor([0, 64], dtype=torch.int32, device=cuda), 64,
                                     dtype=torch.float32)
        a = x.double().abs().amax(-1, keepdim=True)
        err = (got.double().cpu() - x.double()).abs()
        if kind is INT8:
            bound = a / 127 * (0.5 + 127 * 2.0 ** -22)
        else:
            bound = torch.maximum(x.double().abs() * 2.0 ** -4, a / 448 * 2.0 ** -10) * (1 + 2.0 ** -20)
        assert (err <= bound).all()
