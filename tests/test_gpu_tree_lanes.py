"""Drafted-tree attention where the query rows of one warp go different ways: rows
whose largest score comes late and not in the same place, row counts that fill no
whole warp, and special values that only some rows see."""

import random

import pytest
import torch

from litevllm_b200 import _lib
from oracle import kv_q8
from tests.test_gpu_tree import BF16, E4M3, F16, INT8, case, check, run

pytestmark = pytest.mark.gpu


def put_row(c, which, b, key, rows):
    """Rows [H_kv, D] as the K or V (which) of one position of sequence b."""
    bs = c["kd"].shape[1]
    blk, off = c["tables"][b, key // bs], key % bs
    if c["ks"] is None:
        c[which + "d"][blk, off] = rows.to(c["kd"].dtype)
    else:
        q, s = kv_q8.quantise(rows.to(c["q"].dtype), c["kd"].dtype)
        c[which + "d"][blk, off] = q.float().to(c["kd"].dtype)
        c[which + "s"][blk, :, off] = s


def late_maxima(kind, counts, seed, tables_to=256):
    """Contexts of some 700 keys under a wide table (many keys for one CTA of the
    tcgen05 kernel), where a key in each 64 points along one query row, ever
    longer: that row's maximum rises there, and others' where they lie near it."""
    rng = random.Random(seed)
    dtype = kind if kind in (BF16, F16) else BF16
    H, H_kv, D = 32, 8, 128
    ctx = [rng.randint(640, 740) for _ in counts]
    c = case(kind, dtype, H, H_kv, D, 16, ctx, counts, seed=seed)
    extra = tables_to - c["tables"].shape[1]
    c["tables"] = torch.cat([c["tables"], torch.zeros((len(ctx), extra), dtype=torch.int32)], 1)
    at = 0
    for b, n in enumerate(counts):
        for j in range((ctx[b] - n) // 64):
            token = at + rng.randrange(n)
            q = c["q"][token].float().view(H_kv, H // H_kv, D)[:, rng.randrange(H // H_kv)]
            put_row(c, "k", b, 64 * j + rng.randrange(64), q / q.norm(dim=-1, keepdim=True) * 9.0 * (j + 1))
        at += n
    return c


@pytest.mark.parametrize("kind", [BF16, F16, INT8, E4M3])
@pytest.mark.parametrize("counts", [[5, 9, 13, 7, 1, 11, 8, 10, 3, 12, 6, 13], [33, 40, 17, 64] * 3],
                         ids=["one tile", "two tiles"])
def test_maxima_that_rise_late(cuda, kind, counts):
    c = late_maxima(kind, counts, seed=len(set(counts)))
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    got = run(c, cuda, status=status)
    check(c, got)
    assert status.item() == 0
    assert all(torch.equal(got, run(c, cuda)) for _ in range(3))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_special_values_beside_rows_that_fill_no_warp(cuda, dtype):
    """Drafted V rows with infinities, seen by some of 36 to 52 query rows."""
    counts = [13, 9, 11] * 4
    c = late_maxima(dtype, counts, seed=5)
    for b, n in enumerate(counts):
        rows = torch.ones((8, 128))
        rows[:, 70 + b] = float("inf")
        put_row(c, "v", b, c["ctx"][b] - n + 2, rows)
    got = run(c, cuda)
    assert torch.isinf(got).any() and not torch.isnan(got).any()
    check(c, got)


@pytest.mark.parametrize("kind", [INT8, E4M3])
def test_rows_and_scales_stored_right_before_are_read(cuda, kind):
    """Steps of store, tree attention, store, ... with no wait between them, each of rows of
    another size in the same slots, give what the same steps give one at a time."""
    from litevllm_b200 import ops
    from tests.spec_inputs import on, randn

    c = late_maxima(kind, [9, 13, 11, 13] * 3, seed=7)
    k, v = on(cuda, c["kd"], c["ks"]), on(cuda, c["vd"], c["vs"])
    slots = []
    for b, (n, ctx) in enumerate(zip(c["counts"], c["ctx"])):
        slots += [c["tables"][b, p // 16].item() * 16 + p % 16 for p in range(ctx - n, ctx)]
    slots = torch.tensor(slots, device=cuda)
    rows = [randn(i, len(slots), 8, 128, dtype=BF16, std=2.0 ** (3 * (i % 4) - 6)).to(cuda) for i in range(8)]
    args = (c["q"].to(cuda), k, v, c["tables"].to(cuda), torch.tensor(c["ctx"], dtype=torch.int32).to(cuda),
            c["cu"].to(cuda), max(c["counts"]), c["scale"])
    mask = c["mask"].to(cuda)

    def step(i, wait):
        ops.store_kvcache_q8(rows[i], rows[(i + 3) % 8], k, v, slots)
        if wait:
            torch.cuda.synchronize()
        return ops.paged_tree_attention(*args, tree_mask=mask)

    want = [step(i, True) for i in range(8)]
    torch.cuda.synchronize()
    for _ in range(20):
        got = [step(i, False) for i in range(8)]
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("width", [None, 256], ids=["few rows", "many rows"])
@pytest.mark.parametrize("ends", [(2 ** 31 - 8, -2 ** 31), (2 ** 31 - 1, 2 ** 31 - 1), (-2 ** 31, 5),
                                  (2 ** 31 - 8, 2 ** 31 - 4)])
def test_sequence_bounds_that_pass_32_bits(cuda, width, ends):
    """Entries of cu_seqlens_q whose difference, or whose rows' end, does not fit 32
    bits: flagged, the first sequence's rows up to max_q_len computed, no other touched."""
    counts = [13] + [9] * 11
    c = late_maxima(BF16, counts, seed=9) if width else case(BF16, BF16, 8, 2, 128, 16, [250] * 12, counts, seed=9)
    good = run(c, cuda)
    c["cu"] = torch.tensor([0, *ends] + [0] * 10, dtype=torch.int32)
    out = torch.full_like(good, 5.0)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    run(c, cuda, out=out, status=status)
    torch.cuda.synchronize()
    assert status.item() & _lib.LK_STATUS_CTX_OOB
    rows = 13 if ends[0] > 0 else 0
    assert torch.equal(out[:rows], good[:rows]) and (out[rows:] == 5).all()


@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("counts", [[9, 13, 11, 13] * 3, [3, 2, 4] * 4], ids=["many rows", "few rows"])
def test_rows_of_scale_zero_outweigh_far_smaller_scores(cuda, kind, counts):
    """A slot that was never written (scale 0: its key scores 0, its value is 0) behind
    keys whose scores are about -120: it takes all the weight, and the result is 0."""
    c = late_maxima(kind, counts, seed=3)
    c["q"] = c["q"][:1, :1].expand_as(c["q"]).contiguous()
    q = c["q"][0, 0].float()
    rows = (-120.0 * q / q.norm()).expand(8, 128) * (128 ** 0.5 / q.norm())
    for b, ctx in enumerate(c["ctx"]):
        for p in range(ctx):
            put_row(c, "k", b, p, rows)
        blk, off = c["tables"][b, 100 // 16], 100 % 16
        for x in "kv":
            c[x + "d"].view(torch.uint8)[blk, off] = 0
            c[x + "s"][blk, :, off] = 0.0
    got = run(c, cuda)
    check(c, got)
    assert (got == 0).all()


def test_mask_on_a_device_given_by_its_number(cuda):
    from litevllm_b200 import ops

    for device in (0, "cuda", cuda):
        m = ops.tree_mask_from_parents([[-1, 0, 0]], device)
        assert m.device == cuda and m.flatten().tolist() == [1, 3, 5]
        assert ops.tree_mask_from_parents([], device).device == cuda
    assert ops.tree_mask_from_parents([[-1]]).device.type == "cpu"
