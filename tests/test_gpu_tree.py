"""Drafted-tree attention on the GPU against the 64-bit oracle, over 16-bit and
8-bit caches: trees, chains, rows that see nothing, special values in hidden
rows, ragged batches, splits, streams and captured graphs."""

import random
import types

import pytest
import torch

from litevllm_b200 import _lib, model_hooks, ops
from litevllm_b200.attention import Attention
from litevllm_b200.sampler import Sampler
from oracle import kv_q8
from oracle import logits as olog
from oracle import tree_attention
from tests.spec_inputs import (EPS, assert_attention, bits_of, cache_for, on, randn, random_tree,
                               row_bounds, tables_for)

pytestmark = pytest.mark.gpu

INT8, E4M3 = torch.int8, torch.float8_e4m3fn
BF16, F16 = torch.bfloat16, torch.float16


def case(kind, dtype, H, H_kv, D, bs, ctx, counts, seed, chain=False):
    rng = random.Random(seed)
    tables, pool = tables_for(ctx, bs, seed)
    kd, ks = cache_for(kind, pool, bs, H_kv, D, seed * 7 + 1, dtype)
    vd, vs = cache_for(kind, pool, bs, H_kv, D, seed * 7 + 2, dtype)
    q = randn(seed * 7 + 3, sum(counts), H, D, dtype=dtype)
    parents = [random_tree(rng, n) for n in counts]
    masks = [None if chain else bits_of(p) for p in parents]
    cu = torch.tensor([0] + counts, dtype=torch.int32).cumsum(0).int()
    return dict(q=q, kd=kd, ks=ks, vd=vd, vs=vs, tables=tables, ctx=ctx, counts=counts, cu=cu,
                masks=masks, mask=None if chain else ops.tree_mask_from_parents(parents),
                scale=D ** -0.5)


def run(c, dev, **kw):
    return ops.paged_tree_attention(
        c["q"].to(dev), on(dev, c["kd"], c["ks"]), on(dev, c["vd"], c["vs"]), c["tables"].to(dev),
        torch.tensor(c["ctx"], dtype=torch.int32).to(dev), c["cu"].to(dev), max(c["counts"]),
        c["scale"], tree_mask=None if c["mask"] is None else c["mask"].to(dev), **kw)


def expect(c):
    return tree_attention.tree(c["q"], c["kd"], c["ks"], c["vd"], c["vs"], c["tables"], c["ctx"],
                               c["counts"], c["masks"], c["scale"])


def check(c, got):
    want, size = expect(c)
    eps = EPS[c["q"].dtype] if c["ks"] is None else 2.0 ** -11
    assert_attention(got, want, size, c["q"], row_bounds(c["kd"], c["ks"], c["vd"], c["vs"]), c["scale"], max(c["ctx"]), eps)


SHAPES = [  # (H, H_kv, D, bs, ctx, counts)
    (1, 1, 64, 16, [1], [1]),
    (4, 1, 128, 16, [5], [5]),                                       # the whole context is drafted
    (32, 8, 128, 16, [40, 300, 17, 1000], [5, 5, 5, 5]),
    (32, 8, 128, 16, [333, 64, 65, 33, 0], [1, 64, 33, 0, 0]),       # ragged, empty
    (8, 8, 64, 24, [700, 90], [20, 31]),                             # G = 1
    (15, 3, 128, 8, [259, 259, 2100], [7, 3, 12]),                   # G = 5, drafts across a split
    (16, 2, 64, 16, [600, 128, 45], [2, 1, 2]),                      # 16 rows
    (12, 1, 128, 32, [515, 80], [64, 40]),                           # G = 12
    (4, 2, 64, 16, [400, 129], [130, 70]),                           # masks of three words
    # enough work for the tcgen05 kernel: 16-row groups to several tiles of 128 rows
    (32, 8, 128, 16, [2100, 700, 64, 33], [40, 64, 64, 1]),
    (8, 2, 64, 32, [1500, 900], [100, 130]),
    (20, 4, 128, 48, [900, 1300, 0], [60, 17, 0]),                   # G = 5
    (24, 1, 64, 16, [4097], [24]),                                   # G = 24, many splits
    (32, 8, 128, 16, [2049] * 3, [8] * 3),                           # one key past a split
]


@pytest.mark.parametrize("kind", [None, INT8, E4M3])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape", SHAPES, ids=range(len(SHAPES)))
def test_tree_matches_oracle(cuda, kind, dtype, shape):
    for chain in (False, True):
        c = case(kind or dtype, dtype, *shape, seed=len(shape[4]), chain=chain)
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        check(c, run(c, cuda, status=status))
        assert status.item() == 0


@pytest.mark.parametrize("kind", [BF16, INT8])
def test_rows_that_see_nothing_are_nan(cuda, kind):
    """No prior and an empty mask row; with a prior an empty mask row sees that."""
    c = case(kind, BF16, 4, 2, 64, 16, [6, 40], [6, 6], seed=3)
    for b in range(2):
        for i in (0, 4):
            c["masks"][b][i] = 0
            c["mask"][6 * b + i] = 0
    got = run(c, cuda)
    assert torch.isnan(got[[0, 4]]).all() and torch.isfinite(got[[1, 2, 3, 5]]).all()
    assert torch.isfinite(got[6:]).all()
    check(c, got)


@pytest.mark.parametrize("kind", [BF16, F16, INT8, E4M3])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("shape", [(8, 2, 128, 16, [50, 37], [9, 20]),
                                   (32, 8, 128, 16, [600, 337], [40, 64]),
                                   (32, 8, 64, 32, [651, 300], [40, 64]),
                                   (32, 8, 128, 16, [600, 337], [9, 20])], ids=range(4))
def test_special_values_in_hidden_drafts_do_not_leak(cuda, kind, where, value, shape):
    """A drafted token with a NaN or an infinity changes the rows that see it and
    no other."""
    dtype = kind if kind in (BF16, F16) else BF16
    c = case(kind, dtype, *shape, seed=8)
    bad = 2  # of both sequences, seen by its descendants only
    for b, (n, ctx) in enumerate(zip(c["counts"], c["ctx"])):
        key = ctx - n + bad
        bs = c["kd"].shape[1]
        blk, off = c["tables"][b, key // bs], key % bs
        if c["ks"] is None:
            c[where + "d"][blk, off, :, 5:7] = value
        else:  # the 8-bit store keeps such a row as zeros with scale NaN
            c[where + "d"].view(torch.uint8)[blk, off] = 0
            c[where + "s"][blk, :, off] = float("nan")
    got = run(c, cuda).cpu()
    clean = [not m >> bad & 1 for ms in c["masks"] for m in ms]
    assert any(clean) and not all(clean)
    assert torch.isfinite(got[clean]).all()
    if where == "v" or c["ks"] is not None or value != value:  # an infinite K may give a weight of 0
        assert not torch.isfinite(got[[not x for x in clean]]).all(-1).any()
    if where == "v" and c["ks"] is None:  # only the two columns are touched
        assert torch.isfinite(got[..., :5]).all() and torch.isfinite(got[..., 7:]).all()
    check(c, got)


def test_out_rows_of_no_sequence_are_left(cuda):
    c = case(BF16, BF16, 4, 2, 64, 16, [30, 600], [3, 4], seed=4)
    c["q"] = torch.cat([randn(1, 2, 4, 64, dtype=BF16), c["q"], randn(2, 3, 4, 64, dtype=BF16)])
    c["mask"] = torch.cat([torch.zeros(2, 1, dtype=torch.int64), c["mask"],
                           torch.zeros(3, 1, dtype=torch.int64)])
    c["cu"] = c["cu"] + 2
    out = torch.full((12, 4, 64), 5.0, dtype=BF16, device=cuda)
    got = run(c, cuda, out=out)
    assert got is out and (out[:2] == 5).all() and (out[9:] == 5).all()
    c["q"] = c["q"][2:9]
    check(c, out[2:9])


def test_strided_query_and_out(cuda):
    c = case(INT8, BF16, 8, 2, 64, 16, [300, 31], [6, 6], seed=5)
    wide = torch.zeros((12, 10, 64), dtype=BF16)
    wide[:, 1:9] = c["q"]
    out = torch.empty((12, 3, 8, 64), dtype=BF16, device=cuda)[:, 1]
    got = ops.paged_tree_attention(
        wide.cuda()[:, 1:9], on(cuda, c["kd"], c["ks"]), on(cuda, c["vd"], c["vs"]),
        c["tables"].cuda(), torch.tensor(c["ctx"], dtype=torch.int32).cuda(), c["cu"].cuda(), 6,
        c["scale"], tree_mask=c["mask"].cuda(), out=out)
    check(c, got)


def test_bad_sequences_are_flagged(cuda):
    """cu_seqlens_q past the queries, more tokens than max_q_len, a context
    shorter than its drafts: flagged, and nothing outside is touched."""
    c = case(BF16, BF16, 4, 2, 64, 16, [40, 40], [4, 4], seed=6)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    args = (c["q"].cuda(), on(cuda, c["kd"], None), on(cuda, c["vd"], None), c["tables"].cuda())
    good = run(c, cuda)
    for ctx, cu, most in (((40, 40), (0, 4, 30), 4), ((40, 40), (0, 4, 30), 64),
                          ((40, 40), (0, 4, 8), 3), ((40, 2), (0, 4, 8), 4),
                          ((40, 999), (0, 4, 8), 4), ((40, 40), (0, 4, -9), 4)):
        status.zero_()
        got = ops.paged_tree_attention(*args, i32(*ctx), i32(*cu), most, c["scale"],
                                       tree_mask=c["mask"].cuda(), status=status)
        torch.cuda.synchronize()
        if cu[2] > 0:
            assert status.item() & _lib.LK_STATUS_CTX_OOB, (ctx, cu, most)
        if most >= 4:
            assert torch.equal(got[:4], good[:4])


def test_decode_and_chain_of_one_agree(cuda):
    """One token per sequence: paged_decode_q8 and the tree call give one result;
    over a 16-bit cache the tree call agrees with paged_decode."""
    ctx = [1, 90, 700]
    for kind in (INT8, BF16):
        c = case(kind, BF16, 8, 2, 128, 16, ctx, [1, 1, 1], seed=7, chain=True)
        got = run(c, cuda)
        k, v = on(cuda, c["kd"], c["ks"]), on(cuda, c["vd"], c["vs"])
        lens = torch.tensor(ctx, dtype=torch.int32, device=cuda)
        if kind is INT8:
            assert torch.equal(got, ops.paged_decode_q8(c["q"].cuda(), k, v, c["tables"].cuda(),
                                                        lens, c["scale"]))
        else:
            check(c, ops.paged_decode(c["q"].cuda(), k, v, c["tables"].cuda(), lens, c["scale"]))
        check(c, got)


@pytest.mark.parametrize("kind", [BF16, F16, INT8, E4M3])
@pytest.mark.parametrize("D", [64, 128])
def test_stale_rows_behind_a_context_are_not_used(cuda, kind, D):
    """What other sequences left behind a context in its last block may be NaN; more
    than one split, and a last chunk with few keys."""
    dtype = kind if kind in (BF16, F16) else BF16
    c = case(kind, dtype, 32, 8, D, 32, [2055, 1000, 37], [8, 40, 33], seed=6)
    for b, ctx in enumerate(c["ctx"]):
        blk, off = c["tables"][b, ctx // 32], ctx % 32
        for x in ("k", "v"):
            if c["ks"] is None:
                c[x + "d"][blk, off:] = float("nan")
            else:
                c[x + "d"].view(torch.uint8)[blk, off:] = 0x7F  # NaN in e4m3
                c[x + "s"][blk, :, off:] = float("nan")
    check(c, run(c, cuda))
    q = c["q"][:3]
    if c["ks"] is not None:
        got = ops.paged_decode_q8(q.cuda(), on(cuda, c["kd"], c["ks"]), on(cuda, c["vd"], c["vs"]),
                                  c["tables"].cuda(), torch.tensor(c["ctx"], dtype=torch.int32).cuda(),
                                  c["scale"])
        want, size = tree_attention.decode(q, c["kd"], c["ks"], c["vd"], c["vs"], c["tables"], c["ctx"], c["scale"])
        assert_attention(got, want, size, q, row_bounds(c["kd"], c["ks"], c["vd"], c["vs"]), c["scale"],
                         max(c["ctx"]), 2.0 ** -11)


@pytest.mark.parametrize("kind", [BF16, INT8])
@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_any_scale(cuda, kind, scale):
    for shape in ((8, 2, 64, 16, [90, 300], [6, 9]), (32, 8, 64, 16, [700, 300], [40, 64])):
        c = case(kind, BF16, *shape, seed=2)
        c["scale"] = scale
        check(c, run(c, cuda))


@pytest.mark.parametrize("kind", [BF16, E4M3])
@pytest.mark.parametrize("rows", ["few", "many"])
def test_streams_and_graphs_do_not_share_state(cuda, kind, rows):
    """Two captured graphs of split calls replayed at once on two streams, and
    eager calls beside them, give each its own result."""
    n = [6, 3] if rows == "few" else [64, 50]
    cs = [case(kind, BF16, 8, 2, 128, 16, [3000 + 50 * i, 900], n, seed=10 + i) for i in range(2)]
    state, want, graphs, outs = [], [], [], []
    for c in cs:
        state.append((c["q"].cuda(), on(cuda, c["kd"], c["ks"]), on(cuda, c["vd"], c["vs"]),
                      c["tables"].cuda(), torch.tensor(c["ctx"], dtype=torch.int32).cuda(),
                      c["cu"].cuda(), max(n), c["scale"], c["mask"].cuda()))
    call = lambda s: ops.paged_tree_attention(*s[:8], tree_mask=s[8])  # noqa: E731
    want = [call(s) for s in state]
    for c, w in zip(cs, want):
        check(c, w)
    torch.cuda.synchronize()
    for s in state:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(s))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        eager = call(state[1])
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
        assert torch.equal(eager, want[1])


def test_caller_owned_workspace(cuda):
    c = case(INT8, BF16, 8, 2, 128, 16, [9000, 20], [4, 4], seed=12)
    need = ops.tree_workspace_bytes(8, 2, 4, 8, 2, 128, 16, c["tables"].shape[1], INT8)
    assert need > 0
    got = run(c, cuda, workspace=torch.empty(need, dtype=torch.uint8, device=cuda))
    assert torch.equal(got, run(c, cuda))
    with pytest.raises(ValueError, match="workspace"):
        run(c, cuda, workspace=torch.empty(need - 1, dtype=torch.uint8, device=cuda))


@pytest.mark.parametrize("kind", [None, INT8, E4M3])
def test_speculative_step(cuda, kind):
    """The whole step through the drop-in classes: the prompt is stored and
    attended, drafted tokens are stored and attended as a tree, their logits are
    processed and sampled greedily; then the accepted path is decoded."""
    H, H_kv, D, bs, V = 8, 2, 128, 16, 1000
    B, prompt, n = 2, 45, 6
    attn = Attention(H, D, H_kv)
    blocks = 5
    tables = torch.arange(B * blocks, dtype=torch.int32, device=cuda).view(B, blocks).flip(0)
    if kind is None:
        kc, vc = (torch.zeros((B * blocks, bs, H_kv, D), dtype=BF16, device=cuda) for _ in range(2))
    else:
        kc, vc = (ops.new_quantized_cache(B * blocks, bs, H_kv, D, kind) for _ in range(2))
    ctx0 = torch.full((B,), prompt, dtype=torch.int32, device=cuda)

    def slots_of(b, lo, hi):
        p = torch.arange(lo, hi, device=cuda)
        return tables[b, p // bs].long() * bs + p % bs

    # prompts: stored, then chunked prefill over the cache
    pk, pv = (randn(s, B * prompt, H_kv, D, dtype=BF16).cuda() for s in (1, 2))
    pq = randn(3, B * prompt, H, D, dtype=BF16).cuda()
    slots = torch.cat([slots_of(b, 0, prompt) for b in range(B)])
    cu = torch.arange(0, B * prompt + 1, prompt, dtype=torch.int32, device=cuda)
    o = attn.forward(pq, pk, pv, kc, vc, tables, slots, ctx0, is_prefill=True, cu_seqlens_q=cu,
                     max_q_len=prompt)
    host = lambda c: (c.cpu(), None) if kind is None else (c.data.cpu(), c.scale.cpu())  # noqa: E731
    want, size = tree_attention.tree(pq.cpu(), *host(kc), *host(vc), tables.cpu(), [prompt] * B,
                                     [prompt] * B, [None] * B, attn.scale)
    # the 8-bit rows are rounded to bf16 for the prefill kernel (K: the score moves
    # by 2^-8 of its terms), its weights too
    assert (o.double().cpu() - want).abs().max() <= 2 ** -8 * want.abs().max() + 8 * 2 ** -8 * size.max()

    parents = [[-1, 0, 0, 1, 2, 2], [-1, 0, 1, 0, 3, 4]]
    mask = ops.tree_mask_from_parents(parents, cuda)
    dk, dv = (randn(s, B * n, H_kv, D, dtype=BF16).cuda() for s in (4, 5))
    dq = randn(6, B * n, H, D, dtype=BF16).cuda()
    slots = torch.cat([slots_of(b, prompt, prompt + n) for b in range(B)])
    ctx1 = ctx0 + n
    cu = torch.arange(0, B * n + 1, n, dtype=torch.int32, device=cuda)
    o = attn.forward_tree(dq, dk, dv, kc, vc, tables, slots, ctx1, cu, n, mask)
    want, size = tree_attention.tree(dq.cpu(), *host(kc), *host(vc), tables.cpu(), [prompt + n] * B,
                                     [n] * B, [bits_of(p) for p in parents], attn.scale)
    bounds = lambda: row_bounds(*host(kc), *host(vc))  # noqa: E731
    assert_attention(o, want, size, dq.cpu(), bounds(), attn.scale, prompt + n,
                     EPS[BF16] if kind is None else EPS[F16])

    # their logits: penalties, a bias and a grammar, then greedy ids
    logits = randn(7, B * n, V, dtype=BF16, std=3.0)
    past = torch.randint(0, V, (B * n, 30), generator=torch.Generator().manual_seed(1))
    allowed = torch.rand((B * n, V), generator=torch.Generator().manual_seed(2)) < 0.3
    words = torch.zeros((B * n, -(-V // 32)), dtype=torch.int64)
    for v in range(V):
        words[:, v // 32] |= allowed[:, v].long() << (v % 32)
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words).int()
    freq = torch.full((B * n,), 0.5)
    ids = Sampler.sample_batch(logits.cuda(), processing=dict(
        output_ids=past.cuda(), frequency=freq.cuda(), allowed=words.cuda()))
    x = olog.process(logits.double().numpy(), output=past.tolist(), frequency=freq.numpy(),
                     allowed=allowed.numpy())
    x = torch.from_numpy(x).float().bfloat16().float()
    assert torch.equal(ids.cpu(), x.argmax(-1))

    # decode the next token of each sequence over what was stored
    q = randn(8, B, H, D, dtype=BF16).cuda()
    k, v = (randn(s, B, H_kv, D, dtype=BF16).cuda() for s in (9, 10))
    slots = torch.cat([slots_of(b, prompt + n, prompt + n + 1) for b in range(B)])
    o = attn.forward(q, k, v, kc, vc, tables, slots, ctx1 + 1, is_prefill=False)
    want, size = tree_attention.decode(q.cpu(), *host(kc), *host(vc), tables.cpu(),
                                       [prompt + n + 1] * B, attn.scale)
    assert_attention(o, want, size, q.cpu(), bounds(), attn.scale, prompt + n + 1,
                     EPS[BF16] if kind is None else EPS[F16])


@pytest.mark.parametrize("kind", [INT8, E4M3])
def test_mixed_step_over_an_8bit_cache(cuda, kind):
    """Prefill chunks and decodes of one merged step read the 8-bit cache."""
    H, H_kv, D, bs = 8, 2, 128, 16
    ctx, q_lens = [60, 33, 20], [20, 1, 1]
    tables, pool = tables_for(ctx, bs, 9)
    kd, ks = cache_for(kind, pool, bs, H_kv, D, 1, BF16)
    vd, vs = cache_for(kind, pool, bs, H_kv, D, 2, BF16)
    q = randn(3, 22, H, D, dtype=BF16)
    attn = Attention(H, D, H_kv)
    got = attn.forward_mixed(q.cuda(), None, None, on(cuda, kd, ks), on(cuda, vd, vs), tables.cuda(),
                             None, torch.tensor(ctx, dtype=torch.int32).cuda(),
                             torch.tensor([0, 20], dtype=torch.int32).cuda(), 1, 20, 20)
    want, size = tree_attention.tree(q, kd, ks, vd, vs, tables, ctx, q_lens, [None] * 3, attn.scale)
    assert (got.double().cpu() - want).abs().max() <= 2 ** -8 * want.abs().max() + 16 * 2 ** -8 * size.max()


@pytest.mark.parametrize("kind", [INT8, E4M3])
def test_fused_block_writes_and_reads_an_8bit_cache(cuda, kind):
    """The fused attention block over an 8-bit cache: it holds the rows that the
    16-bit cache gets, quantised, and a decode step attends to them."""
    H, H_kv, D, bs, hidden, S = 8, 2, 128, 16, 64, 21
    dev = dict(device=cuda, dtype=BF16)
    m = types.SimpleNamespace(num_heads=H, num_kv_heads=H_kv, head_dim=D, o_proj=lambda x: x)
    for i, (name, n) in enumerate((("q_proj", H), ("k_proj", H_kv), ("v_proj", H_kv))):
        w = randn(40 + i, hidden, n * D, dtype=BF16).to(cuda)
        setattr(m, name, lambda x, w=w: x @ w)
    angle = torch.arange(64, device=cuda)[:, None] * 0.01 * torch.arange(D // 2, device=cuda)
    m.rotary_emb = types.SimpleNamespace(cos_cached=angle.cos(), sin_cached=angle.sin())
    queries = []

    class Recording(Attention):
        def forward(self, query, *args, **kw):
            queries.append(query.clone())
            return super().forward(query, *args, **kw)

    m.attn = Recording(H, D, H_kv)
    x = randn(44, S + 1, hidden, dtype=BF16).to(cuda)
    pos, slots = torch.arange(S + 1, device=cuda), torch.arange(16, S + 17, device=cuda)
    table = torch.tensor([[1, 2]], dtype=torch.int32, device=cuda)
    out = {}
    for cache in ("16", "8"):
        kc, vc = ([torch.zeros(4, bs, H_kv, D, **dev) for _ in range(2)] if cache == "16" else
                  [ops.new_quantized_cache(4, bs, H_kv, D, kind, device=cuda) for _ in range(2)])
        for rows, prefill in ((slice(0, S), True), (slice(S, S + 1), False)):
            y = model_hooks.fused_forward(
                m, x[rows], pos[rows], (kc, vc), slots[rows], None if prefill else table,
                None if prefill else torch.tensor([S + 1], dtype=torch.int32, device=cuda), prefill)
        out[cache] = kc, vc, y
    for wide, (data, scale) in zip(out["16"][:2], out["8"][:2]):
        q, s = kv_q8.quantise(wide.view(-1, H_kv, D)[16:S + 17].cpu(), kind)
        assert torch.equal(data.view(-1, H_kv, D)[16:S + 17].float().cpu().double(), q)
        assert torch.equal(scale.transpose(1, 2).reshape(-1, H_kv)[16:S + 17].cpu(), s)
    (kd, ks), (vd, vs), y = out["8"]
    kd, ks, vd, vs = (t.cpu() for t in (kd, ks, vd, vs))
    q = queries[-1].cpu()
    want, size = tree_attention.tree(q, kd, ks, vd, vs, table.cpu(), [S + 1], [1], [None], m.attn.scale)
    assert_attention(y.view(1, H, D), want, size, q, row_bounds(kd, ks, vd, vs), m.attn.scale, S + 1, EPS[F16])
