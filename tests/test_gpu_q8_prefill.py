"""Prefill over an 8-bit cache on the GPU: the contexts are read back into 16-bit
blocks, rounded once more, and attended by the prefill kernel."""

import sys
import types

import pytest
import torch

from litevllm_b200 import _lib, attention, engine_hooks, ops
from litevllm_b200.attention import Attention
from oracle import kv_q8, tree_attention
from tests.spec_inputs import EPS, assert_attention, cache_for, on, randn, row_bounds, tables_for

pytestmark = pytest.mark.gpu

INT8, E4M3 = torch.int8, torch.float8_e4m3fn
BF16, F16 = torch.bfloat16, torch.float16


def rounded(data, scale, dtype):
    """A 16-bit cache of an 8-bit one's rows: fp32 products, rounded to the type."""
    return (data.float() * scale.transpose(1, 2)[..., None]).to(dtype)


def case(kind, dtype, H, H_kv, D, bs, ctx, q_lens, seed, width=0):
    tables, pool = tables_for(ctx, bs, seed)
    if width > tables.shape[1]:
        tables = torch.cat([tables, torch.zeros((len(ctx), width - tables.shape[1]), dtype=torch.int32)], 1)
    kd, ks = cache_for(kind, pool, bs, H_kv, D, seed * 5 + 1, dtype)
    vd, vs = cache_for(kind, pool, bs, H_kv, D, seed * 5 + 2, dtype)
    q = randn(seed * 5 + 3, sum(q_lens), H, D, dtype=dtype)
    return dict(q=q, kd=kd, ks=ks, vd=vd, vs=vs, tables=tables, ctx=ctx, q_lens=q_lens,
                cu=torch.tensor([0] + q_lens).cumsum(0).int(), attn=Attention(H, D, H_kv))


def run(c, dev):
    return c["attn"].forward(
        c["q"].to(dev), None, None, on(dev, c["kd"], c["ks"]), on(dev, c["vd"], c["vs"]), c["tables"].to(dev),
        None, torch.tensor(c["ctx"], dtype=torch.int32).to(dev), is_prefill=True,
        cu_seqlens_q=c["cu"].to(dev), max_q_len=max(c["q_lens"]))


def check(c, got):
    """Within the bound of attention over the rounded rows: weights and result are
    rounded to the query's type."""
    dtype = c["q"].dtype
    kd, vd = rounded(c["kd"], c["ks"], dtype), rounded(c["vd"], c["vs"], dtype)
    want, size = tree_attention.tree(c["q"], kd, None, vd, None, c["tables"], c["ctx"], c["q_lens"],
                                     [None] * len(c["ctx"]), c["attn"].scale)
    assert_attention(got, want, size, c["q"], row_bounds(kd, None, vd, None), c["attn"].scale,
                     max(c["ctx"]), EPS[dtype])


SHAPES = [  # (H, H_kv, D, bs, ctx, q_lens, table width)
    (8, 2, 128, 16, [45, 45], [45, 45], 0),
    (32, 8, 128, 16, [1, 300, 129, 64], [1, 40, 129, 1], 200),
    (8, 8, 128, 32, [65, 31], [2, 31], 7),
    (4, 2, 64, 16, [100, 33], [50, 33], 40),      # the generic kernel
    (6, 2, 128, 24, [100, 23], [9, 23], 30),      # the same: G = 3, blocks of 24
]


@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape", SHAPES, ids=range(len(SHAPES)))
def test_equals_attention_over_the_rounded_rows(cuda, monkeypatch, kind, dtype, shape):
    c = case(kind, dtype, *shape[:6], seed=len(shape[4]), width=shape[6])
    check(c, run(c, cuda))
    # a sequence at a time
    monkeypatch.setattr(attention, "Q8_PREFILL_BYTES", 1)
    check(c, run(c, cuda))


def test_space_does_not_pass_the_limit(cuda, monkeypatch):
    """Sixteen short contexts under a table of 512 blocks: 32 MB of K and V blocks a
    sequence, 64 MB at a time."""
    c = case(INT8, BF16, 32, 8, 128, 16, [40] * 16, [8] * 16, seed=4, width=512)
    monkeypatch.setattr(attention, "Q8_PREFILL_BYTES", 64 << 20)
    check(c, run(c, cuda))
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    run(c, cuda)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < (64 << 20) + (4 << 20)


@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [torch.float32, BF16, F16])
@pytest.mark.parametrize("H_kv,D,bs", [(1, 64, 16), (8, 128, 16), (3, 128, 24), (2, 64, 1)])
def test_blocks_of_a_context_are_written_and_no_other(cuda, kind, dtype, H_kv, D, bs):
    ctx, width = [0, 1, bs, 3 * bs + 1, 2 * bs], 9
    tables, pool = tables_for(ctx, bs, 3)
    tables = torch.cat([tables, torch.full((len(ctx), width - tables.shape[1]), 1 << 20, dtype=torch.int32)], 1)
    kd, ks = cache_for(kind, pool, bs, H_kv, D, 11, BF16)
    vd, vs = cache_for(kind, pool, bs, H_kv, D, 12, BF16)
    n = len(ctx) * width
    outs = [torch.full((n, bs, H_kv, D), 9.0, dtype=dtype, device=cuda) for _ in range(2)]
    numbers = torch.full((n,), -5, dtype=torch.int32, device=cuda)
    dev = [t.to(cuda) for t in (kd, ks, vd, vs, tables, torch.tensor(ctx, dtype=torch.int32))]
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    code = {torch.float32: 0, F16: 1, BF16: 2}[dtype]
    fmt = _lib.LK_KV_INT8 if kind is INT8 else _lib.LK_KV_E4M3
    _lib.check(_lib.lib().lk_load_kv_q8_blocks(
        outs[0].data_ptr(), outs[1].data_ptr(), numbers.data_ptr(), *(t.data_ptr() for t in dev[:5]), width,
        dev[5].data_ptr(), len(ctx), H_kv, D, pool, bs, width, code, fmt, status.data_ptr(),
        torch.cuda.current_stream().cuda_stream))
    assert status.item() == 0 and numbers.tolist() == list(range(n))
    for out, d, s in ((outs[0], kd, ks), (outs[1], vd, vs)):
        want = torch.full((len(ctx), width * bs, H_kv, D), 9.0, dtype=torch.float64)
        for b, c in enumerate(ctx):
            want[b, :-(-c // bs) * bs] = 0.0
            want[b, :c] = kv_q8.rows(d, s, tables[b], c).float().to(dtype).double()
        assert torch.equal(out.double().cpu().view_as(want), want)
    # the same through ops, where what is not written may hold anything
    k, v, t = ops.load_kvcache_q8_blocks(ops.QuantizedCache(*dev[:2]), ops.QuantizedCache(*dev[2:4]), dev[4],
                                         dev[5], dtype=dtype)
    assert t.flatten().tolist() == list(range(n))
    for b, c in enumerate(ctx):
        some = slice(b * width, b * width + -(-c // bs))
        assert torch.equal(k[some], outs[0][some]) and torch.equal(v[some], outs[1][some])


def test_bad_tables_are_flagged(cuda):
    kd, ks = cache_for(INT8, 2, 16, 1, 64, 1, BF16)
    c = on(cuda, kd, ks)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    k, _, _ = ops.load_kvcache_q8_blocks(c, c, i32(1, 2).view(1, 2), i32(20), status=status)
    assert status.item() == _lib.LK_STATUS_BLOCK_OOB
    assert (k[0] != 0).any() and (k[1] == 0).all()
    status.zero_()
    k, _, _ = ops.load_kvcache_q8_blocks(c, c, i32(1).view(1, 1), i32(20), status=status)
    assert status.item() == _lib.LK_STATUS_CTX_OOB and (k[0] != 0).any()
    status.zero_()
    k, v, t = ops.load_kvcache_q8_blocks(c, c, i32().view(0, 3), i32(), status=status)
    assert k.shape == v.shape == (0, 16, 1, 64) and t.shape == (0, 3)
    assert ops.load_kvcache_q8_blocks(c, c, i32().view(2, 0), i32(0, 0))[2].shape == (2, 0)
    assert ops.load_kvcache_q8_blocks(c, c, i32(0, 1).view(1, 2), i32(-4), status=status)[2].tolist() == [[0, 1]]
    assert status.item() == 0


def test_refusals(cuda):
    kd, ks = cache_for(INT8, 2, 16, 1, 64, 1, BF16)
    c = on(cuda, kd, ks)
    bt, ctx = (torch.ones(s, dtype=torch.int32, device=cuda) for s in ((2, 3), 2))
    f = ops.load_kvcache_q8_blocks
    for error, match, args, kw in (
            (TypeError, "block_tables", (c, c, bt.long(), ctx), {}), (TypeError, "block_tables", (c, c, bt[0], ctx), {}),
            (TypeError, "context_lens", (c, c, bt, ctx[:1]), {}), (TypeError, "context_lens", (c, c, bt, ctx.long()), {}),
            (TypeError, "dtype", (c, c, bt, ctx), dict(dtype=torch.float64)),
            (TypeError, "dtype", (c, c, bt, ctx), dict(dtype="bf16")),
            (TypeError, "both", (c, c.data, bt, ctx), {}), (RuntimeError, "CUDA", (c, c, bt.cpu(), ctx), {}),
            (TypeError, "status", (c, c, bt, ctx), dict(status=ctx.long()))):
        with pytest.raises(error, match=match):
            f(*args, **kw)
    with pytest.raises(ValueError, match="columns"):
        Attention(2, 64, 1).forward(torch.zeros((3, 2, 64), dtype=BF16, device=cuda), None, None, c, c, bt[:1, :0],
                                    None, ctx[:1], is_prefill=True)


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


def test_captured_graph_follows_the_contexts(cuda):
    c = case(INT8, BF16, 8, 2, 128, 16, [100, 70], [20, 30], seed=6, width=12)
    dev = dict(q=c["q"].to(cuda), k=on(cuda, c["kd"], c["ks"]), v=on(cuda, c["vd"], c["vs"]), t=c["tables"].to(cuda),
               ctx=torch.tensor(c["ctx"], dtype=torch.int32, device=cuda), cu=c["cu"].to(cuda))
    call = lambda: c["attn"].forward(  # noqa: E731
        dev["q"], None, None, dev["k"], dev["v"], dev["t"], None, dev["ctx"], is_prefill=True,
        cu_seqlens_q=dev["cu"], max_q_len=30)
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    for ctx in ([100, 70], [20, 70], [93, 31]):
        dev["ctx"].copy_(torch.tensor(ctx, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        c["ctx"] = ctx
        check(c, out)


@pytest.mark.parametrize("kind", [INT8, E4M3])
def test_merged_step_beside_a_long_decode(cuda, monkeypatch, kind):
    """engine_hooks.prepare_inputs_mixed gives the prefill rows' own width: eight
    short prompts beside one decode of 8000 tokens take space for their contexts."""
    H, H_kv, D, bs = 8, 2, 128, 16
    prompts, long = [37, 20, 5, 64, 65, 100, 1, 30], 8000
    ctx = prompts + [long]
    tables, pool = tables_for(ctx, bs, 2)
    groups = []
    for i, n in enumerate(ctx):
        data = types.SimpleNamespace(prompt_len=min(n, long - 1), prompt_token_ids=[3] * n, all_token_ids=[3] * n,
                                     total_len=n)
        seq = types.SimpleNamespace(seq_id=i, data=data, num_computed_tokens=0 if n < long else n, is_prefill=n < long)
        groups.append(types.SimpleNamespace(get_unfinished_seqs=lambda s=seq: [s]))
    held = lambda i: types.SimpleNamespace(physical_block_ids=tables[i, :-(-ctx[i] // bs)].tolist())  # noqa: E731
    runner = types.SimpleNamespace(config=types.SimpleNamespace(cache_config=types.SimpleNamespace(block_size=bs)),
                                   device=str(cuda))
    monkeypatch.setattr(sys.modules[type(runner).__module__], "InputMetadata", types.SimpleNamespace, raising=False)
    md = engine_hooks.prepare_inputs_mixed(runner, groups[:-1], groups[-1:],
                                           types.SimpleNamespace(get_block_table=held))
    try:
        assert attention._MIXED_STEP["max_prefill_blocks"] == 7 and md.block_tables.shape == (9, 500)
        kd, ks = cache_for(kind, pool, bs, H_kv, D, 21, BF16)
        vd, vs = cache_for(kind, pool, bs, H_kv, D, 22, BF16)
        k, v = on(cuda, kd, ks), on(cuda, vd, vs)
        N = md.input_ids.numel()
        q, new_k, new_v = (randn(s, N, h, D, dtype=BF16) for s, h in ((1, H), (2, H_kv), (3, H_kv)))
        attn = Attention(H, D, H_kv)
        args = (q.to(cuda), new_k.to(cuda), new_v.to(cuda), k, v, md.block_tables, md.slot_mapping, md.context_lens)
        attn.forward(*args, md.is_prefill)  # the kernels' own workspaces exist from here on
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        got = attn.forward(*args, md.is_prefill)
        torch.cuda.synchronize()
        # eight tables of 500 blocks would be 64 MB, of seven 0.9 MB
        assert torch.cuda.max_memory_allocated() - before < 16 << 20
        host = [t.cpu() for t in (*k, *v)]
        TP = sum(prompts)
        c = dict(q=q[:TP], kd=host[0], ks=host[1], vd=host[2], vs=host[3], tables=tables, ctx=prompts, q_lens=prompts,
                 attn=attn)
        check(c, got[:TP])
        want, size = tree_attention.decode(q[TP:], *host, tables[8:], [long], attn.scale)
        assert_attention(got[TP:], want, size, q[TP:], row_bounds(*host), attn.scale, long, EPS[F16])
    finally:
        attention.set_mixed_step_hint(None)
