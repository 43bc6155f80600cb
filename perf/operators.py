"""Measured cases of the speculative-decoding operators: the 8-bit KV cache
(quantised as it is written, read back, read by decode attention), attention
for a tree of drafted tokens over the paged cache, and the processing of a
step's logits (penalties, biases, grammar masks).

With `own` false, run() computes each operator from its formula in elementary
torch operations (32 bits, rounded once); with `own` true it calls
litevllm_b200.ops. exact() gives the same results in 64 bits.

Quantised row x[0..D) of one token and KV head, M = 127 (int8) or 448 (e4m3):
    a = max(max|x|, 2^-100), scale = RN32(a / M), r = RN32(M / a)
    int8: q = rint(x r) of the exact product;  e4m3: q = RN_e4m3(RN32(x r))
Cache data [num_blocks, bs, H_kv, D], scales [num_blocks, H_kv, bs] fp32.
"""

import math
import random

import torch

own = False

M_OF = {"int8": 127.0, "e4m3": 448.0}
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "int8": torch.int8,
         "e4m3": torch.float8_e4m3fn}
FLOOR = 2.0 ** -100


def _case(name, op, **kw):
    return dict(name=name, op=op, **kw)


def listed():
    gqa = dict(H=32, H_kv=8, D=128, bs=16)  # the attention shapes of configurations 2 to 5
    return [
        # one decode step's 256 new tokens into an int8 cache
        _case("store_step_int8", "store", T=256, H_kv=8, D=128, bs=16, dtype="bf16", cache="int8", plan=1),
        # prompts of 16K tokens in all into an e4m3 cache
        _case("store_prompts_e4m3", "store", T=16384, H_kv=8, D=128, bs=16, dtype="bf16", cache="e4m3", plan=2),
        # four prefill chunks read their prior context back (configuration 3's priors)
        _case("load_priors_int8", "load", B=4, lo=0, hi=3584, H_kv=8, D=128, bs=16, dtype="bf16", cache="int8", plan=3),
        # two long contexts read back
        _case("load_long_e4m3", "load", B=2, lo=30000, hi=40000, H_kv=8, D=128, bs=16, dtype="bf16", cache="e4m3", plan=4),
        # one user's step: latency
        _case("decode_one_int8", "decode", B=1, lo=777, hi=777, **gqa, dtype="bf16", cache="int8", plan=5),
        # configuration 2's batch over an e4m3 cache
        _case("decode_batch_e4m3", "decode", B=256, lo=16, hi=4096, **gqa, dtype="bf16", cache="e4m3", plan=6),
        # long contexts, few rows: split over the context
        _case("decode_long_int8", "decode", B=8, lo=16384, hi=32768, **gqa, dtype="bf16", cache="int8", plan=7),
        # a chain of four drafted tokens after the last accepted one, four users
        _case("tree_chain_bf16", "tree", B=4, lo=200, hi=1100, n_lo=5, n_hi=5, **gqa, dtype="bf16", cache="bf16", plan=8),
        # trees of up to 32 nodes for a batch (configuration 3's decode contexts)
        _case("tree_batch_bf16", "tree", B=32, lo=64, hi=2048, n_lo=20, n_hi=32, **gqa, dtype="bf16", cache="bf16", plan=9),
        # wide trees over an int8 cache
        _case("tree_wide_int8", "tree", B=16, lo=1024, hi=8192, n_lo=48, n_hi=64, **gqa, dtype="bf16", cache="int8", plan=10),
        # a serving step's logits: penalties over the histories, biases, every fourth row under a grammar
        _case("logits_step_bf16", "logits", B=128, V=151936, dtype="bf16", prompt=1024, output=512, bias=16, grammar=4, plan=11),
        # the drafted nodes of one constrained user, fp32 logits
        _case("logits_nodes_f32", "logits", B=8, V=128256, dtype="f32", prompt=300, output=40, bias=0, grammar=1, plan=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["store", "load", "decode", "decode", "tree", "tree", "logits"])
    plan = rng.randrange(1 << 30)
    if op == "logits":
        B = _log(rng, 1, 128)
        return dict(op=op, B=B, V=_log(rng, 1000, 151936), dtype=rng.choice(["bf16", "f16", "f32"][: 2 + (B <= 64)]),
                    prompt=_log(rng, 1, 1024), output=_log(rng, 1, 512), bias=rng.choice([0, 1, 7, 16]),
                    grammar=rng.choice([0, 1, 3, 4]), plan=plan)
    H_kv = rng.choice([1, 2, 4, 8])
    base = dict(op=op, H_kv=H_kv, D=rng.choice([64, 128]), bs=rng.choice([8, 16, 16, 24, 32]),
                dtype=rng.choice(["bf16", "f16"]), plan=plan)
    if op == "store":
        return dict(base, T=_log(rng, 1, 16384), cache=rng.choice(["int8", "e4m3"]))
    hi = _log(rng, 1, 16384)
    lo = rng.choice([hi, max(1, hi // 2), max(1, hi // 16), 1])
    if op == "load":
        return dict(base, B=max(1, min(_log(rng, 1, 64), 40000 // hi)), lo=lo, hi=hi, cache=rng.choice(["int8", "e4m3"]),
                    dtype=rng.choice(["bf16", "f16", "f32"]))
    G = rng.choice([1, 2, 3, 4, 5, 7, 8])
    if op == "decode":
        return dict(base, H=H_kv * G, B=max(1, min(_log(rng, 1, 256), 131072 // hi)), lo=lo, hi=hi, cache=rng.choice(["int8", "e4m3"]))
    n_hi = _log(rng, 1, 64)
    hi = max(min(hi, 8192), n_hi)
    return dict(base, H=H_kv * G, B=max(1, min(_log(rng, 1, 32), 65536 // hi, 2048 // (n_hi * G))), lo=max(n_hi, min(lo, hi)), hi=hi,
                n_lo=rng.choice([n_hi, max(1, n_hi // 2), 1]), n_hi=n_hi, cache=rng.choice([base["dtype"], "int8", "e4m3"]))


def _lengths(case):
    """Context lengths, and drafted tokens of a tree case, of the case's sequences."""
    rng = random.Random(case["plan"])
    if case["op"] == "decode" and case["B"] == 256 and case["hi"] == 4096:
        ctx = [min(max(round(math.exp(rng.gauss(math.log(1024.0), 0.5))), 16), 4096) for _ in range(256)]
    else:
        ctx = [rng.randint(case["lo"], case["hi"]) for _ in range(case["B"])]
    n = [rng.randint(case["n_lo"], case["n_hi"]) for _ in ctx] if case["op"] == "tree" else [1] * len(ctx)
    return ctx, n, rng


def _randn(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _rows(g, n, H_kv, D, dtype):
    """Keys or values as a model makes them: rows of different size, a few wide channels."""
    size = torch.exp(torch.randn((n, H_kv, 1), generator=g, device="cuda") * 0.3)
    wide = 1.0 + 3.0 * (torch.rand((1, H_kv, D), generator=g, device="cuda") < 0.03)
    return (torch.randn((n, H_kv, D), generator=g, device="cuda") * size * wide).to(dtype)


def _quantise(x, cache):
    """(data, scale) of rows x [..., D]."""
    m = M_OF[cache]
    x = x.float()
    a = x.abs().amax(-1, keepdim=True).clamp_min(FLOOR)
    fine = torch.isfinite(a)
    m = torch.full_like(a, m)  # a tensor: one correctly rounded division each
    scale = torch.where(fine, a / m, float("nan"))
    r = m / a
    if cache == "int8":
        q = (x.double() * r.double()).round()
    else:
        q = x * r
    return torch.where(fine, q, 0.0).to(TYPES[cache]), scale.squeeze(-1)


def _cache_of(g, case, blocks):
    """The paged K and V caches of a running server: every slot holds some token's row."""
    bs, H_kv, D = case["bs"], case["H_kv"], case["D"]
    got = []
    for _ in range(2):
        if case["cache"] in M_OF:
            data = torch.empty((blocks, bs, H_kv, D), dtype=TYPES[case["cache"]], device="cuda")
            scale = torch.empty((blocks, H_kv, bs), dtype=torch.float32, device="cuda")
            step = max(1, (1 << 26) // (bs * H_kv * D))
            for at in range(0, blocks, step):
                n = min(step, blocks - at)
                q, s = _quantise(_rows(g, n * bs, H_kv, D, torch.bfloat16), case["cache"])
                data[at:at + n] = q.view(n, bs, H_kv, D)
                scale[at:at + n] = s.view(n, bs, H_kv).transpose(1, 2)
            got += [data, scale]
        else:
            got += [_rows(g, blocks * bs, H_kv, D, TYPES[case["cache"]]).view(blocks, bs, H_kv, D), None]
    return got


def _tree_masks(n, rng):
    """One 64-bit word per drafted token: its ancestors and itself."""
    words = []
    for count in n:
        sees = []
        for i in range(count):
            parent = rng.randrange(max(0, i - 6), i) if i else -1
            sees.append((sees[parent] if i else 0) | (1 << i))
        words += [w - (1 << 64) if w >> 63 else w for w in sees]
    return torch.tensor(words, dtype=torch.int64).view(-1, 1).cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 17)
    s = dict(case=case)
    if case["op"] == "logits":
        B, V, Lp, Lo = case["B"], case["V"], case["prompt"], case["output"]
        rand = lambda *shape: torch.rand(shape, generator=g, device="cuda")  # noqa: E731
        s["logits"] = _randn(g, B, V, dtype=TYPES[case["dtype"]], std=3.0)
        s["prompt_ids"] = (V * rand(B, Lp) ** 3).long().clamp_max(V - 1)
        s["output_ids"] = (V * rand(B, Lo) ** 6).long().clamp_max(V - 1)
        s["prompt_lens"] = (1 + Lp * rand(B)).int().clamp_max(Lp)
        s["output_lens"] = ((1 + Lo) * rand(B)).int().clamp_max(Lo)
        s["repetition"] = torch.where(rand(B) < 0.3, 1.0, 1.0 + 0.3 * rand(B))
        s["presence"] = torch.where(rand(B) < 0.3, 0.0, rand(B))
        s["frequency"] = torch.where(rand(B) < 0.3, 0.0, 0.5 * rand(B))
        s["bias_ids"] = (V * rand(B, case["bias"])).long().clamp_max(V - 1) if case["bias"] else None
        s["bias"] = _randn(g, B, case["bias"], std=4.0) if case["bias"] else None
        s["allowed"] = None
        if case["grammar"]:
            words = torch.full((B, -(-V // 32)), -1, dtype=torch.int32, device="cuda")
            few = rand(B, words.shape[1]) < 0.05  # the grammar allows single tokens here and there
            bits = torch.where(few, 1 << (32 * rand(B, words.shape[1])).int().clamp_max(31), 0).int()
            held = torch.arange(B, device="cuda") % case["grammar"] == 0
            s["allowed"] = torch.where(held[:, None], bits, words)
        return s
    H_kv, D, bs = case["H_kv"], case["D"], case["bs"]
    rng = random.Random(case["plan"])
    if case["op"] == "store":
        T = case["T"]
        blocks = -(-T // bs) + 2
        # key and value are slices of one fused projection's output
        qkv = torch.cat([_rows(g, T, H_kv, D, TYPES[case["dtype"]]) for _ in range(3)], dim=1)
        s["key"], s["value"] = qkv[:, H_kv:2 * H_kv], qkv[:, 2 * H_kv:]
        s["slots"] = torch.randperm(blocks * bs, generator=g, device="cuda")[:T].clone()
        s["slots"][7::29] = -1  # padded tokens
        for x in ("k", "v"):
            s[x] = torch.zeros((blocks, bs, H_kv, D), dtype=TYPES[case["cache"]], device="cuda")
            s[x + "_scale"] = torch.zeros((blocks, H_kv, bs), dtype=torch.float32, device="cuda")
        return s
    ctx, n, rng = _lengths(case)
    need = [-(-c // bs) for c in ctx]
    pool = sum(need) + 3
    order = torch.randperm(pool, generator=g, device="cuda").int()
    table = torch.zeros((len(ctx), max(need + [1])), dtype=torch.int32, device="cuda")
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += k
    s["k"], s["k_scale"], s["v"], s["v_scale"] = _cache_of(g, case, pool)
    s["table"] = table
    s["ctx"] = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    if case["op"] == "load":
        rows = [0]
        for k in need:
            rows.append(rows[-1] + k * bs)
        s["cu_rows"], s["rows"] = torch.tensor(rows, dtype=torch.int32, device="cuda"), rows[-1]
        return s
    s["query"] = _randn(g, sum(n), case["H"], D, dtype=TYPES[case["dtype"]])
    s["scale"] = 1.0 / math.sqrt(D)
    if case["op"] == "tree":
        cu = [0]
        for k in n:
            cu.append(cu[-1] + k)
        s["cu"], s["most"] = torch.tensor(cu, dtype=torch.int32, device="cuda"), max(n)
        s["mask"] = _tree_masks(n, rng)
    return s


def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state, op)
    return {"store": _store, "load": _load, "decode": _decode, "tree": _tree, "logits": _logits}[op](state)


def _own(s, op):
    from litevllm_b200 import ops

    if op == "logits":
        return ops.process_logits(
            s["logits"], prompt_ids=s["prompt_ids"], prompt_lens=s["prompt_lens"], output_ids=s["output_ids"],
            output_lens=s["output_lens"], repetition=s["repetition"], presence=s["presence"], frequency=s["frequency"],
            bias_ids=s["bias_ids"], bias=s["bias"], allowed=s["allowed"])
    k, v = s["k"], s["v"]
    if s["k_scale"] is not None:
        k, v = ops.QuantizedCache(k, s["k_scale"]), ops.QuantizedCache(v, s["v_scale"])
    if op == "store":
        ops.store_kvcache_q8(s["key"], s["value"], k, v, s["slots"])
        return {x: s[x] for x in ("k", "k_scale", "v", "v_scale")}
    if op == "load":
        return ops.load_kvcache_q8(k, v, s["table"], s["ctx"], s["cu_rows"], s["rows"], dtype=TYPES[s["case"]["dtype"]])
    if op == "decode":
        return ops.paged_decode_q8(s["query"], k, v, s["table"], s["ctx"], s["scale"])
    return ops.paged_tree_attention(s["query"], k, v, s["table"], s["ctx"], s["cu"], s["most"], s["scale"], tree_mask=s["mask"])


# ------------------------------------------------------------ plain forms ---
def _store(s):
    at = s["slots"] >= 0
    slots = s["slots"][at]
    bs = s["k"].shape[1]
    for x, rows in (("k", s["key"]), ("v", s["value"])):
        data, scale = _quantise(rows[at], s["case"]["cache"])
        s[x].view(torch.uint8)[slots // bs, slots % bs] = data.view(torch.uint8)
        s[x + "_scale"][slots // bs, :, slots % bs] = scale
    return {x: s[x] for x in ("k", "k_scale", "v", "v_scale")}


def _gathered(s, x, n):
    """Positions 0..n-1 of every sequence's keys or values, [B, n, H_kv, D] in 32 bits."""
    pos = torch.arange(n, device="cuda")
    bs = s[x].shape[1]
    blocks = s["table"].long()[:, pos // bs]
    rows = s[x][blocks, pos % bs].float()
    if s[x + "_scale"] is not None:
        rows *= s[x + "_scale"][blocks, :, pos % bs].unsqueeze(-1)
    return rows


def _load(s):
    n = s["table"].shape[1] * s["k"].shape[1]
    pos = torch.arange(n, device="cuda")
    kept = pos < (s["cu_rows"][1:] - s["cu_rows"][:-1])[:, None]
    inside = (pos < s["ctx"][:, None])[kept]
    dtype = TYPES[s["case"]["dtype"]]
    return [torch.where(inside[:, None, None], _gathered(s, x, n)[kept], 0.0).to(dtype) for x in ("k", "v")]


def _attend(q, k, v, seen, scale):
    """q [B, n, H, D], k and v [B, S, H_kv, D], seen [B, n, S] -> [B, n, H, D] in 32 bits."""
    B, n, H, D = q.shape
    H_kv = k.shape[2]
    q = q.float().view(B, n, H_kv, H // H_kv, D).permute(0, 2, 3, 1, 4).reshape(B, H_kv, -1, D)
    x = torch.matmul(q, k.permute(0, 2, 3, 1)).view(B, H_kv, H // H_kv, n, -1) * scale
    x = x.masked_fill_(~seen[:, None, None], float("-inf"))
    x -= x.amax(-1, keepdim=True)
    x = x.exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(B, H_kv, -1, x.shape[-1]), v.permute(0, 2, 1, 3)).view(B, H_kv, H // H_kv, n, D) / total
    return o.permute(0, 3, 1, 2, 4).reshape(B, n, H, D)


def _decode(s):
    n = s["table"].shape[1] * s["k"].shape[1]
    seen = (torch.arange(n, device="cuda") < s["ctx"][:, None])[:, None]
    o = _attend(s["query"][:, None], _gathered(s, "k", n), _gathered(s, "v", n), seen, s["scale"])
    return o[:, 0].to(s["query"].dtype)


def _tree(s):
    n = s["table"].shape[1] * s["k"].shape[1]
    count = (s["cu"][1:] - s["cu"][:-1])[:, None]
    i = torch.arange(s["most"], device="cuda")
    kept = i < count
    row = torch.where(kept, s["cu"][:-1, None] + i, 0).long()
    prior = s["ctx"][:, None] - count
    j = torch.arange(n, device="cuda") - prior
    bit = (s["mask"][row, 0].unsqueeze(-1) >> j.clamp(0, 63)[:, None]) & 1
    seen = (j < 0)[:, None] | ((j < count)[:, None] & (bit == 1))
    o = _attend(s["query"][row], _gathered(s, "k", n), _gathered(s, "v", n), seen, s["scale"])
    return o[kept].to(s["query"].dtype)


def _logits(s):
    x = s["logits"].float()
    B, V = x.shape
    counts = []
    for ids, lens in ((s["prompt_ids"], s["prompt_lens"]), (s["output_ids"], s["output_lens"])):
        there = torch.arange(ids.shape[1], device="cuda") < lens[:, None]
        counts.append(torch.zeros((B, V), device="cuda").scatter_add_(1, ids, there.float()))
    seen = (counts[0] + counts[1]) > 0
    rep = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - (s["frequency"][:, None] * counts[1] + s["presence"][:, None] * (counts[1] > 0))
    if s["bias_ids"] is not None:
        x = x + torch.zeros_like(x).scatter_add_(1, s["bias_ids"], s["bias"])
    if s["allowed"] is not None:
        v = torch.arange(V, device="cuda")
        x = x.masked_fill((s["allowed"][:, v // 32] >> (v % 32)) & 1 == 0, float("-inf"))
    return x.to(s["logits"].dtype)


# ------------------------------------------------------------- in 64 bits ---
def _near_e4m3(y):
    """The e4m3 value nearest to y (ties to even), in 64 bits."""
    e = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -20))).clamp_min(-6.0)
    step = torch.exp2(e - 3.0)
    return ((y / step).round() * step).clamp(-448.0, 448.0)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "logits":
        x = s["logits"].double()
        for b in range(case["B"]):
            out = s["output_ids"][b, : s["output_lens"][b]]
            past = torch.cat([s["prompt_ids"][b, : s["prompt_lens"][b]], out]).unique()
            rep = s["repetition"][b].double()
            x[b, past] = torch.where(x[b, past] > 0, x[b, past] / rep, x[b, past] * rep)
            ids, times = out.unique(return_counts=True)
            x[b, ids] -= s["frequency"][b].double() * times + s["presence"][b].double()
            if case["bias"]:
                x[b].index_add_(0, s["bias_ids"][b], s["bias"][b].double())
            if case["grammar"]:
                bits = (s["allowed"][b][:, None] >> torch.arange(32, device="cuda")) & 1
                x[b, bits.reshape(-1)[: case["V"]] == 0] = -math.inf
        return x
    if op == "store":
        got, m = {}, M_OF[case["cache"]]
        bs = case["bs"]
        for name, rows in (("k", s["key"]), ("v", s["value"])):
            values = torch.zeros_like(s[name], dtype=torch.float64)
            scales = torch.zeros_like(s[name + "_scale"], dtype=torch.float64)
            x = rows.double()
            a = x.abs().amax(-1).clamp_min(FLOOR)
            # r and x r are 32-bit numbers by definition
            near = _near_e4m3((x * torch.div(torch.full_like(a, m), a).float().double()[..., None]).float().double())
            there = (s["slots"] >= 0).nonzero()[:, 0]
            at = s["slots"][there]
            values[at // bs, at % bs], scales[at // bs, :, at % bs] = near[there], a[there] / m
            got[name] = values if case["cache"] == "e4m3" else None  # int8 data are whole numbers
            got[name + "_scale"] = scales
        return got

    def rows_of(x, b, n):
        blocks = s["table"][b, : -(-n // case["bs"])].long()
        data = s[x][blocks].double()
        if s[x + "_scale"] is not None:
            data = data * s[x + "_scale"][blocks].double().transpose(1, 2).unsqueeze(-1)
        return data.reshape(-1, case["H_kv"], case["D"])[:n]

    ctx, n, _ = _lengths(case)
    if op == "load":
        got = []
        for x in ("k", "v"):
            whole = torch.zeros((s["rows"], case["H_kv"], case["D"]), dtype=torch.float64, device="cuda")
            for b, c in enumerate(ctx):
                at = int(s["cu_rows"][b])
                whole[at:at + c] = rows_of(x, b, c)
            got.append(whole)
        return got
    parts, at = [], 0
    for b, c in enumerate(ctx):
        q = s["query"][at:at + n[b]].double().view(n[b], case["H_kv"], -1, case["D"])
        x = torch.einsum("nhgd,shd->hgns", q, rows_of("k", b, c)) * s["scale"]
        if op == "tree":
            for i in range(n[b]):
                word = int(s["mask"][at + i, 0])
                hidden = [c - n[b] + j for j in range(n[b]) if not word >> j & 1]
                x[:, :, i, hidden] = -math.inf
        o = torch.einsum("hgns,shd->nhgd", torch.softmax(x, -1), rows_of("v", b, c))
        parts.append(o.reshape(n[b], case["H"], case["D"]))
        at += n[b]
    return torch.cat(parts)


# ------------------------------------------------------------------- work ---
def work(case):
    op = case["op"]
    size = {"bf16": 2, "f16": 2, "f32": 4, "int8": 1, "e4m3": 1}
    if op == "logits":
        B, V = case["B"], case["V"]
        mask = B * -(-V // 32) * 4 if case["grammar"] else 0
        past = B * (case["prompt"] + case["output"]) // 2 * 8 + B * case["bias"] * 12
        return {"bytes": 2 * B * V * size[case["dtype"]] + mask + past + 20 * B, "flops": 2 * B * V}
    row = case["H_kv"] * case["D"]
    if op == "store":
        T = case["T"]
        return {"bytes": 2 * T * (row * (size[case["dtype"]] + 1) + 4 * case["H_kv"]) + 8 * T, "flops": 4 * T * row}
    ctx, n, _ = _lengths(case)
    held = size[case["cache"]] * row + (4 * case["H_kv"] if case["cache"] in M_OF else 0)
    tables = sum(4 * -(-c // case["bs"]) + 4 for c in ctx)
    if op == "load":
        rows = sum(-(-c // case["bs"]) * case["bs"] for c in ctx)
        return {"bytes": 2 * sum(ctx) * held + 2 * rows * row * size[case["dtype"]] + tables, "flops": 2 * sum(ctx) * row}
    T = sum(n)
    return {"bytes": 2 * sum(ctx) * held + 2 * T * case["H"] * case["D"] * size[case["dtype"]] + tables + 8 * T,
            "flops": 4 * case["H"] * case["D"] * sum(a * b for a, b in zip(ctx, n))}
