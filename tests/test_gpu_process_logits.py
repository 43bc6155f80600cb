"""Logits processing on the GPU against the 64-bit oracle."""

import random

import numpy as np
import pytest
import torch

from litevllm_b200 import _lib, ops
from litevllm_b200.sampler import Sampler
from oracle import logits as olog
from tests.spec_inputs import randn

pytestmark = pytest.mark.gpu

# half a step of the type, plus five fp32 roundings of the largest operand
STEP = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make(B, V, dtype, Lp, Lo, nb, grammar, seed):
    rng = random.Random(seed)
    ids = lambda n: [[min(V - 1, int(V * rng.random() ** 3)) for _ in range(n)] for _ in range(B)]  # noqa: E731
    c = dict(x=randn(seed, B, V, dtype=dtype, std=4.0), prompt=ids(Lp), output=ids(Lo))
    c["plen"] = [rng.randint(0, Lp) for _ in range(B)]
    c["olen"] = [rng.randint(0, Lo) for _ in range(B)]
    c["rep"] = [rng.choice([1.0, 1.3, 0.8]) for _ in range(B)]
    c["pres"] = [rng.choice([0.0, 0.7, -0.4]) for _ in range(B)]
    c["freq"] = [rng.choice([0.0, 0.3]) for _ in range(B)]
    c["bias"] = [[(rng.choice([0, V - 1, rng.randrange(V)]), rng.uniform(-5, 5)) for _ in range(nb)]
                 for _ in range(B)]
    c["allowed"] = torch.rand((B, V), generator=torch.Generator().manual_seed(seed)) < 0.5 if grammar else None
    return c


def words_of(allowed):
    B, V = allowed.shape
    pad = torch.zeros((B, -(-V // 32) * 32), dtype=torch.int64)
    pad[:, :V] = allowed
    w = (pad.view(B, -1, 32) << torch.arange(32)).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).int()


def args(c, dev):
    f = lambda v: torch.tensor(v, dtype=torch.float32, device=dev)  # noqa: E731
    i = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    B = c["x"].shape[0]
    l = lambda v: torch.tensor(v, dtype=torch.int64, device=dev).view(B, -1)  # noqa: E731,E741
    kw = dict(prompt_ids=l(c["prompt"]), prompt_lens=i(c["plen"]), output_ids=l(c["output"]),
              output_lens=i(c["olen"]), repetition=f(c["rep"]), presence=f(c["pres"]),
              frequency=f(c["freq"]))
    if c["bias"][0]:
        kw["bias_ids"] = l([[t for t, _ in r] for r in c["bias"]])
        kw["bias"] = f([[v for _, v in r] for r in c["bias"]])
    if c["allowed"] is not None:
        kw["allowed"] = words_of(c["allowed"]).to(dev)
    return kw


def expect(c):
    cut = lambda rows, n: [r[:k] for r, k in zip(rows, n)]  # noqa: E731
    f32 = lambda v: np.asarray(v, np.float32)  # noqa: E731
    bias = [[(t, float(np.float32(v))) for t, v in r] for r in c["bias"]]
    return olog.process(c["x"].double().numpy(), cut(c["prompt"], c["plen"]),
                        cut(c["output"], c["olen"]), f32(c["rep"]), f32(c["pres"]), f32(c["freq"]),
                        bias, None if c["allowed"] is None else c["allowed"].numpy())


def check(got, c):
    want = torch.from_numpy(expect(c))
    got = got.double().cpu()
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and (got[inf] < 0).all()
    # |x|, frequency * count, |presence| and the biases' sum bound every operand
    big = c["x"].double().abs() * 1.3 + 0.3 * len(c["output"][0]) + 1 + 5 * len(c["bias"][0])
    bound = STEP[c["x"].dtype] * want.abs() + 2.0 ** -24 * (5 + len(c["bias"][0])) * big
    assert ((got - want).abs() <= bound)[~inf].all()


CASES = [  # (B, V, prompt, output, biases, grammar)
    (1, 1, 1, 1, 0, False),
    (1, 7, 3, 2, 1, True),
    (3, 31, 5, 9, 2, True),
    (2, 32, 0, 4, 0, True),
    (5, 1003, 40, 17, 9, True),       # rows at odd addresses
    (3, 8192, 300, 100, 16, True),    # exactly one part of 16-bit logits
    (2, 8193, 10, 0, 3, False),
    (4, 20011, 1000, 700, 300, True),
    (130, 517, 6, 6, 1, True),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", CASES, ids=range(len(CASES)))
def test_matches_oracle(cuda, dtype, shape):
    B, V, Lp, Lo, nb, grammar = shape
    c = make(B, V, dtype, Lp, Lo, nb, grammar, seed=V)
    kw = args(c, cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    x = c["x"].cuda()
    got = ops.process_logits(x, status=status, **kw)
    check(got, c)
    assert torch.equal(x.cpu(), c["x"]) and status.item() == 0  # the input is left
    assert torch.equal(ops.process_logits(x, **kw), got)        # and a second call agrees
    # into a wider buffer, aligned differently from the input
    wide = torch.full((B, V + 5), 3.0, dtype=dtype, device=cuda)
    assert torch.equal(ops.process_logits(x, out=wide[:, 3:3 + V], **kw), got)
    assert (wide[:, :3] == 3).all() and (wide[:, 3 + V:] == 3).all()
    # in place, in rows of a wider buffer
    wide.fill_(3.0)
    wide[:, 1:1 + V] = x
    there = ops.process_logits(wide[:, 1:1 + V], out=wide[:, 1:1 + V], **kw)
    assert torch.equal(there, got) and (wide[:, :1] == 3).all() and (wide[:, 1 + V:] == 3).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_each_operand_alone(cuda, dtype):
    c = make(3, 2050, dtype, 50, 40, 5, True, seed=1)
    full = args(c, cuda)
    none = dict(plen=[0] * 3, olen=[0] * 3, rep=[1.0] * 3, pres=[0.0] * 3, freq=[0.0] * 3,
                bias=[[]] * 3, allowed=None)
    x = c["x"].cuda()
    assert torch.equal(ops.process_logits(x), x)
    one = lambda *names: {k: full[k] for k in names}  # noqa: E731
    hist = one("prompt_ids", "prompt_lens", "output_ids", "output_lens")
    for keys, kw in ((("plen", "olen", "rep"), dict(hist, **one("repetition"))),
                     (("olen", "pres"), dict(hist, **one("presence"))),
                     (("olen", "freq"), dict(one("output_ids", "output_lens", "frequency"))),
                     (("bias",), one("bias_ids", "bias")),
                     (("allowed",), one("allowed"))):
        d = dict(c, **none)
        d.update({k: c[k] for k in keys})
        check(ops.process_logits(x, **kw), d)
    # lengths left out: the whole rows count
    d = dict(c, **none)
    d.update(plen=[50] * 3, olen=[40] * 3, rep=c["rep"])
    check(ops.process_logits(x, **one("prompt_ids", "output_ids", "repetition")), d)


def test_repetition_agrees_with_the_existing_kernel(cuda):
    x = randn(1, 4, 5000, dtype=torch.bfloat16, std=3.0).cuda()
    past = torch.randint(0, 5000, (4, 200), device=cuda)
    pen = torch.tensor([1.0, 1.2, 0.7, 2.0], device=cuda)
    want = ops.repetition_penalty_(x.clone(), past, pen)
    assert torch.equal(ops.process_logits(x, prompt_ids=past, repetition=pen), want)


def test_special_logits_and_closed_rows(cuda):
    """Infinities and NaN under the mask vanish, elsewhere they pass through; a row
    that the mask closes altogether is all -inf and greedy sampling takes id 0."""
    x = torch.zeros((3, 100))
    x[0, :50:5] = float("nan")
    x[0, 1] = float("inf")
    x[1, :] = float("nan")
    x[2, 3], x[2, 4] = -float("inf"), float("inf")
    allowed = torch.ones((3, 100), dtype=torch.bool)
    allowed[0, ::5] = False
    allowed[0, 1] = False
    allowed[1] = False
    for dtype in (torch.float32, torch.bfloat16):
        got = ops.process_logits(
            x.to(dtype).cuda(), output_ids=torch.tensor([[7], [7], [4]], device=cuda),
            frequency=torch.ones(3, device=cuda), bias_ids=torch.tensor([[0, 1], [0, 1], [3, 4]], device=cuda),
            bias=torch.full((3, 2), 2.0, device=cuda), allowed=words_of(allowed).cuda()).float().cpu()
        assert not torch.isnan(got).any()
        assert torch.equal(got == -float("inf"), ~allowed | (x == -float("inf")))
        assert got[2, 4] == float("inf") and got[0, 7] == -1
    ids = Sampler.sample_batch(x.cuda()[1:2], processing=dict(allowed=words_of(allowed[1:2]).cuda()))
    assert ids.tolist() == [0]


def test_padding_and_foreign_ids(cuda):
    """Negative ids are padding; ids of V and above are skipped and flagged."""
    x = randn(3, 1, 40).cuda()
    f = lambda v: torch.tensor([v], device=cuda)  # noqa: E731
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    got = ops.process_logits(x, output_ids=torch.tensor([[-1, 5, -2 ** 40, 5]], device=cuda),
                             frequency=f(0.5), status=status)
    want = x.clone()
    want[0, 5] -= 1.0
    assert torch.equal(got, want) and status.item() == 0
    for kw in (dict(output_ids=torch.tensor([[40, 5, 5]], device=cuda), frequency=f(0.5)),
               dict(output_ids=torch.tensor([[5, 2 ** 40, 5]], device=cuda), frequency=f(0.5)),
               dict(output_ids=torch.tensor([[5, 5]], device=cuda), frequency=f(0.5),
                    bias_ids=torch.tensor([[40, -3]], device=cuda), bias=torch.ones((1, 2), device=cuda))):
        status.zero_()
        assert torch.equal(ops.process_logits(x, status=status, **kw), want)
        assert status.item() == _lib.LK_STATUS_TOKEN_OOB


def test_repeated_biases_add_in_list_order(cuda):
    ids = torch.tensor([[4, 9, 4, 4, 9]], device=cuda)
    val = torch.tensor([[1e8, 1.0, -1e8, 0.5, 2.0]], device=cuda)
    got = ops.process_logits(torch.zeros((1, 16), device=cuda), bias_ids=ids, bias=val).cpu()
    assert got[0, 4] == 0.5 and got[0, 9] == 3.0 and got.count_nonzero() == 2


def test_views_and_broadcast_operands(cuda):
    """Histories and masks shared by all rows (expanded), transposed logits."""
    x = randn(5, 300, 4, dtype=torch.bfloat16).cuda().t()
    hist = torch.tensor([[3, 3, 8]], device=cuda)
    words = words_of(torch.arange(300).remainder(3).ne(0)[None]).cuda()
    freq = torch.full((4,), 0.25, device=cuda)
    a = ops.process_logits(x, output_ids=hist.expand(4, 3), frequency=freq,
                           allowed=words.expand(4, words.shape[1]))
    b = ops.process_logits(x.contiguous(), output_ids=hist.repeat(4, 1), frequency=freq,
                           allowed=words.repeat(4, 1))
    assert torch.equal(a, b)
    assert torch.equal(ops.process_logits(x[1], out=None), x[1:2].contiguous())


def test_captured_graph_replays(cuda):
    c = make(4, 5000, torch.bfloat16, 60, 30, 4, True, seed=2)
    kw, x = args(c, cuda), c["x"].cuda()
    ops.process_logits(x, **kw)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.process_logits(x, **kw)
    x.copy_(randn(9, 4, 5000, dtype=torch.bfloat16).cuda())
    kw["output_lens"].fill_(30)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ops.process_logits(x, **kw))


def test_long_history(cuda):
    """More history than a CTA's threads, with counts in the thousands."""
    V = 9000
    ids = torch.randint(0, 3, (2, 70000), device=cuda)
    got = ops.process_logits(torch.zeros((2, V), device=cuda), output_ids=ids,
                             frequency=torch.full((2,), 0.5, device=cuda)).cpu()
    for b in range(2):
        assert torch.equal(got[b, :3], -0.5 * torch.bincount(ids[b].cpu(), minlength=3).float())
        assert got[b, 3:].count_nonzero() == 0
