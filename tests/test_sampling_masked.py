"""Sampling from logits that masks and biases have made infinite: what is forbidden is never drawn."""
import math

import pytest
import torch

from distributed_pytorch_amd import ops
from distributed_pytorch_amd.config import LLMconfig
from distributed_pytorch_amd.models.llm import LLM


def masked_row(V, share, seed, device, dtype):
    """One row of random logits of which about ``share`` are allowed (at least one), and the allowed set."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(V, generator=g) * 2
    ok = torch.rand(V, generator=g) < share
    ok[V // 3] = True
    return x.masked_fill(~ok, -math.inf).to(dtype).to(device), ok.to(device)


def infinite_rows(V):
    """Logits and the set that may be drawn: nothing allowed, one token, one and two forced by +inf, a plain row."""
    x = torch.randn(5, V, generator=torch.Generator().manual_seed(3))
    x[0] = -math.inf
    x[1, 1:] = -math.inf
    x[2, V - 1] = math.inf
    x[2, : V // 2] = -math.inf
    x[3, 5], x[3, V - 3] = math.inf, math.inf
    return x, [{0}, {0}, {V - 1}, {5, V - 3}, set(range(V))]


def check_infinite_rows(sample, V, device, dtype):
    x, sets = infinite_rows(V)
    x = x.to(dtype).to(device)
    for topk in (None, 1, 2, 7, V):
        seen = set()
        for _ in range(30):
            tok = sample(x, 0.7, topk)
            assert tok.shape == (5, 1) and tok.dtype == torch.int64
            for t, ok in zip(tok[:, 0].tolist(), sets):
                assert t in ok
            seen.add(int(tok[3]))
        if topk != 1:
            assert seen == sets[3]       # 30 draws of a fair coin: both, but for 2^-29


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_eager_sampler_on_rows_of_infinite_logits(dtype):
    torch.manual_seed(0)
    check_infinite_rows(ops.sample_eager, 64, "cpu", dtype)


def test_eager_sampler_draws_what_it_drew():
    """Finite logits: the same tokens as the plain chain from the same random numbers."""
    x = torch.randn(50, 97, generator=torch.Generator().manual_seed(1)) * 3
    for topk in (None, 1, 10, 200):
        torch.manual_seed(4)
        got = ops.sample_eager(x, 0.8, topk)
        y = x / 0.8
        if topk is not None:
            y = y.masked_fill(y < torch.topk(y, min(topk, 97)).values[:, -1:], -math.inf)
        torch.manual_seed(4)
        assert torch.equal(got, torch.multinomial(torch.softmax(y, -1), 1))


def test_generation_where_nothing_is_allowed():
    m = LLM(LLMconfig(vocab_size=97, block_size=48, n_embd=32, n_layer=1, n_head=4, up_dim=48, attn="mha", pos_emb="learn",
                      non_linearity="gelu").finalize()).eval()
    none = dict(allowed=torch.zeros(4, dtype=torch.int32))
    idx = torch.randint(1, 97, (2, 3))
    assert (m.generate(idx, 5, penalties=none)[:, 3:] == 0).all()
    assert all((o[3:] == 0).all() for o in m.generate_ragged(list(idx), 5, penalties=none))


# ---- GPU ---------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("topk", [None, 400, 2000])
def test_fused_sampler_never_draws_what_the_mask_forbids(dtype, topk):
    """The fp32 scan leaves a few of the 2^24 draws between two threads' intervals: they too land on an allowed token.
    Fewer tokens are allowed than ``topk``, so the filter removes none of them."""
    V, rows = 50304, 1 << 20
    for seed in range(4):
        x, ok = masked_row(V, 0.004, seed, "cuda", dtype)
        assert topk is None or int(ok.sum()) < topk
        for draw in range(4):
            tok = ops.sample_fused(x.expand(rows, V), 1.0, topk, torch.tensor([1000 * seed + draw], device="cuda"))
            assert bool(ok[tok[:, 0]].all()), (seed, draw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("topk", [None, 1, 3, 600, 3000])
def test_fused_sampler_on_masked_rows_follows_the_softmax(dtype, topk):
    """Frequencies over the allowed tokens, with more and with fewer of them than ``topk``."""
    V, rows = 4096, 1 << 16
    for share in (0.0, 0.001, 0.5):
        x, ok = masked_row(V, share, 7, "cuda", dtype)
        p = torch.softmax(x.double(), -1)
        if topk is not None:
            p = torch.where(x.double() >= torch.topk(x.double(), topk).values[-1], p, torch.zeros_like(p))
            p = p / p.sum()
        tok = ops.sample_fused(x.expand(rows, V), 1.0, topk, torch.tensor([5], device="cuda"))[:, 0]
        assert bool((p[tok] > 0).all())
        freq = torch.bincount(tok, minlength=V).double() / rows
        # Bernstein: a count X of n draws has P(|X - np| > t) <= 2 exp(-t^2 / (2 np(1 - p) + 2t / 3)), which is 2 exp(-L)
        # at t = L / 3 + sqrt(L^2 / 9 + 2 L np(1 - p)). L = 30: 2e-13 for each of the 4096 tokens, 1e-9 in all. (The normal
        # bound of five standard deviations does not hold here: many tokens expect less than one draw.)
        L, var = 30.0, rows * p * (1 - p)
        assert ((freq - p).abs() * rows <= L / 3 + (L * L / 9 + 2 * L * var).sqrt()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_samplers_on_rows_of_infinite_logits(dtype):
    torch.manual_seed(0)
    for V in (64, 8200):
        check_infinite_rows(ops.sample_fused, V, "cuda", dtype)
        check_infinite_rows(ops.sample_eager, V, "cuda", dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
def test_generation_under_a_mask_on_the_gpu(graph):
    """Dense and ragged generation, eager and captured: allowed tokens only, and token 0 where none is allowed."""
    torch.manual_seed(0)
    m = LLM(LLMconfig(vocab_size=512, block_size=256, n_embd=256, n_layer=2, n_head=4, up_dim=512, attn="mha", pos_emb="learn",
                      non_linearity="gelu").finalize()).cuda().to(torch.bfloat16).eval()
    idx = torch.randint(1, 512, (4, 9), device="cuda")
    some = torch.zeros(16, dtype=torch.int32, device="cuda")
    some[3], some[9] = 0b1010, 1
    for allowed, may in ((some, {97, 99, 288}), (torch.zeros_like(some), {0})):
        for topk in (None, 50):
            pen = dict(allowed=allowed)
            out = m.generate(idx, 40, topk=topk, hip_graph=graph, penalties=pen)
            assert m.last_decode_graphed == graph and set(out[:, 9:].unique().tolist()) <= may
            out = m.generate_ragged(list(idx), 40, topk=topk, hip_graph=graph, penalties=pen)
            assert m.last_decode_graphed == graph and set(torch.stack(out)[:, 9:].unique().tolist()) <= may


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1, 7, 97, 4099, 50257])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_fused_sampler_on_odd_vocabularies(V, dtype):
    """Rows that 16-byte loads cannot take: the largest logit at top-1, the top-k set, the whole row without a filter."""
    g = torch.Generator(device="cuda").manual_seed(V)
    x = (torch.randn(40, V, device="cuda", generator=g) * 2).to(dtype)
    tok = ops.sample_fused(x, 1.0, 1)
    assert tok.shape == (40, 1) and torch.equal(x.gather(1, tok)[:, 0], x.amax(-1))
    for k in (5, V):
        kth = torch.topk(x.float(), min(k, V)).values[:, -1:]
        for _ in range(20):
            tok = ops.sample_fused(x, 0.7, k)
            assert int(tok.max()) < V and (x.float().gather(1, tok) >= kth).all()
    wide = torch.full((40, V + 3), 99.0, device="cuda").to(dtype)      # rows off 16 bytes inside a larger buffer
    wide[:, 1:V + 1] = x
    assert torch.equal(x.gather(1, ops.sample_fused(wide[:, 1:V + 1], 1.0, 1))[:, 0], x.amax(-1))
    seed = torch.tensor([11], device="cuda")
    assert torch.equal(ops.sample_fused(x, 0.7, None, seed), ops.sample_fused(wide[:, 1:V + 1], 0.7, None, seed))


@pytest.mark.gpu
@pytest.mark.parametrize("V,graphed", [(509, True), (50257, True), (57350, False)])
def test_captured_generation_over_odd_vocabularies(V, graphed):
    """Sampling is part of a captured step only as the kernel: a larger vocabulary decodes eagerly, with the same tokens."""
    torch.manual_seed(0)
    m = LLM(LLMconfig(vocab_size=V, block_size=64, n_embd=128, n_layer=1, n_head=2, up_dim=128, attn="mha", pos_emb="learn",
                      non_linearity="gelu").finalize()).cuda().eval()    # fp32: bf16 logits tie, and ties are drawn
    idx = torch.randint(0, V, (3, 5), device="cuda")
    pen = dict(frequency=1e4)                      # no token twice: every step has to see the ones before it
    want = m.generate_ragged(list(idx), 30, topk=1, hip_graph=False, penalties=pen)
    got = m.generate_ragged(list(idx), 30, topk=1, penalties=pen)
    assert m.last_decode_graphed == graphed
    for a, b in zip(want, got):
        assert torch.equal(a, b) and len(set(a[5:].tolist())) == 30
    m.to(torch.bfloat16)                           # what the dense captured step takes
    out = m.generate(idx, 30, topk=1, penalties=pen)
    assert m.last_decode_graphed == graphed
    assert all(len(set(row[5:].tolist())) == 30 and int(row.max()) < V for row in out)
    free = m.generate_ragged(list(idx), 30, topk=20)
    assert all(int(o.max()) < V and int(o.min()) >= 0 for o in free)
