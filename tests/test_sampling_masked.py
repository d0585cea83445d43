"""Sampling from logits that masks and biases have made infinite: what is forbidden is never drawn."""
import math

import pytest
import torch

from distributed_pytorch_amd import ops


def masked_row(V, share, seed, device, dtype):
    """One row of random logits of which about ``share`` are allowed (at least one), and the allowed set."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(V, generator=g) * 2
    ok = torch.rand(V, generator=g) < share
    ok[V // 3] = True
    return x.masked_fill(~ok, -math.inf).to(dtype).to(device), ok.to(device)


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
