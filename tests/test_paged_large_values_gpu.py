"""Paged attention over values near the end of bf16's range."""
import pytest
import torch

from distributed_pytorch_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("rows", [1, 130])
@pytest.mark.parametrize("bits", [10, 27, 60])
@pytest.mark.parametrize("width", [64, 128])
def test_large_values_under_rising_scores(rows, bits, width):
    """Scores that rise by ``bits`` powers of two over 640 keys whose values are about 1e33: every result is finite, and
    sums of probabilities times values stay so too while a probability is at most 2^8 (1e33 * 640 * 2^8 = 1.6e38)."""
    n, page = 640, 16
    g = torch.Generator(device=DEV).manual_seed(bits)
    ramp = torch.arange(n, device=DEV) * (bits / n) * 0.6931472
    k = (ramp[:, None] / width).expand(n, width).reshape(n // page, page, 1, width).to(torch.bfloat16)
    v = (torch.rand(n // page, page, 1, width, device=DEV, generator=g) * 1e33).to(torch.bfloat16)
    q = torch.ones(rows, 2, width, dtype=torch.bfloat16, device=DEV)
    table = torch.arange(n // page, dtype=torch.int32, device=DEV)[None]
    cu, kv = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, rows], [n]))
    o = ops.paged_attention(q, k.contiguous(), v, table, cu, kv, scale=1.0)
    want = ops.paged_attention_eager(q.double(), k.double(), v.double(), table, cu, kv, 1.0)
    assert torch.isfinite(o).all()
    # all values positive: the result bounds the sum of its terms. Roundings: the probability and the result to bf16 (2^-8
    # each), scores below 60 in fp32 (width + 4 roundings of their size, in numerator and denominator), fp32 sums of n.
    score = (width + 4) * 2.0 ** -24 * (bits * 0.7 + 1)
    tol = want * (2 * 2.0 ** -8 + 2 * score + (n + 4) * 2.0 ** -24) * 1.01
    assert ((o.double() - want).abs() <= tol).all()
