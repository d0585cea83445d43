"""Single tokens over pages: nothing but the result is rounded to the type."""
import math

import pytest
import torch

from distributed_pytorch_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype,parts", [(torch.bfloat16, 2.0 ** -16), (torch.float16, 2.0 ** -22)])
@pytest.mark.parametrize("nh,nkv,width", [(12, 12, 64), (32, 8, 128), (6, 2, 96)])
@pytest.mark.parametrize("mixed", [False, True])
def test_single_tokens_keep_their_probabilities(dtype, parts, nh, nkv, width, mixed):
    """A probability in two parts of the type is off by the square of a half step (2^-16, 2^-22) of itself, scores and sums
    by their fp32 roundings: all that relative to the sum of weighted |v|. The result's rounding, a half step, is relative
    to the result alone, which is far smaller than that sum. With a prompt in the batch another kernel does the work."""
    page, lens = 16, [1, 7, 300, 2500, 5000]
    g = torch.Generator(device=DEV).manual_seed(width)
    per = -(-max(lens) // page)
    k, v = (torch.randn(per * len(lens), page, nkv, width, device=DEV, generator=g).to(dtype) for _ in range(2))
    table = torch.randperm(per * len(lens), device=DEV, generator=g).int().view(len(lens), per)
    n = [1] * len(lens)
    if mixed:
        n[2] = 100
    cu = [0]
    for x in n:
        cu.append(cu[-1] + x)
    one = [cu[r] for r in range(len(lens)) if n[r] == 1]
    q = torch.randn(cu[-1], nh, width, device=DEV, generator=g).to(dtype)
    cu, kv = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (cu, lens))
    o = ops.paged_attention(q, k, v, table, cu, kv, max_q=max(n))[one].double()
    args = (table, cu, kv, 1 / math.sqrt(width))
    want = ops.paged_attention_eager(q.double(), k.double(), v.double(), *args)[one]
    size = ops.paged_attention_eager(q.double(), k.double(), v.double().abs(), *args)[one]
    f, u = 2.0 ** -24, torch.finfo(dtype).eps / 2
    top = q.float().norm(dim=-1).max().item() * k.float().norm(dim=-1).max().item() / math.sqrt(width)
    score = (width + 4) * f * top + 4 * f * (1 + top)
    tol = want.abs() * u + size * (parts + 2 * score + (max(lens) + 4) * f) * 1.01 + torch.finfo(dtype).tiny
    err = (o - want).abs()
    assert bool((err <= tol).all()), f"error up to {(err / tol).max().item():.2f} of the bound"
