"""Operands of the ragged-batch operators that share memory without being dense."""
import pytest
import torch

from distributed_pytorch_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def test_strided_operands_that_overlap_are_refused():
    logits = torch.randn(4, 1000, device=DEV)
    fused = torch.randn(6, 32 * 64, device=DEV).to(BF)
    q, late = fused[:, : 8 * 64].view(6, 8, 64), fused[:, 4 * 64: 12 * 64].view(6, 8, 64)
    both = torch.randn(3, 16, 2, 2, 64, device=DEV).to(BF)            # keys and values of a row next to each other
    k, v = both[:, :, 0], both[:, :, 1]
    table, cu, kv = torch.zeros(1, 1, dtype=torch.int32, device=DEV), i32(0, 6), i32(6)
    rows = torch.randn(6, 2, 64, device=DEV).to(BF)
    slots = i32(*range(6))
    bad = [
        lambda: ops.penalize_logits(logits[:, :992], out=logits[:, 8:]),
        lambda: ops.penalize_logits(logits[:2, :992], out=logits[1:3, 8:]),
        lambda: ops.penalize_logits(logits[:, :500], bias=logits[:, 400:900], out=logits[:, 500:]),
        lambda: ops.paged_attention(q, k, v, table, cu, kv, out=late),
        lambda: ops.paged_attention(rows[:, :, :].repeat(1, 1, 1), k, v, table, cu, kv, out=k[0, 4:10]),
        lambda: ops.paged_append(k, k[:, :, :], rows, rows, slots),
        lambda: ops.paged_append(k, v, k[0, :6], rows, slots),
        lambda: ops.paged_append(k, v, rows, both[1, 2:8, 1], slots),
    ]
    for i, call in enumerate(bad):
        before = [t.clone() for t in (logits, fused, both)]
        with pytest.raises(RuntimeError, match="share memory"):
            call()
            print("not refused:", i)
        assert all(torch.equal(a, b) for a, b in zip(before, (logits, fused, both)))


def test_strided_operands_side_by_side_are_not():
    logits = torch.randn(4, 1000, device=DEV)
    want = ops.penalize_logits(logits[:, :496].contiguous(), bias=torch.ones(496, device=DEV))
    ops.penalize_logits(logits[:, :496], bias=torch.ones(496, device=DEV), out=logits[:, 496:992])
    assert torch.equal(logits[:, 496:992], want)
    ops.penalize_logits(logits[:, :496], bias=torch.ones(496, device=DEV), out=logits[:, :496])
    assert torch.equal(logits[:, :496], want)
    fused = torch.randn(6, 20 * 64, device=DEV).to(BF)
    q, k_new, v_new, out = (fused[:, a * 64: b * 64].view(6, b - a, 64) for a, b in ((0, 8), (8, 10), (10, 12), (12, 20)))
    table, cu, kv, slots = torch.zeros(1, 1, dtype=torch.int32, device=DEV), i32(0, 6), i32(6), i32(*range(6))
    got = []
    for both in (torch.zeros(3, 16, 2, 2, 64, device=DEV, dtype=BF), torch.zeros(3, 2, 16, 2, 64, device=DEV, dtype=BF).transpose(1, 2),
                 torch.zeros(3, 16, 2, 128, device=DEV, dtype=BF).view(3, 16, 2, 2, 64).transpose(2, 3)):
        k, v = both[:, :, 0], both[:, :, 1]
        ops.paged_append(k, v, k_new, v_new, slots)
        assert torch.equal(k[0, :6], k_new) and torch.equal(v[0, :6], v_new) and (both[1:] == 0).all() and (both[0, 6:] == 0).all()
        ops.paged_attention(q, k, v, table, cu, kv, out=out)
        got.append(out.clone())
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2]) and got[0].abs().max().item() > 0
