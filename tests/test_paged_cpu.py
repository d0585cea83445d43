"""Paged cache operators and logit penalties on the CPU: meaning, edges and refusals."""
import math

import pytest
import torch

from distributed_pytorch_amd import ops


def i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def test_plan_hands_out_pages_and_slots():
    table = torch.full((3, 4), -1, dtype=torch.int32)
    table[0, :2] = i32(7, 2)                     # 5 rows in two pages of 4
    table[2, 0] = 9                              # 4 rows: the page is full
    free = i32(10, 11, 12, 13, 99, 98)           # four are free, taken from the end of those
    p = ops.paged_plan(i32(1, 9, 1), i32(5, 0, 4), table, free, i32(4), 4, 13)
    assert p.cu_q.tolist() == [0, 1, 10, 11] and p.kv_lens.tolist() == [6, 9, 5]
    assert table.tolist() == [[7, 2, -1, -1], [13, 12, 11, -1], [9, 10, -1, -1]]
    assert p.positions.tolist() == [5, *range(9), 4, 0, 0]
    assert p.slots.tolist() == [9, 52, 53, 54, 55, 48, 49, 50, 51, 44, 40, -1, -1]
    assert p.free_left.tolist() == [0, 0]


def test_plan_counts_pages_it_could_not_give():
    table = torch.full((2, 2), -1, dtype=torch.int32)
    p = ops.paged_plan(i32(3, 9), i32(0, 0), table, i32(5, 6), i32(2, 0), 4, 12)
    assert table.tolist() == [[6, -1], [5, -1]]              # the third page is missing, the fourth column does not exist
    assert p.slots.tolist() == [24, 25, 26, 20, 21, 22, 23, -1, -1, -1, -1, -1]
    assert p.free_left.tolist() == [0, 2]


def test_plan_edges():
    none = torch.zeros(0, dtype=torch.int32)
    p = ops.paged_plan(none, none, torch.zeros(0, 3, dtype=torch.int32), none, i32(0), 16, 2)
    assert p.cu_q.tolist() == [0] and p.slots.tolist() == [-1, -1] and p.free_left.tolist() == [0, 0]
    table = torch.full((3, 2), -1, dtype=torch.int32)
    p = ops.paged_plan(i32(0, 5, 4), i32(0, 0, 0), table, i32(1, 2, 3), i32(3), 16, 6)    # cut at six rows
    assert p.cu_q.tolist() == [0, 0, 5, 6] and p.kv_lens.tolist() == [0, 5, 1]


def test_append_skips_slots_outside_and_takes_strided_rows():
    k_pages, v_pages = torch.zeros(3, 4, 2, 8), torch.zeros(3, 4, 2, 6)
    qkv = torch.randn(5, 40)
    k, v = qkv[:, 4:20].view(5, 2, 8), qkv[:, 20:32].view(5, 2, 6)
    ops.paged_append(k_pages, v_pages, k, v, i32(11, -1, 0, 12, 5))
    want_k, want_v = torch.zeros(12, 2, 8), torch.zeros(12, 2, 6)
    for i, s in ((0, 11), (2, 0), (4, 5)):
        want_k[s], want_v[s] = k[i], v[i]
    assert torch.equal(k_pages.view(12, 2, 8), want_k) and torch.equal(v_pages.view(12, 2, 6), want_v)


@pytest.mark.parametrize("window", [None, 1, 5])
def test_attention_matches_the_cached_form(window):
    torch.manual_seed(0)
    nh, nkv, d, page = 4, 2, 16, 3
    kv, q = [7, 1, 0, 12], [3, 1, 0, 12]
    table = torch.full((4, 4), -1, dtype=torch.int32)
    ids, at = torch.randperm(20, dtype=torch.int32), 0
    for r, n in enumerate(kv):
        c = -(-n // page)
        table[r, :c] = ids[at:at + c]
        at += c
    k_pages, v_pages = torch.randn(20, page, nkv, d), torch.randn(20, page, nkv, d)
    cu = [0, 3, 4, 4, 16]
    x = torch.randn(18, nh, d)
    out = torch.full_like(x, 7.0)
    assert ops.paged_attention(x, k_pages, v_pages, table, i32(*cu), i32(*kv), window=window, out=out) is out
    for r in range(4):
        if q[r] == 0:
            continue
        rows = torch.cat([torch.arange(page) + int(p) * page for p in table[r, : -(-kv[r] // page)]])[:kv[r]]
        k, v = k_pages.view(-1, nkv, d)[rows], v_pages.view(-1, nkv, d)[rows]
        for i in range(q[r]):
            pos = kv[r] - q[r] + i
            lo = 0 if window is None else max(0, pos - window + 1)
            want = ops.causal_attention_eager(x[None, cu[r] + i: cu[r] + i + 1], k[None, lo:pos + 1], v[None, lo:pos + 1],
                                              1 / math.sqrt(d))[0, 0]
            assert torch.allclose(out[cu[r] + i], want, atol=1e-5)
    assert (out[16:] == 7.0).all()
    assert (ops.paged_attention(x, k_pages, v_pages, table, i32(*cu), i32(*kv), window=window)[16:] == 0).all()


def test_attention_rows_without_keys_missing_pages_and_values_nobody_may_see():
    k_pages, v_pages = torch.randn(4, 2, 1, 8), torch.randn(4, 2, 1, 8)
    x = torch.randn(4, 2, 8)
    # four rows, two keys: rows 0 and 1 come before the first key
    o = ops.paged_attention(x, k_pages, v_pages, i32(3, 0).view(1, 2), i32(0, 4), i32(2))
    assert (o[:2] == 0).all() and torch.allclose(o[2], v_pages[3, 0].expand(2, 8))
    # the second page is missing: its keys are left out
    whole = ops.paged_attention(x[:1], k_pages, v_pages, i32(3, 1).view(1, 2), i32(0, 1), i32(2))
    for bad in (-1, 4, 2 ** 31 - 1):
        o = ops.paged_attention(x[:1], k_pages, v_pages, i32(3, bad).view(1, 2), i32(0, 1), i32(4))
        assert torch.equal(o, whole)
    # the later row's value is infinite: the earlier row does not see it
    v_pages[3, 1] = float("inf")
    k_pages[1] = float("nan")
    o = ops.paged_attention(x[:2], k_pages, v_pages, i32(3, 1).view(1, 2), i32(0, 2), i32(2))
    assert torch.isfinite(o[0]).all() and torch.isinf(o[1]).all()


def test_penalties_by_hand():
    x = torch.tensor([[2.0, -2.0, 1.0, 0.5, 3.0]])
    tokens = torch.tensor([[0, 1, 1, 2, 2, 9, -4, 4]])
    y = ops.penalize_logits(x, tokens, i32(2), i32(7), repetition=2.0, presence=0.5, frequency=0.25)
    # 0: prompt only; 1: prompt and once generated; 2: twice generated; 4: past the total
    assert torch.allclose(y, torch.tensor([[1.0, -4.75, -0.5, 0.5, 3.0]]))
    bias = torch.tensor([0.0, 0, 0, 1, float("nan")])
    y = ops.penalize_logits(x, bias=bias, allowed=i32(0b01011))
    assert y[0, :2].tolist() == [2.0, -2.0] and y[0, 2] == -math.inf and y[0, 3] == 1.5 and y[0, 4] == -math.inf
    assert (ops.penalize_logits(x, allowed=i32(0)) == -math.inf).all()
    z = x.clone()
    assert ops.penalize_logits(z, tokens, repetition=torch.tensor([2.0]), out=z) is z
    assert torch.allclose(z, torch.tensor([[1.0, -4.0, 0.5, 0.5, 1.5]]))


def test_refusals():
    t = torch.zeros(1, 2, dtype=torch.int32)
    one = i32(1)
    k = torch.zeros(2, 4, 1, 8)
    q = torch.zeros(1, 2, 8)
    cu = i32(0, 1)
    bad = [
        lambda: ops.paged_plan(one.long(), one, t, one, one, 4, 1),
        lambda: ops.paged_plan(one, i32(1, 2), t, one, one, 4, 1),
        lambda: ops.paged_plan(one, one, t, one, one, 0, 1),
        lambda: ops.paged_plan(one, one, t, one, one, 4, -1),
        lambda: ops.paged_plan(one, one, t.view(-1), one, one, 4, 1),
        lambda: ops.paged_plan(one, one, t, one, i32(), 4, 1),
        lambda: ops.paged_append(k, k.clone(), torch.zeros(1, 2, 8), torch.zeros(1, 1, 8), one),
        lambda: ops.paged_append(k, k.clone(), torch.zeros(1, 1, 8).half(), torch.zeros(1, 1, 8), one),
        lambda: ops.paged_append(k, k.clone(), torch.zeros(1, 1, 8), torch.zeros(1, 1, 8), i32(1, 2)),
        lambda: ops.paged_append(k[0], k[0], torch.zeros(1, 1, 8), torch.zeros(1, 1, 8), one),
        lambda: ops.paged_attention(q[..., :4], k, k, t, cu, one),
        lambda: ops.paged_attention(q, k, k, t, cu, i32(1, 1)),
        lambda: ops.paged_attention(q, k, k, t.long(), cu, one),
        lambda: ops.paged_attention(q, k, k, t, cu, one, window=0),
        lambda: ops.paged_attention(q, k.expand(2, 4, 3, 8), k.expand(2, 4, 3, 8), t, cu, one),
        lambda: ops.paged_attention(q, k, k, t, cu, one, out=q[:, :1]),
        lambda: ops.paged_attention(q.half(), k, k, t, cu, one),
        lambda: ops.penalize_logits(torch.zeros(4)),
        lambda: ops.penalize_logits(torch.zeros(2, 4), torch.zeros(1, 3, dtype=torch.int64)),
        lambda: ops.penalize_logits(torch.zeros(2, 4), torch.zeros(2, 3, dtype=torch.int64), total_lens=i32(1, 2, 3)),
        lambda: ops.penalize_logits(torch.zeros(2, 4), bias=torch.zeros(3)),
        lambda: ops.penalize_logits(torch.zeros(2, 40), allowed=i32(0)),
        lambda: ops.penalize_logits(torch.zeros(2, 4), out=torch.zeros(2, 5)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            print("not refused:", i)
