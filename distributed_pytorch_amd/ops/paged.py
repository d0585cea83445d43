"""A paged key / value cache for batches of requests of different lengths: page planning, append and attention.

A pool of pages ``[P, page, nkv, width]`` holds the rows of all requests; row ``j`` of request ``r`` lives in page
``block_table[r, j // page]`` at row ``j % page``. The batch of a step is ragged: the new tokens of all requests lie
one after another (``cu_q[r] .. cu_q[r + 1]``), one token of a decoding request next to a chunk of another's prompt.
A step is

    plan = paged_plan(q_lens, ctx_lens, block_table, free_pages, free_count, page, num_tokens)   # once per step
    paged_append(k_pages, v_pages, k, v, plan.slots)                                             # per layer
    o = paged_attention(q, k_pages, v_pages, block_table, plan.cu_q, plan.kv_lens)               # per layer

Lengths, tables and slots are int32 in device memory and never read by the host, so a step can be captured in a
hipGraph whose replays see growing requests. No gradients: on the GPU, tensors that require them are refused outside
``torch.no_grad()``.

GPU: ``csrc/paged_plan.hip``, ``paged_append.hip``, ``paged_attn.hip`` (bf16, fp16, fp32). CPU: stock ops.
Replaces, for ragged batches, the per-batch cache the reference grows by concatenation and its attention over it
(reference: single-gpu/model.py:136-149, 699-747).
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch

from .._ext import ops, refuse_grad, use_hip

_MAX_WIDTH = 256


class PagedPlan(NamedTuple):
    """All int32 on the device: ``cu_q [R + 1]`` first batch row of every request, ``kv_lens [R]`` rows in the cache after
    the step, ``positions [num_tokens]`` and ``slots [num_tokens]`` of the batch rows (0 and -1 behind the last request),
    ``free_left [2]`` = pages left on the free list, and pages that it could not give."""
    cu_q: torch.Tensor
    kv_lens: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor
    free_left: torch.Tensor


def _check(ok: bool, message: str) -> None:
    if not ok:
        raise RuntimeError(message)


def _int_vec(t: torch.Tensor, n: int | None = None) -> bool:
    return t.dtype == torch.int32 and t.dim() == 1 and t.is_contiguous() and (n is None or t.numel() == n)


# ---- planning -------------------------------------------------------------------------------
def paged_plan(q_lens: torch.Tensor, ctx_lens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
               free_count: torch.Tensor, page_size: int, num_tokens: int) -> PagedPlan:
    """Pages for the new tokens of every request, and where their rows go; all in one launch.

    ``q_lens, ctx_lens [R]``: new tokens and tokens already in the cache. ``block_table [R, M]``: its columns below
    ``ceil(ctx / page)`` are read, those of the new pages are written, in place. ``free_pages``: the free list, of
    which the first ``free_count[0]`` entries are free; pages are taken off its end, in the order of requests and
    positions. Neither it nor ``free_count`` is changed: the next step's ``free_count`` is ``free_left`` (or a copy).
    ``num_tokens``: rows of the batch, at least ``q_lens.sum()``; rows behind the last request are padding, requests
    that reach past it are cut off there. Tokens for which there is no page (free list empty, table full) get slot
    -1, their table entry is -1 and ``free_left[1]`` counts the missing pages. Lengths below 2^30."""
    if use_hip(q_lens):
        return PagedPlan(*ops().paged_plan(q_lens, ctx_lens, block_table, free_pages, free_count, page_size, num_tokens))
    R = q_lens.numel()
    _check(_int_vec(q_lens) and _int_vec(ctx_lens, R) and _int_vec(free_pages) and _int_vec(free_count)
           and free_count.numel() >= 1, "paged_plan: lengths and free list must be contiguous int32 vectors")
    _check(block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] == R,
           "paged_plan: block_table must be int32 [requests, columns]")
    _check(1 <= page_size <= 1 << 20, "paged_plan: page size must be in [1, 2^20]")
    _check(0 <= num_tokens <= 1 << 29, "paged_plan: num_tokens must be in [0, 2^29]")
    M = block_table.shape[1]
    count = min(max(int(free_count[0]), 0), free_pages.numel())
    cu, kv, positions, slots, taken, wanted = [0], [], [], [], 0, 0
    for r in range(R):
        n = min(max(int(q_lens[r]), 0), num_tokens - cu[-1])
        c = min(max(int(ctx_lens[r]), 0), 1 << 30)
        have, want = -(-c // page_size), -(-(c + n) // page_size)
        wanted += want - have
        for col in range(have, min(want, M)):
            block_table[r, col] = free_pages[count - 1 - taken] if taken < count else -1
            taken += 1
        for pos in range(c, c + n):
            held = int(block_table[r, pos // page_size]) if pos // page_size < M else -1
            positions.append(pos)
            slot = held * page_size + pos % page_size
            slots.append(slot if held >= 0 and slot < 2 ** 31 - 1 else -1)
        cu.append(cu[-1] + n)
        kv.append(c + n)
    rest = num_tokens - cu[-1]
    had = min(taken, count)
    return PagedPlan(*(torch.tensor(x, dtype=torch.int32, device=q_lens.device) for x in
                       (cu, kv, positions + [0] * rest, slots + [-1] * rest, [count - had, wanted - had])))


# ---- append -----------------------------------------------------------------------------------
def paged_append(k_pages: torch.Tensor, v_pages: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Rows ``k, v [N, nkv, width]`` (any strides with unit inner stride, e.g. the columns of a fused projection) into
    rows ``slots [N]`` of the pools ``[P, page, nkv, width]`` (any page, row and head strides). Slots outside
    ``[0, P * page)`` are skipped; the others must be distinct. Key and value widths may differ; the new rows lie outside
    the pools."""
    if use_hip(k_pages, k):
        refuse_grad("paged_append", k_pages, v_pages, k, v)
        ops().paged_append(k_pages, v_pages, k, v, slots)
        return
    _check(k_pages.dim() == 4 and v_pages.dim() == 4 and k_pages.shape[:3] == v_pages.shape[:3],
           "paged_append: pools must be [pages, page, kv heads, width] and agree in all but their width")
    _check(k.dim() == 3 and v.dim() == 3 and k.shape[0] == v.shape[0] and k.shape[1:] == k_pages.shape[2:]
           and v.shape[1:] == v_pages.shape[2:], "paged_append: the new rows must be [tokens, kv heads, width] of the pages")
    _check(k.dtype == v.dtype == k_pages.dtype == v_pages.dtype, "paged_append: all tensors share a type")
    _check(_int_vec(slots, k.shape[0]), "paged_append: slots must be a contiguous int32 vector of the right length")
    page = k_pages.shape[1]
    keep = (slots >= 0) & (slots < k_pages.shape[0] * page)
    at = slots[keep].long()
    k_pages[at // page, at % page] = k[keep]
    v_pages[at // page, at % page] = v[keep]


# ---- attention ----------------------------------------------------------------------------------
def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                    cu_q: torch.Tensor, kv_lens: torch.Tensor, scale: float | None = None, window: int | None = None,
                    max_q: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``q [N, nh, width]``, the newest tokens of every request (rows ``cu_q[r] .. cu_q[r + 1]``), over the request's
    ``kv_lens[r]`` cached rows, their own among them: the request's last row sees all of them, each row before it one
    less, and with ``window`` only the newest ``window`` of those. Grouped-query heads as in ``causal_attention``. A row
    without any key gives zeros; keys whose table entry names no page of the pool are left out. ``cu_q`` must not decrease:
    what the rows then hold is unspecified (nothing outside the buffers is touched).

    ``max_q``: an upper bound of the new tokens of a request, if the host knows one (a decode step: 1); it selects
    kernels, not results. ``out``: the result's buffer, apart from the inputs; rows outside every request keep what it holds (without
    ``out`` they are zero)."""
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    _check(window is None or window >= 1, "paged_attention: window must be positive or None")
    if use_hip(q, k_pages):
        refuse_grad("paged_attention", q, k_pages, v_pages, out)
        o = ops().paged_attention(q, k_pages, v_pages, block_table, cu_q, kv_lens, scale, window or 0, max_q or 0, out)
        return o if out is None else out
    return paged_attention_eager(q, k_pages, v_pages, block_table, cu_q, kv_lens, scale, window, out)


def paged_attention_eager(q, k_pages, v_pages, block_table, cu_q, kv_lens, scale: float, window: int | None = None,
                          out=None) -> torch.Tensor:
    """The same computation with stock ops, one request at a time (CPU, fp32 or fp64 checks); reads the lengths back."""
    R, page, nkv = cu_q.numel() - 1, k_pages.shape[1], k_pages.shape[2]
    _check(q.dim() == 3 and k_pages.dim() == 4 and v_pages.shape == k_pages.shape and k_pages.shape[3] == q.shape[2]
           and 1 <= q.shape[2] <= _MAX_WIDTH, "paged_attention: keys and values must share the queries' width, at most 256")
    _check(q.shape[1] % nkv == 0, "paged_attention: heads must be a multiple of the kv heads")
    _check(q.dtype == k_pages.dtype == v_pages.dtype, "paged_attention: all tensors share a type")
    _check(R >= 0 and _int_vec(cu_q) and _int_vec(kv_lens, R), "paged_attention: cu_q and kv_lens must be int32 vectors")
    _check(block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] == R,
           "paged_attention: block_table must be int32 [requests, columns]")
    _check(out is None or (out.shape == q.shape and out.dtype == q.dtype), "paged_attention: out must look like q")
    o = torch.zeros_like(q) if out is None else out
    N, group = q.shape[0], q.shape[1] // nkv
    real = torch.float64 if q.dtype == torch.float64 else torch.float32
    cu, lens = cu_q.tolist(), kv_lens.tolist()
    for r in range(R):
        a, b = max(cu[r], 0), min(cu[r + 1], N)
        if a >= b:
            continue
        pos = torch.arange(a, b, device=q.device) + (lens[r] - cu[r + 1])
        n = min(max(lens[r], 0), block_table.shape[1] * page)
        key = torch.arange(n, device=q.device)
        held = block_table[r, key // page].long()
        ok = (held >= 0) & (held < k_pages.shape[0])
        at = torch.where(ok, held, torch.zeros_like(held))
        k = k_pages[at, key % page].to(real).repeat_interleave(group, 1)
        v = v_pages[at, key % page].to(real).repeat_interleave(group, 1)
        seen = (key[None, :] <= pos[:, None]) & ok[None, :]
        if window is not None:
            seen &= key[None, :] > pos[:, None] - window
        # what no row sees takes no part, whatever it holds; what some rows see is masked row by row
        score = torch.einsum("qhd,khd->hqk", q[a:b].to(real), k) * scale
        score = score.masked_fill(~seen, float("-inf"))
        top = score.amax(-1, keepdim=True) if n else score.new_zeros(*score.shape[:2], 1)
        top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
        p = torch.exp(score - top)
        total = p.sum(-1, keepdim=True)
        w = torch.where(total > 0, p / total, p)
        finite = torch.isfinite(v).all(-1).all(-1)
        y = torch.einsum("hqk,khd->qhd", w[..., finite], v[finite])
        for j in torch.nonzero(~finite).flatten().tolist():
            rows = seen[:, j]
            y[rows] += w[:, rows, j].t()[:, :, None] * v[j]
        o[a:b] = y.to(q.dtype)
    return o
