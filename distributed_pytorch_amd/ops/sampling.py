"""Next-token sampling: temperature, top-k filter, softmax and one multinomial draw.

GPU: one HIP kernel per call (``csrc/sample.hip``), seeded by one device integer drawn from torch's
generator of that device, so it is reproducible under ``manual_seed`` and can be captured in a hipGraph
(every replay draws a new seed). CPU / fallback: the reference's chain of stock ops
(reference: single-gpu/model.py:733-745)."""
from __future__ import annotations

import torch
import torch.nn.functional as F

from .._ext import ops, refuse_grad, use_hip


def sample_eager(logits: torch.Tensor, temperature: float = 1.0, topk: int | None = None) -> torch.Tensor:
    """``logits [B, V]`` -> token ids ``[B, 1]`` with stock ops (no host-built index tensors). Tokens of -inf are never
    drawn, those of +inf share the draw equally, and a row of nothing but -inf gives token 0."""
    logits = logits.float()
    if temperature > 0:
        logits = logits / temperature
    if topk is not None:
        v, _ = torch.topk(logits, min(topk, logits.size(-1)))
        logits = logits.masked_fill(logits < v[:, -1:], -float("inf"))
    # The softmax of infinite logits has no value: it gets the largest numbers instead, and what is -inf is taken out of its
    # result. The 1e-37 goes to token 0 and decides where nothing else is left. (No reduction over the row, here: over a
    # long one torch clears its semaphores with a memset, which a captured step must not hold.)
    most = torch.finfo(logits.dtype).max
    p = F.softmax(logits.clamp(-most, most), dim=-1).masked_fill(logits == -float("inf"), 0.0)
    p[:, :1] += 1e-37
    return torch.multinomial(p, num_samples=1)


_MAX_VOCAB = 57344      # of the kernel: a row stays in one workgroup's registers


def _fused_ok(logits: torch.Tensor) -> bool:
    V = logits.shape[-1]
    return (use_hip(logits) and logits.dim() == 2 and logits.dtype in (torch.bfloat16, torch.float32)
            and logits.stride(1) == 1 and V % 8 == 0 and 8 <= V <= _MAX_VOCAB
            and (logits.stride(0) * logits.element_size()) % 16 == 0 and logits.data_ptr() % 16 == 0)


def sample_captures(weight: torch.Tensor) -> bool:
    """Whether sampling from the logits of this head ``[V, C]`` may be part of a captured step: it is the kernel then. The
    stock chain holds reductions over whole rows, which clear their semaphores with a memset, and such nodes have given
    wrong results on replays."""
    return use_hip(weight) and weight.shape[0] <= _MAX_VOCAB


def sample_step_supported(logits: torch.Tensor) -> bool:
    return _fused_ok(logits) and hasattr(ops(), "sample_topk_step")


def sample_step(logits: torch.Tensor, temperature: float, topk: int | None, seed: torch.Tensor, tok: torch.Tensor,
                history: torch.Tensor, history_pos: torch.Tensor, pos: torch.Tensor, len_after: torch.Tensor,
                ticket: torch.Tensor) -> None:
    """Sampling and the bookkeeping of one captured decode step in one launch: the drawn tokens go to ``tok
    [B, 1]`` (the next step's input) and to ``history[:, history_pos]``; the device counters ``pos``,
    ``len_after`` and ``history_pos`` then advance by one. ``seed`` is fixed for the generation (the kernel
    mixes ``pos`` into the random stream), ``ticket`` a zeroed int32 ``[1]`` the kernel keeps at zero."""
    ops().sample_topk_step(logits, float(temperature), int(topk or 0), seed, tok, history, history_pos, pos, len_after,
                           ticket)


def sample_fused(logits: torch.Tensor, temperature: float = 1.0, topk: int | None = None,
                 seed: torch.Tensor | None = None) -> torch.Tensor:
    """Same distribution from one kernel launch, infinite logits included. ``seed``: int64 ``[1]`` on the device (default:
    drawn)."""
    if not _fused_ok(logits):
        if not (use_hip(logits) and logits.dim() == 2 and logits.is_floating_point() and 1 <= logits.shape[1] <= _MAX_VOCAB):
            return sample_eager(logits, temperature, topk)
        # rows that the kernel's 16-byte loads cannot take (a vocabulary that is no multiple of 8, odd strides): a copy,
        # filled up with logits of -inf, which are never drawn
        B, V = logits.shape
        dtype = torch.bfloat16 if logits.dtype == torch.bfloat16 else torch.float32
        rows = torch.full((B, (V + 7) // 8 * 8), -float("inf"), dtype=dtype, device=logits.device)
        rows[:, :V] = logits
        logits = rows
    if seed is None:
        seed = torch.randint(-(1 << 62), 1 << 62, (1,), dtype=torch.int64, device=logits.device)
    return ops().sample_topk(logits, float(temperature), int(topk or 0), seed)


def _row_value(x, logits: torch.Tensor):
    """(device vector or None, host value) of a penalty given as a number or an fp32 tensor (one value, or one per row)."""
    return (x, 0.0) if isinstance(x, torch.Tensor) else (None, float(x))


def penalize_logits(logits: torch.Tensor, tokens: torch.Tensor | None = None, prompt_lens: torch.Tensor | None = None,
                    total_lens: torch.Tensor | None = None, repetition=1.0, presence=0.0, frequency=0.0,
                    bias: torch.Tensor | None = None, allowed: torch.Tensor | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Logits ``[R, V]`` (bf16, fp16, fp32) with penalties for repeated tokens, biases and a grammar mask applied, for the
    sampler that follows. ``tokens [R, L]`` (int64 or int32) is the rows' history, of which the first ``total_lens``
    entries count (default: all) and the first ``prompt_lens`` are the prompt (default: none); ids outside the
    vocabulary are ignored. In fp32, rounded once:

    * ``repetition``: the logit of every token in the history is divided by it where positive, multiplied elsewhere;
    * ``presence`` and ``frequency``: a token generated n > 0 times loses ``presence + n * frequency``;
    * ``bias`` (fp32 ``[V]`` or ``[R, V]``) is added;
    * ``allowed`` (int32 ``[ceil(V / 32)]`` or one such row per row of logits): tokens whose bit ``v % 32`` of word ``v // 32``
      is clear become -inf, whatever their logit was. A row that allows nothing is -inf throughout, and the samplers
      give token 0 for it.

    The penalties are numbers or fp32 tensors with one value or one per row, lengths int32 tensors likewise; they are
    read by the kernel, so a captured step sees what a replay's buffers hold. ``out`` may be ``logits`` itself,
    but not overlap it otherwise. No
    gradients: on the GPU, tensors that require them are refused outside ``torch.no_grad()``."""
    if use_hip(logits):
        refuse_grad("penalize_logits", logits, repetition, presence, frequency, bias, out)
        rep, rep_v = _row_value(repetition, logits)
        pres, pres_v = _row_value(presence, logits)
        freq, freq_v = _row_value(frequency, logits)
        y = ops().penalize_logits(logits, tokens, prompt_lens, total_lens, rep, pres, freq, rep_v, pres_v, freq_v, bias, allowed,
                                  out)
        return y if out is None else out
    return penalize_logits_eager(logits, tokens, prompt_lens, total_lens, repetition, presence, frequency, bias, allowed, out)


def penalize_logits_eager(logits, tokens=None, prompt_lens=None, total_lens=None, repetition=1.0, presence=0.0, frequency=0.0,
                          bias=None, allowed=None, out=None) -> torch.Tensor:
    """The same computation with stock ops (CPU; fp64 logits for checks)."""
    def check(ok, message):
        if not ok:
            raise RuntimeError("penalize_logits: " + message)

    check(logits.dim() == 2, "logits must be [rows, vocabulary]")
    R, V = logits.shape
    dev = logits.device
    real = torch.float64 if logits.dtype == torch.float64 else torch.float32
    x = logits.to(real)

    def column(value, name, dtype):
        if not isinstance(value, torch.Tensor):
            return torch.full((1, 1), value, dtype=real, device=dev)
        check(value.dtype == dtype and value.dim() == 1 and value.numel() in (1, R), f"{name} must be one value or one per row")
        return value.view(-1, 1)

    if tokens is not None:
        check(tokens.dim() == 2 and tokens.shape[0] == R and tokens.dtype in (torch.int64, torch.int32),
              "tokens must be int64 or int32 [rows, history]")
        L = tokens.shape[1]
        j = torch.arange(L, device=dev)[None, :]
        total = column(L if total_lens is None else total_lens, "total_lens", torch.int32)
        prompt = column(0 if prompt_lens is None else prompt_lens, "prompt_lens", torch.int32)
        live = (j < total) & (tokens >= 0) & (tokens < V)
        at = torch.where(live, tokens.long(), torch.zeros_like(tokens, dtype=torch.int64))
        seen = torch.zeros(R, V, dtype=torch.int32, device=dev).scatter_add_(1, at, live.int()) > 0
        count = torch.zeros(R, V, dtype=torch.int32, device=dev).scatter_add_(1, at, (live & (j >= prompt)).int())
        rep = column(repetition, "repetition", torch.float32).to(real)
        x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
        lost = column(frequency, "frequency", torch.float32).to(real) * count.to(real) + \
            column(presence, "presence", torch.float32).to(real)
        x = torch.where(count > 0, x - lost, x)
    if bias is not None:
        check(bias.dtype == torch.float32 and bias.shape in ((V,), (R, V)), "bias must be fp32 [vocabulary] or [rows, vocabulary]")
        x = x + bias.to(real)
    if allowed is not None:
        words = (V + 31) // 32
        check(allowed.dtype == torch.int32 and allowed.shape in ((words,), (R, words)),
              "allowed must be int32 [(vocabulary + 31) / 32] or one such row per row of logits")
        v = torch.arange(V, device=dev)
        bit = (allowed[..., v // 32] >> (v % 32).to(torch.int32)) & 1
        x = x.masked_fill(bit == 0, float("-inf"))
    if out is None:
        return x.to(logits.dtype)
    check(out.shape == logits.shape and out.dtype == logits.dtype, "out must look like the logits")
    return out.copy_(x)
