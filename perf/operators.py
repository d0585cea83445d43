"""Cases of the ragged-batch generation operators: page planning, cache append, attention over a paged cache and
logit penalties.

``own = False`` computes every operator in its plain form (elementary torch operations, fp32, rounded once);
``own = True`` calls the framework's operators. ``exact`` is the definition in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one decode step of 64 chats: every request adds a token, a few cross into a new page
        dict(name="plan decode 64", op="plan", requests=64, single=64, tokens=64, pad=0, ctx=1000, page=16),
        # a step of chunked prefill: 200 decoding requests and 57 prompt chunks, padded to a fixed number of rows
        dict(name="plan mixed 257", op="plan", requests=257, single=200, tokens=8000, pad=192, ctx=4000, page=16),
        # the largest step: offline generation from thousands of prompts at once
        dict(name="plan prefill 4096", op="plan", requests=4096, single=0, tokens=524288, pad=0, ctx=64, page=16),
        # GPT-2 124M decode step (12 heads of 64), 64 requests
        dict(name="append decode 64", op="append", requests=64, tokens=64, pad=0, kv_heads=12, width=64, page=16, dtype="bf16"),
        # prompts of grouped-query heads, an odd number of rows and a padded tail
        dict(name="append prefill 32785", op="append", requests=9, tokens=32785, pad=111, kv_heads=8, width=128, page=32,
             dtype="bf16"),
        # GPT-2 124M: eight requests within its context, the smallest attention call of a decode step
        dict(name="attn decode 8 x 1k", op="attn", requests=8, single=8, tokens=8, pad=0, ctx=1000, heads=12, kv_heads=12, width=64,
             page=16, window=0, dtype="bf16"),
        # a full serving batch of grouped-query heads with uneven contexts
        dict(name="attn decode 64 x 8k", op="attn", requests=64, single=64, tokens=64, pad=0, ctx=8000, heads=32, kv_heads=8,
             width=128, page=16, window=0, dtype="bf16"),
        # two long documents, one token each: only a split along the keys fills the card
        dict(name="attn decode 2 x 128k", op="attn", requests=2, single=2, tokens=2, pad=0, ctx=131000, heads=32, kv_heads=8,
             width=128, page=64, window=0, dtype="fp16"),
        # chunked prefill next to decoding requests, sliding window, padded rows, pages that do not divide a tile
        dict(name="attn mixed window", op="attn", requests=33, single=31, tokens=1531, pad=5, ctx=3000, heads=16, kv_heads=4,
             width=64, page=24, window=1024, dtype="bf16"),
        # prompts of 1024 and more tokens worked off whole, on top of cached context: products, not bytes
        dict(name="attn prefill 16k", op="attn", requests=8, single=0, tokens=16000, pad=0, ctx=2000, heads=32, kv_heads=8,
             width=128, page=16, window=0, dtype="bf16"),
        # one request's next token
        dict(name="penalties 1", op="penalties", requests=1, vocab=50304, history=300, bias=False, mask=False, dtype="bf16"),
        # a serving batch under grammars, with logit biases and long histories
        dict(name="penalties 256", op="penalties", requests=256, vocab=50304, history=4000, bias=True, mask=True, dtype="fp32"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    """One more case: sizes spread over the logarithm of their ranges, none dearer than the dearest listed case."""
    top = [work(c) for c in listed() if c["op"] != "plan"]
    while True:
        case = _draw(rng)
        w = work(case)
        if w["bytes"] <= max(t["bytes"] for t in top) and w["flops"] <= max(t["flops"] for t in top):
            return case


def _draw(rng):
    op = rng.choice(["plan", "append", "attn", "attn", "penalties"])
    if op == "plan":
        requests = _log(rng, 1, 4096)
        single = rng.choice([requests, requests // 2, 0])
        tokens = single + (_log(rng, requests - single, 500000) if single < requests else 0)
        return dict(op=op, requests=requests, single=single, tokens=tokens, pad=rng.choice([0, rng.randrange(1, 300)]),
                    ctx=_log(rng, 1, 4000), page=rng.choice([1, 8, 16, 24, 32, 64, 128]))
    if op == "append":
        return dict(op=op, requests=_log(rng, 1, 64), tokens=_log(rng, 64, 32000), pad=rng.choice([0, rng.randrange(1, 200)]),
                    kv_heads=rng.choice([1, 2, 3, 4, 8, 12]), width=rng.choice([32, 64, 80, 128]),
                    page=rng.choice([1, 8, 16, 24, 32, 64, 128]), dtype=rng.choice(["bf16", "fp16", "fp32"]))
    if op == "attn":
        kv_heads = rng.choice([1, 2, 4, 8, 12])
        heads = kv_heads * rng.choice([1, 1, 3, 4, 8] if kv_heads <= 4 else [1, 2, 4])
        requests = _log(rng, 1, 64)
        # decode steps, a few chunks among decoding requests, or chunks alone
        single = rng.choice([requests, requests, max(0, requests - 2), 0])
        tokens = single + (_log(rng, requests - single, 16000) if single < requests else 0)
        ctx = _log(rng, 1, min(131000, 512000 // requests))
        return dict(op=op, requests=requests, single=single, tokens=tokens, pad=rng.choice([0, rng.randrange(1, 40)]), ctx=ctx,
                    heads=heads, kv_heads=kv_heads, width=rng.choice([32, 64, 64, 80, 128, 128]),
                    page=rng.choice([8, 16, 16, 24, 32, 64, 128]), window=rng.choice([0, 0, 0, _log(rng, 1, 4000)]),
                    dtype=rng.choice(["bf16", "bf16", "fp16"]))
    return dict(op=op, requests=_log(rng, 1, 256), vocab=rng.choice([50304, 50257, 65, 32000, _log(rng, 1000, 50000)]),
                history=_log(rng, 1, 4000), bias=rng.choice([False, True]), mask=rng.choice([False, True]),
                dtype=rng.choice(["bf16", "fp16", "fp32"]))


# ---- lengths ------------------------------------------------------------------------------------
def _lengths(case):
    """(new tokens, cached tokens) of every request: a function of the case alone, so that ``work`` knows them."""
    rng = random.Random("lengths %d %d %d %d" % (case["requests"], case["tokens"], case.get("ctx", 0), case["page"]))
    n, single = case["requests"], case.get("single", 0)
    rest = n - single
    chunks = []
    if rest:
        spread = [rng.uniform(0.5, 1.5) for _ in range(rest)]
        total = case["tokens"] - single
        chunks = [int(total * s / sum(spread)) for s in spread]
        chunks[-1] += total - sum(chunks)
    q = chunks + [1] * single
    top = case.get("ctx", 0)
    c = [rng.randint(max(0, top // 4), top) for _ in range(n)]
    return q, c


def _shuffled(case, seed):
    """The lengths in the seed's order of requests."""
    q, c = _lengths(case)
    order = list(range(len(q)))
    random.Random(seed).shuffle(order)
    return [q[i] for i in order], [c[i] for i in order]


def _pages(n, page):
    return (n + page - 1) // page


def _visible(q, c, window):
    """(query, key) pairs and keys that at least one query of the request sees."""
    pairs = keys = 0
    for n, ctx in zip(q, c):
        if n == 0:
            continue
        if window == 0:
            pairs += n * ctx + n * (n + 1) // 2
            keys += ctx + n
        else:
            pairs += sum(min(window, ctx + i + 1) for i in range(n))
            keys += min(ctx + n, window + n - 1)
    return pairs, keys


def work(case):
    op = case["op"]
    if op == "plan":
        q, c = _lengths(case)
        rows = sum(q) + case["pad"]
        fresh = sum(_pages(a + b, case["page"]) - _pages(b, case["page"]) for a, b in zip(q, c))
        return {"bytes": 16 * len(q) + 8 * rows + 8 * fresh, "flops": 0}
    if op == "append":
        row = 2 * case["kv_heads"] * case["width"] * _SIZE[case["dtype"]]
        return {"bytes": case["tokens"] * (2 * row + 4) + 4 * case["pad"], "flops": 0}
    if op == "attn":
        q, c = _lengths(case)
        pairs, keys = _visible(q, c, case["window"])
        size = _SIZE[case["dtype"]]
        return {"bytes": 2 * keys * case["kv_heads"] * case["width"] * size + 2 * sum(q) * case["heads"] * case["width"] * size,
                "flops": 4 * pairs * case["heads"] * case["width"]}
    per = 2 * _SIZE[case["dtype"]] + (4 if case["bias"] else 0)
    return {"bytes": case["requests"] * (case["vocab"] * per + (case["vocab"] // 8 if case["mask"] else 0) + 8 * case["history"]),
            "flops": 0}


# ---- inputs -------------------------------------------------------------------------------------
def _ints(values, device="cuda"):
    return torch.tensor(values, dtype=torch.int32).to(device)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _tables(lens, page, spare, g, width=None):
    """Pages of requests of the given lengths, scattered over a pool: (table [R, M], ids not in use)."""
    counts = [_pages(n, page) for n in lens]
    total = sum(counts) + spare
    ids = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    cols = max(counts) if width is None else width
    own_cols = torch.arange(cols, device="cuda")[None, :]
    n = _ints(counts)[:, None]
    first = torch.cumsum(n, 0) - n
    at = (first + own_cols).clamp_(max=max(total - 1, 0))
    table = torch.where(own_cols < n, ids[at], torch.full_like(at, -1).to(torch.int32))
    return table.to(torch.int32).contiguous(), ids[sum(counts):].contiguous()


def _randn(shape, dtype, g):
    """Normal values, drawn in pieces of bounded size in the target type."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    step = 1 << 26
    for i in range(0, flat.numel(), step):
        n = min(step, flat.numel() - i)
        flat[i:i + n] = torch.randn(n, generator=g, device="cuda")
    return out


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    s = dict(case)
    if op == "plan":
        q, c = _shuffled(case, seed)
        page = case["page"]
        fresh = sum(_pages(a + b, page) - _pages(b, page) for a, b in zip(q, c))
        cols = max(_pages(a + b, page) for a, b in zip(q, c))
        s["table"], s["free"] = _tables(c, page, fresh + 7, g, cols)
        s["q_lens"], s["ctx_lens"] = _ints(q), _ints(c)
        s["free_count"] = _ints([s["free"].numel()])
        s["rows"] = sum(q) + case["pad"]
        return s
    if op == "append":
        dt = _DT[case["dtype"]]
        rng = random.Random(seed)
        rows, page, heads, d = case["tokens"] + case["pad"], case["page"], case["kv_heads"], case["width"]
        # every request's tokens run through whole pages from some offset on; the pages lie anywhere in the pool
        cuts = sorted(rng.sample(range(1, case["tokens"]), case["requests"] - 1)) if case["requests"] > 1 else []
        lens = [b - a for a, b in zip([0] + cuts, cuts + [case["tokens"]])]
        offs = [rng.randrange(page) for _ in lens]
        used = sum(_pages(n + o, page) for n, o in zip(lens, offs))
        pool = _pages(case["tokens"], page) + 2 * case["requests"] + 5      # holds any cut
        table, _ = _tables([n + o for n, o in zip(lens, offs)], page, pool - used, g)
        slots = []
        host = table.cpu()
        for r, (n, o) in enumerate(zip(lens, offs)):
            pos = torch.arange(o, o + n)
            slots.append(host[r, pos // page] * page + pos % page)
        slots = torch.cat(slots + [torch.full((case["pad"],), -1)])
        s["slots"] = slots.to(torch.int32).cuda()
        s["k_pages"] = torch.zeros(pool, page, heads, d, dtype=dt, device="cuda")
        s["v_pages"] = torch.zeros_like(s["k_pages"])
        # the key and value columns of a fused projection with as many query heads again
        qkv = _randn((rows, 3 * heads * d), dt, g)
        s["k"] = qkv[:, heads * d: 2 * heads * d].view(rows, heads, d)
        s["v"] = qkv[:, 2 * heads * d:].view(rows, heads, d)
        return s
    if op == "attn":
        dt = _DT[case["dtype"]]
        q, c = _shuffled(case, seed)
        kv = [a + b for a, b in zip(q, c)]
        page, d = case["page"], case["width"]
        s["table"], _ = _tables(kv, page, 3, g)
        pool = sum(_pages(n, page) for n in kv) + 3
        s["k_pages"] = _randn((pool, page, case["kv_heads"], d), dt, g)
        s["v_pages"] = _randn((pool, page, case["kv_heads"], d), dt, g)
        rows = sum(q) + case["pad"]
        s["q"] = _randn((rows, case["heads"], d), dt, g) * 2
        cu = [0]
        for n in q:
            cu.append(cu[-1] + n)
        s["cu"], s["kv_lens"] = _ints(cu), _ints(kv)
        s["host_cu"], s["host_kv"] = cu, kv
        s["max_q"] = max(q)
        # rows behind the last sequence keep what the caller's buffer holds
        s["out"] = torch.zeros_like(s["q"])
        s["scale"] = 1.0 / math.sqrt(d)
        return s
    R, V, L = case["requests"], case["vocab"], case["history"]
    rng = random.Random(seed)
    s["logits"] = (torch.randn(R, V, generator=g, device="cuda") * 4).to(_DT[case["dtype"]])
    # a skewed vocabulary: few words make most of a text, so tokens repeat
    u = torch.rand(R, L, generator=g, device="cuda")
    s["tokens"] = (u.pow(4) * V).long().clamp_(max=V - 1)
    total = [rng.randint((L + 1) // 2, L) for _ in range(R)]
    prompt = [rng.randint(0, n) for n in total]
    s["prompt_lens"], s["total_lens"] = _ints(prompt), _ints(total)
    s["repetition"] = (torch.rand(R, generator=g, device="cuda") * 0.5 + 1).float()
    s["presence"] = torch.rand(R, generator=g, device="cuda").float()
    s["frequency"] = (torch.rand(R, generator=g, device="cuda") * 0.5).float()
    s["bias_v"] = (torch.randn(R, V, generator=g, device="cuda") * (torch.rand(R, V, generator=g, device="cuda") < 0.01)
                   ).float() if case["bias"] else None
    words = (V + 31) // 32
    s["allowed"] = torch.randint(-(1 << 31), 1 << 31, (R, words), generator=g, device="cuda",
                                 dtype=torch.int64).to(torch.int32) if case["mask"] else None
    return s


# ---- one pass -----------------------------------------------------------------------------------
def run(state):
    op = state["op"]
    if own:
        from distributed_pytorch_amd import ops
        if op == "plan":
            p = ops.paged_plan(state["q_lens"], state["ctx_lens"], state["table"], state["free"], state["free_count"],
                               state["page"], state["rows"])
            return [state["table"], p.cu_q, p.kv_lens, p.positions, p.slots, p.free_left]
        if op == "append":
            ops.paged_append(state["k_pages"], state["v_pages"], state["k"], state["v"], state["slots"])
            return [state["k_pages"], state["v_pages"]]
        if op == "attn":
            return ops.paged_attention(state["q"], state["k_pages"], state["v_pages"], state["table"], state["cu"],
                                       state["kv_lens"], state["scale"], window=state["window"] or None,
                                       max_q=state["max_q"], out=state["out"])
        return ops.penalize_logits(state["logits"], state["tokens"], state["prompt_lens"], state["total_lens"],
                                   repetition=state["repetition"], presence=state["presence"], frequency=state["frequency"],
                                   bias=state["bias_v"], allowed=state["allowed"])
    return {"plan": _plain_plan, "append": _plain_append, "attn": _plain_attn, "penalties": _plain_penalties}[op](state)


def _plain_plan(s):
    page, rows, table = s["page"], s["rows"], s["table"]
    cols = table.shape[1]
    q, c = s["q_lens"].clamp(min=0).long(), s["ctx_lens"].clamp(min=0).long()
    cu = torch.cat([q.new_zeros(1), q.cumsum(0)]).clamp_(max=rows)
    kv = c + cu[1:] - cu[:-1]
    have = ((c + page - 1) // page).clamp(max=cols)
    need = (((kv + page - 1) // page).clamp(max=cols) - have).clamp(min=0)
    first = need.cumsum(0) - need
    count = s["free_count"][0].long()
    col = torch.arange(cols, device=table.device)[None, :]
    nth = first[:, None] + col - have[:, None]
    fresh = (col >= have[:, None]) & (col < (have + need)[:, None])
    at = (count - 1 - nth).clamp(min=0, max=s["free"].numel() - 1)
    page_of = torch.where(nth < count, s["free"][at], torch.full_like(at, -1).int())
    table.copy_(torch.where(fresh, page_of, table))
    i = torch.arange(rows, device=table.device)
    r = torch.searchsorted(cu[1:].contiguous(), i, right=True)
    live = r < q.numel()
    r = r.clamp(max=q.numel() - 1)
    pos = torch.where(live, c[r] + i - cu[r], torch.zeros_like(i))
    in_table = live & (pos // page < cols)
    held = table[r, (pos // page).clamp(max=cols - 1)].long()
    slot = torch.where(in_table & (held >= 0), held * page + pos % page, torch.full_like(i, -1))
    total = need.sum()
    wanted = ((kv + page - 1) // page - (c + page - 1) // page).sum()
    had = torch.minimum(total, count)
    left = torch.stack([count - had, wanted - had])
    return [table, cu.int(), kv.int(), pos.int(), slot.int(), left.int()]


def _plain_append(s):
    n = s["tokens"]
    slots = s["slots"][:n].long()
    for pages, new in ((s["k_pages"], s["k"]), (s["v_pages"], s["v"])):
        pages.view(-1, *pages.shape[2:]).index_copy_(0, slots, new[:n])
    return [s["k_pages"], s["v_pages"]]


def _attend(s, real):
    """The rows of every request in the type ``real``: scores, mask, softmax and products one after another, a bounded
    number of rows at a time."""
    cu, kv, page, window = s["host_cu"], s["host_kv"], s["page"], s["window"]
    heads, kvh, d = s["heads"], s["kv_heads"], s["width"]
    group = heads // kvh
    outs = []
    for r, n_kv in enumerate(kv):
        a, b = cu[r], cu[r + 1]
        if a == b:
            continue
        ids = s["table"][r, :_pages(n_kv, page)].long()
        k = s["k_pages"][ids].reshape(-1, kvh, d)[:n_kv].to(real).permute(1, 2, 0).contiguous()       # [kvh, d, n_kv]
        v = s["v_pages"][ids].reshape(-1, kvh, d)[:n_kv].to(real).permute(1, 0, 2).contiguous()       # [kvh, n_kv, d]
        key = torch.arange(n_kv, device=k.device)
        step = max(1, (1 << 28) // (n_kv * heads))
        for i in range(a, b, step):
            j = min(b, i + step)
            q = s["q"][i:j].to(real).view(j - i, kvh, group, d).permute(1, 2, 0, 3).reshape(kvh, group * (j - i), d)
            score = torch.matmul(q, k).view(kvh, group, j - i, n_kv) * s["scale"]
            pos = torch.arange(i, j, device=k.device) + (n_kv - b)
            seen = key[None, :] <= pos[:, None]
            if window:
                seen = seen & (key[None, :] > pos[:, None] - window)
            score = score.masked_fill(~seen, float("-inf"))
            top = score.max(-1, keepdim=True).values
            p = torch.exp(score - top)
            o = torch.matmul(p.view(kvh, group * (j - i), n_kv), v) / p.sum(-1).view(kvh, -1, 1)
            outs.append(o.view(kvh, group, j - i, d).permute(2, 0, 1, 3).reshape(j - i, heads, d))
    return torch.cat(outs)


def _plain_attn(s):
    o = _attend(s, torch.float32)
    s["out"][:o.shape[0]] = o.to(s["out"].dtype)
    return s["out"]


def _penalties(s, real):
    x = s["logits"].to(real)
    R, V = x.shape
    L = s["tokens"].shape[1]
    j = torch.arange(L, device=x.device)[None, :]
    live = (j < s["total_lens"][:, None])
    made = live & (j >= s["prompt_lens"][:, None])
    count = torch.zeros(R, V, dtype=torch.int32, device=x.device).scatter_add_(1, s["tokens"], made.int())
    any_ = torch.zeros(R, V, dtype=torch.int32, device=x.device).scatter_add_(1, s["tokens"], live.int())
    rep = s["repetition"].to(real)[:, None]
    x = torch.where(any_ > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - (s["frequency"].to(real)[:, None] * count.to(real) + s["presence"].to(real)[:, None] * (count > 0).to(real))
    if s["bias_v"] is not None:
        x = x + s["bias_v"].to(real)
    if s["allowed"] is not None:
        v = torch.arange(V, device=x.device)
        bit = (s["allowed"][:, v // 32] >> (v % 32).int()) & 1
        x = x.masked_fill(bit == 0, float("-inf"))
    return x


def _plain_penalties(s):
    return _penalties(s, torch.float32).to(s["logits"].dtype)


# ---- the definition in 64 bits --------------------------------------------------------------------
def exact(case, seed):
    """From the definitions, one row, page or head at a time; None for the operator that only counts."""
    if case["op"] == "append":
        s = prepare(case, seed)
        pools = []
        for new, pages in ((s["k"], s["k_pages"]), (s["v"], s["v_pages"])):
            pool = torch.zeros(pages.shape, dtype=torch.float64, device="cuda")
            at = s["slots"].long()
            kept = torch.nonzero(at >= 0).flatten()
            pool[at[kept] // case["page"], at[kept] % case["page"]] = new[kept].double()
            pools.append(pool)
        return pools
    if case["op"] == "attn":
        s = prepare(case, seed)
        group, window = case["heads"] // case["kv_heads"], case["window"]
        out = s["out"].double()
        for r, n_kv in enumerate(s["host_kv"]):
            a, b = s["host_cu"][r], s["host_cu"][r + 1]
            slots = (s["table"][r].long()[:, None] * case["page"] + torch.arange(case["page"], device="cuda")).flatten()[:n_kv]
            for g in range(case["kv_heads"]):
                k = s["k_pages"].flatten(0, 1)[slots, g].double()
                v = s["v_pages"].flatten(0, 1)[slots, g].double()
                for i in range(a, b, 512):
                    j = min(b, i + 512)
                    pos = n_kv - b + torch.arange(i, j, device="cuda")
                    hide = torch.arange(n_kv, device="cuda") > pos[:, None]
                    if window:
                        hide |= torch.arange(n_kv, device="cuda") <= pos[:, None] - window
                    for h in range(g * group, (g + 1) * group):
                        z = s["q"][i:j, h].double() @ k.t() * s["scale"]
                        out[i:j, h] = torch.softmax(z.masked_fill_(hide, -math.inf), -1) @ v
        return out
    if case["op"] == "penalties":
        s = prepare(case, seed)
        rows = []
        V = case["vocab"]
        for r in range(case["requests"]):
            n, p = int(s["total_lens"][r]), int(s["prompt_lens"][r])
            made = torch.bincount(s["tokens"][r, p:n], minlength=V).double()
            seen = torch.bincount(s["tokens"][r, :n], minlength=V) > 0
            z = s["logits"][r].double()
            rep = s["repetition"][r].double()
            z = torch.where(seen, torch.where(z > 0, z / rep, z * rep), z)
            z = z - s["frequency"][r].double() * made - s["presence"][r].double() * (made > 0)
            if case["bias"]:
                z = z + s["bias_v"][r].double()
            if case["mask"]:
                bits = (s["allowed"][r][:, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
                z = torch.where(bits.flatten()[:V] == 1, z, torch.full_like(z, -math.inf))
            rows.append(z)
        return torch.stack(rows)
    return None
