"""PagedKVCache over several steps: what its counters and rows say."""
import pytest
import torch

from distributed_pytorch_amd.config import LLMconfig
from distributed_pytorch_amd.models.llm import LLM, PagedKVCache

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def small(device, dtype=torch.float32, **kw):
    torch.manual_seed(0)
    cfg = dict(vocab_size=96, block_size=48, n_embd=128, n_layer=2, n_head=2, up_dim=64, attn="gqa", n_kv_heads=1, pos_emb="rope",
               non_linearity="gelu")
    return LLM(LLMconfig(**{**cfg, **kw}).finalize()).to(device).to(dtype).eval()


def step(m, cache, q_lens, tokens):
    dev = m.lm_head.weight.device
    cache.begin(torch.tensor(q_lens, dtype=torch.int32, device=dev), len(tokens))
    with torch.no_grad():
        logits, _, _ = m(torch.tensor([tokens], device=dev), kv_caches=cache)
    cache.commit()
    return logits


@pytest.mark.parametrize("device", DEVICES)
def test_a_shortage_of_pages_is_not_forgotten(device):
    """Four rows to a page and two pages: the third page is asked for once, in the second step, and the count stays."""
    m = small(device)
    cache = PagedKVCache(m.config, 1, 20, 2, device, torch.float32, 4)
    step(m, cache, [7], list(range(7)))
    assert cache.free_left.tolist() == [0, 0]
    step(m, cache, [2], [1, 2])
    assert cache.free_left.tolist() == [0, 1]
    for _ in range(3):                        # rows of the page that is missing: nothing new is asked for
        step(m, cache, [1], [3])
        assert cache.free_left.tolist() == [0, 1]
    step(m, cache, [1], [3])
    assert cache.free_left.tolist() == [0, 2] and cache.ctx_lens.tolist() == [13]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("pos_emb", ["learn", "sin", "rope"])
def test_steps_past_the_context_stay_inside_the_position_tables(device, pos_emb):
    """Lengths are not known to the host, so nothing refuses such a step: it must not read past the tables."""
    m = small(device, pos_emb=pos_emb, block_size=16)
    cache = PagedKVCache(m.config, 2, 16, 8, device, torch.float32, 8)
    step(m, cache, [16, 1], list(range(17)))
    inside = step(m, cache, [0, 1], [5])[1]
    both = step(m, cache, [3, 1], [7, 8, 9, 5])
    assert cache.ctx_lens.tolist() == [19, 3] and cache.free_left.tolist() == [8 - 3, 1]
    assert torch.isfinite(both).all() and torch.isfinite(inside).all()
    # the request that kept inside is not disturbed
    alone = PagedKVCache(m.config, 1, 16, 8, device, torch.float32, 8)
    want = step(m, alone, [3], [16, 5, 5])
    assert torch.allclose(both[1], want[0], rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("device", DEVICES)
def test_requests_without_new_tokens_have_no_logits(device):
    """Their rows are zero, not another request's logits: at the front, between others and at the end."""
    m = small(device)
    cache = PagedKVCache(m.config, 4, 20, 20, device, torch.float32, 4)
    first = step(m, cache, [0, 3, 0, 2], [1, 2, 3, 4, 5, 0, 0])       # two rows of padding
    assert (first[[0, 2]] == 0).all()
    with torch.no_grad():
        for r, tokens in ((1, [1, 2, 3]), (3, [4, 5])):
            want = m(torch.tensor([tokens], device=device))[0][0, -1]
            assert torch.allclose(first[r, 0], want, rtol=1e-4, atol=1e-4)
    then = step(m, cache, [2, 0, 1, 0], [6, 7, 8])
    assert (then[[1, 3]] == 0).all() and (then[[0, 2]] != 0).any(-1).all()
