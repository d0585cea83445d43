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
