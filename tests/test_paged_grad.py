"""The ragged-batch operators have no gradients, and say so."""
import pytest
import torch

from distributed_pytorch_amd import ops
from distributed_pytorch_amd.config import LLMconfig
from distributed_pytorch_amd.models.llm import LLM, PagedKVCache


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_a_paged_forward_records_nothing(device):
    """With gradients on, as without: logits and pools carry no graph, and no gradient can be asked of them."""
    torch.manual_seed(0)
    m = LLM(LLMconfig(vocab_size=96, block_size=48, n_embd=128, n_layer=2, n_head=2, up_dim=64, attn="mha", pos_emb="learn",
                      non_linearity="gelu").finalize()).to(device).eval()
    got = []
    for grad in (True, False):
        cache = PagedKVCache(m.config, 1, 16, 4, device, torch.float32, 4)
        cache.begin(torch.tensor([5], dtype=torch.int32, device=device), 5)
        with torch.set_grad_enabled(grad):
            logits, _, _ = m(torch.arange(5, device=device)[None], kv_caches=cache)
        cache.commit()
        assert not logits.requires_grad and not any(t.requires_grad for t in cache.k + cache.v)
        got.append(logits)
    assert torch.equal(got[0], got[1])
    with pytest.raises(RuntimeError):
        got[0].sum().backward()


@pytest.mark.gpu
def test_gradients_are_refused_on_the_gpu():
    dev = "cuda"
    t, one, cu = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([[0, 1]], [1], [0, 1]))
    k, v, q, row = (torch.randn(s, device=dev) for s in ((2, 4, 1, 8), (2, 4, 1, 8), (1, 2, 8), (1, 1, 8)))
    lg = torch.randn(2, 40, device=dev)
    def needs(x):
        return x.clone().requires_grad_()
    calls = [
        lambda f: ops.paged_append(k, v, f(row), row, one), lambda f: ops.paged_append(k, v, row, f(row), one),
        lambda f: ops.paged_attention(f(q), k, v, t, cu, one), lambda f: ops.paged_attention(q, f(k), v, t, cu, one),
        lambda f: ops.paged_attention(q, k, f(v), t, cu, one), lambda f: ops.penalize_logits(f(lg)),
        lambda f: ops.penalize_logits(lg, bias=f(lg)), lambda f: ops.penalize_logits(lg, presence=f(torch.ones(1, device=dev))),
    ]
    for call in calls:
        with pytest.raises(RuntimeError, match="no gradient"):
            call(needs)
        with torch.no_grad():
            call(needs)
        call(lambda x: x)
