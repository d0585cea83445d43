"""Greedy ragged generation against the dense model, token by token: the generated tokens alone, up to rounding."""
import pytest
import torch

from distributed_pytorch_amd import ops
from distributed_pytorch_amd.config import LLMconfig
from distributed_pytorch_amd.models.llm import LLM

CFG = dict(vocab_size=512, block_size=256, n_embd=256, n_layer=3, n_head=4, up_dim=512)


def dense_logits(m, tokens, prompt, penalties):
    with torch.no_grad():
        x = m(tokens[None])[0][0, -1:].float()
    if penalties:
        x = ops.penalize_logits_eager(x, tokens[None], torch.tensor([prompt], dtype=torch.int32, device=x.device), **penalties)
    return x[0]


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("penalties", [None, dict(repetition=1.5, frequency=0.2, presence=0.1)])
@pytest.mark.parametrize("variant", [dict(attn="gqa", n_kv_heads=2, pos_emb="rope", non_linearity="swiglu"),
                                     dict(attn="mha", pos_emb="learn", non_linearity="gelu")])
def test_every_generated_token_is_the_dense_models_choice(device, penalties, variant):
    """Each token, given the ones before it, is the largest logit of a dense forward, or as large as it within what the
    roundings of two fp32 evaluations allow: a product of K terms is off by at most K 2^-24 |x| |w|, K is at most 512, the
    hidden state goes through 4 products in each of 3 layers and one at the end (13), and both sides have that error. The
    penalties scale a logit by 1.5 at most."""
    torch.manual_seed(0)
    m = LLM(LLMconfig(**CFG, **variant).finalize()).to(device).eval()
    prompts = [torch.randint(0, 512, (n,), device=device) for n in (3, 100, 1, 17, 64)]
    # |x| of the normalised state is sqrt(256) = 16 (weights 1), |w| that of the longest row
    tol = 1.5 * 2 * 13 * 512 * 2.0 ** -24 * 16 * m.lm_head.weight.detach().float().norm(dim=1).max().item()
    graphs = (False, True) if device == "cuda" else (False,)
    for graph in graphs:
        out = m.generate_ragged(prompts, 20, topk=1, hip_graph=graph, penalties=penalties)
        close = 0
        for p, o in zip(prompts, out):
            assert torch.equal(o[:len(p)], p) and o.numel() == len(p) + 20
            for t in range(len(p), o.numel()):
                x = dense_logits(m, o[:t], len(p), penalties)
                short = (x.max() - x[o[t]]).item()
                assert short <= tol, (graph, len(p), t, short, tol)
                close += short > 0
        assert close <= 5                        # of 100: nearly every choice is the same one
