"""Generation over the paged cache and with penalties: the same function as the dense paths, on the CPU and the GPU."""
import json
import subprocess
import sys

import pytest
import torch

from distributed_pytorch_amd import ops
from distributed_pytorch_amd.config import LLMconfig, Trainconfig
from distributed_pytorch_amd.models.llm import LLM, PagedKVCache

SMALL = dict(vocab_size=97, block_size=48, n_embd=32, n_layer=2, n_head=4, up_dim=48)
VARIANTS = {
    "mha_learn": dict(attn="mha", pos_emb="learn", non_linearity="gelu"),
    "gqa_rope": dict(attn="gqa", n_kv_heads=2, pos_emb="rope", non_linearity="swiglu"),
    "mqa_sin_moe": dict(attn="mqa", pos_emb="sin", non_linearity="gelu", moe=True, n_exp=4, n_shared=1, n_act=2),
}


def model_of(name, base=SMALL, device="cpu", dtype=torch.float32):
    torch.manual_seed(0)
    return LLM(LLMconfig(**{**base, **VARIANTS[name]}).finalize()).to(device).to(dtype).eval()


def paged_logits(m, tokens, steps, page_size, pad=0):
    """Logits of every request's newest row after each step; steps[t][r] = tokens of request r worked off in step t."""
    dev = m.lm_head.weight.device
    R = len(tokens)
    cache = PagedKVCache(m.config, R, max(len(t) for t in tokens), sum(-(-len(t) // page_size) for t in tokens), dev,
                         m.lm_head.weight.dtype, page_size)
    done, out = [0] * R, []
    for step in steps:
        rows = [tokens[r][done[r]: done[r] + n] for r, n in enumerate(step)]
        flat = torch.cat([torch.tensor(x, dtype=torch.int64) for x in rows] + [torch.zeros(pad, dtype=torch.int64)])
        cache.begin(torch.tensor(step, dtype=torch.int32).to(dev), flat.numel())
        with torch.no_grad():
            logits, _, _ = m(flat[None].to(dev), kv_caches=cache)
        cache.commit()
        assert logits.shape == (R, 1, m.config.vocab_size)
        done = [a + b for a, b in zip(done, step)]
        out.append((list(done), logits[:, 0].float()))
    assert cache.free_left[1].item() == 0
    return out


@pytest.mark.parametrize("name", sorted(VARIANTS))
def test_packed_steps_give_the_dense_logits(name):
    m = model_of(name)
    tokens = [torch.randint(0, 97, (n,)).tolist() for n in (20, 5, 33)]
    for done, logits in paged_logits(m, tokens, [[7, 5, 1], [1, 0, 30], [12, 0, 2]], page_size=8, pad=3):
        for r, n in enumerate(done):
            with torch.no_grad():
                want, _, _ = m(torch.tensor(tokens[r][:n])[None])
            # rows of requests without new tokens are another's
            if (r, n) != (1, 5) or done == [7, 5, 1]:
                assert torch.allclose(logits[r], want[0, -1], rtol=1e-4, atol=1e-5)


def test_ragged_generation_equals_one_by_one():
    m = model_of("gqa_rope")
    prompts = [torch.randint(0, 97, (n,)) for n in (3, 17, 1)]
    out = m.generate_ragged(prompts, 9, topk=1, page_size=4)
    for p, o in zip(prompts, out):
        assert torch.equal(o, m.generate(p[None], 9, topk=1)[0])
    pen = dict(repetition=1.8, presence=0.3, frequency=0.4, bias=torch.randn(97))
    out = m.generate_ragged(prompts, 9, topk=1, penalties=pen)
    for p, o in zip(prompts, out):
        assert torch.equal(o, m.generate(p[None], 9, topk=1, penalties=pen)[0])
    assert not m.training


def test_penalties_and_masks_steer_generation():
    m = model_of("mha_learn")
    idx = torch.randint(0, 97, (2, 5))
    allowed = torch.zeros(4, dtype=torch.int32)
    allowed[2] = 0b1010                           # tokens 65 and 67
    out = m.generate(idx, 12, topk=None, penalties=dict(allowed=allowed))
    assert set(out[:, 5:].unique().tolist()) <= {65, 67}
    out = m.generate(idx, 40, topk=1, penalties=dict(frequency=1e4))       # nothing twice while anything is left
    assert all(len(set(row[5:].tolist())) == 40 for row in out)
    assert torch.equal(m.generate(idx, 12, topk=1, penalties={}), m.generate(idx, 12, topk=1))


def test_refusals():
    m = model_of("gqa_rope")
    p = [torch.tensor([1, 2])]
    for bad in ([], [torch.zeros(0, dtype=torch.int64)]):
        with pytest.raises(ValueError):
            m.generate_ragged(bad, 4)
    with pytest.raises(ValueError):
        m.generate_ragged(p, 0)
    with pytest.raises(ValueError):
        m.generate_ragged(p, 48)                  # 2 + 48 - 1 rows in a context of 48
    assert m.generate_ragged(p, 47)[0].numel() == 49
    mla = LLM(LLMconfig(**SMALL, attn="mla", pos_emb="learn", q_latent_dim=8, kv_latent_dim=16).finalize())
    with pytest.raises(ValueError):
        mla.generate_ragged(p, 4)


def test_sampling_script_takes_several_prompts_and_penalties(tmp_path):
    m = model_of("mha_learn", dict(SMALL, vocab_size=256))
    path = str(tmp_path / "m_ckpt.pt")
    torch.save({"model_config_dict": m.config.to_dict(), "train_config": Trainconfig(), "model_state": m.state_dict()}, path)
    r = subprocess.run([sys.executable, "single-gpu/sample.py", "--ckpt", path, "--prompt", "a", "to be", "--tokenizer", "bytes", "--token_ids",
                        "--max_new_tokens", "6", "--device", "cpu", "--repetition_penalty", "1.3", "--num_samples", "2"],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    rows = [json.loads(x) for x in r.stdout.splitlines() if x.startswith("[") and not x.startswith("[sample]")]
    assert [len(x) for x in rows] == [7, 7, 11, 11]


# ---- GPU ---------------------------------------------------------------------------------------------
BIG = dict(vocab_size=512, block_size=256, n_embd=256, n_layer=3, n_head=4, up_dim=512)


@pytest.mark.gpu
@pytest.mark.parametrize("name,heads", [("mha_learn", 4), ("gqa_rope", 4), ("gqa_rope", 2), ("mqa_sin_moe", 8)])
def test_packed_steps_on_the_gpu(name, heads):
    """bf16 over the paged cache is as far from fp32 as the dense bf16 forward is."""
    base = dict(BIG, n_head=heads)
    ref = model_of(name, base, "cuda")
    m = model_of(name, base, "cuda", torch.bfloat16)
    tokens = [torch.randint(0, 512, (n,)).tolist() for n in (200, 40, 131)]
    for done, logits in paged_logits(m, tokens, [[130, 39, 1], [69, 0, 129], [1, 1, 1]], page_size=16, pad=5):
        for r, n in enumerate(done):
            if r == 1 and done == [199, 39, 130]:
                continue                            # no new tokens: another request's row
            x = torch.tensor(tokens[r][:n], device="cuda")[None]
            with torch.no_grad():
                exact, dense = ref(x)[0][0, -1], m(x)[0][0, -1].float()
            assert (logits[r] - exact).norm() <= 2 * (dense - exact).norm() + 1e-2 * exact.norm()


@pytest.mark.gpu
@pytest.mark.parametrize("penalties", [None, dict(repetition=1.5, frequency=0.2)])
def test_ragged_generation_on_the_gpu(penalties):
    """fp32, so that greedy tokens are the dense path's; the captured steps give what the eager ones give."""
    m = model_of("gqa_rope", BIG, "cuda")
    prompts = [torch.randint(0, 512, (n,), device="cuda") for n in (3, 100, 1, 17, 64)]
    eager = m.generate_ragged(prompts, 24, topk=1, hip_graph=False, penalties=penalties)
    graphed = m.generate_ragged(prompts, 24, topk=1, penalties=penalties)
    assert m.last_decode_graphed
    for p, a, b in zip(prompts, eager, graphed):
        assert torch.equal(a, b)
        one = m.generate(p[None], 24, topk=1, hip_graph=False, penalties=penalties)[0]
        assert (a == one).float().mean().item() > 0.9           # (a near-tie may flip and carry on)


@pytest.mark.gpu
@pytest.mark.parametrize("capture", [True, False])
def test_ragged_generation_with_experts(capture, monkeypatch):
    """Whether or not the step can be captured, the tokens are those of the eager steps."""
    m = model_of("mqa_sin_moe", BIG, "cuda", torch.bfloat16)
    prompts = [torch.randint(0, 512, (n,), device="cuda") for n in (70, 2, 33)]
    eager = m.generate_ragged(prompts, 12, topk=1, hip_graph=False)
    assert not m.last_decode_graphed
    if not capture:
        def refuse(*a, **k):
            raise RuntimeError("not captured")
        monkeypatch.setattr(torch.cuda, "graph", refuse)
    out = m.generate_ragged(prompts, 12, topk=1)
    assert capture or not m.last_decode_graphed
    for a, b in zip(eager, out):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_penalties_in_the_captured_dense_step():
    m = model_of("mha_learn", BIG, "cuda", torch.bfloat16)
    idx = torch.randint(0, 512, (3, 9), device="cuda")
    pen = dict(frequency=1e4)
    graphed = m.generate(idx, 60, topk=1, penalties=pen)
    assert m.last_decode_graphed and torch.equal(graphed[:, :9], idx)
    assert all(len(set(row[9:].tolist())) == 60 for row in graphed)
    eager = m.generate(idx, 60, topk=1, hip_graph=False, penalties=pen)
    assert all(len(set(row[9:].tolist())) == 60 for row in eager)
    bf16 = model_of("gqa_rope", BIG, "cuda", torch.bfloat16)
    out = bf16.generate_ragged([idx[0], idx[1, :4]], 50, topk=1, penalties=pen)
    assert bf16.last_decode_graphed and all(len(set(o[n:].tolist())) == 50 for o, n in zip(out, (9, 4)))
    assert ops.penalize_logits(torch.zeros(1, 8, device="cuda")).sum().item() == 0
