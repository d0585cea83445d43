"""The grouped weight gradient inside a captured step."""
import pytest
import torch

from distributed_pytorch_amd._ext import ops

pytestmark = pytest.mark.gpu


def test_grouped_weight_gradient_replayed():
    """Few groups over many rows: the rows are split and summed into a buffer that every replay has to clear first. Whole
    numbers up to 4, so that sums below 2^24 are exact in any order."""
    G, rows, N, K = 2, 4096, 128, 128
    g = torch.Generator(device="cuda").manual_seed(0)
    dy, x = (torch.randint(-4, 5, (G * rows, w), device="cuda", generator=g).bfloat16() for w in (N, K))
    start, seg = torch.tensor([0, rows], device="cuda"), torch.tensor([rows, rows], device="cuda")

    def want():
        return torch.stack([dy[i * rows:(i + 1) * rows].float().t() @ x[i * rows:(i + 1) * rows].float() for i in range(G)])

    assert torch.equal(ops().grouped_wgrad(dy, x, start, seg).view(G, N, K), want())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops().grouped_wgrad(dy, x, start, seg)
    for _ in range(5):
        dy.copy_(torch.randint(-4, 5, dy.shape, device="cuda", generator=g))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.view(G, N, K), want())
        (torch.randn(1000, device="cuda") @ torch.randn(1000, 50, device="cuda")).sum().item()
