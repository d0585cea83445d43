"""Offsets of the requests that decrease: paged attention stays inside its buffers."""
import pytest
import torch

from distributed_pytorch_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


CASES = {
    "more items than workgroups": ([0, 400, 0, 400, 0, 368, 400], [0, 0, 0, 0, 0, 100000], 400, 32, 8),
    "alternating": ([0, 1024] * 128, [1024] * 254 + [100000], 1024, 1, 1),
    "many requests": ([0, 300] * 200, [500] * 398 + [60000], 300, 4, 2),
    "few rows": ([0, 8, 0, 8, 3, 8], [3000, 50000, 20, 7, 90000], 8, 4, 2),
}


@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_decreasing_offsets_leave_everything_outside_alone(name, dtype):
    cu, kv, N, nh, nkv = CASES[name]
    if dtype == torch.float32 and N > 400:
        cu, kv, N = cu[:9], kv[:8], 100
    page, P, d = 16, 64, 64
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v = (torch.randn(P, page, nkv, d, device=DEV, generator=g).to(dtype) for _ in range(2))
    table = torch.randint(0, P, (len(kv), -(-max(kv) // page)), device=DEV, generator=g).int()
    q = torch.randn(N, nh, d, device=DEV, generator=g).to(dtype)
    room = torch.full((3 * N, nh, d), 5.0, dtype=dtype, device=DEV)
    for max_q in (None, 1):
        # scratch memory that comes back from the allocator full of large numbers
        junk = [torch.full((1 << 20,), 0x7f7f7f7f, dtype=torch.int32, device=DEV) for _ in range(8)]
        del junk
        out = room[N:2 * N]
        ops.paged_attention(q, k, v, table, i32(*cu), i32(*kv), max_q=max_q, out=out)
        fresh = ops.paged_attention(q, k, v, table, i32(*cu), i32(*kv), max_q=max_q)
        torch.cuda.synchronize()
        assert (room[:N] == 5).all() and (room[2 * N:] == 5).all()
        if dtype != torch.float32:
            assert (out == 5).all() and (fresh == 0).all()       # no row is computed
    # the same buffers with offsets in order
    good = sorted(min(c, N) for c in cu)
    o = ops.paged_attention(q, k, v, table, i32(*good), i32(*[900] * len(kv)))
    assert torch.isfinite(o).all() and o.abs().max().item() > 0
