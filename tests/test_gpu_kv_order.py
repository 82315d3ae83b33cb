"""GPU checks that attention sees the lengths and tables as the launch just
before it left them, where they change how many splits are joined."""
import pytest
import torch

from test_gpu_kv_attention import Batch, attn  # noqa: F401  (attn: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens", [[(9000, 1)], [(9000, 2), (7000, 1), (8000, 1)], [(9000, 40)]])
def test_lengths_that_change_between_calls(attn, lens):  # noqa: F811
    b = Batch(lens, 8, 2, 128, 16, "bf16", seed=21)
    long = b.seq_lens.clone()
    short = torch.tensor([130 + 40 * i for i in range(len(lens))], dtype=torch.int32, device="cuda")
    away = torch.full_like(b.table, -1)
    table = b.table.clone()
    steps = [(long, table), (short, table), (long, away), (short, table), (long, table)]
    want = []
    for n, t in steps:
        b.seq_lens.copy_(n)
        b.table.copy_(t)
        torch.cuda.synchronize()
        want.append(b.call(attn))
        torch.cuda.synchronize()
    assert bool((want[2] == 0).all()) and not torch.equal(want[0], want[1])
    got = []
    for _ in range(10):
        for n, t in steps:
            b.table.copy_(t)
            b.seq_lens.copy_(n)
            got.append(b.call(attn))
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert torch.equal(out, want[i % len(steps)]), i
