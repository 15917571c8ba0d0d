"""Edges of the training operators on a GPU.  Whole numbers make every fp32 sum exact in any order, so
results on them are compared for equality after the one rounding."""
import pytest
import torch

import deepgemm
from deepgemm import grouped_bf16_input_grad, grouped_bf16_weight_grad

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def whole(gen, *shape, lim=4):
    return torch.randint(-lim, lim + 1, shape, generator=gen).bfloat16()


def packed(w):  # [G, N, K] -> [G, K/64, N, 64]
    g, n, k = w.shape
    return w.view(g, n, k // 64, 64).transpose(1, 2).contiguous()


@pytest.mark.parametrize("tile", [128, 256, 1])
def test_ragged_steps_are_read_after_they_are_written(tile):
    """Blocks whose rows that count lie between others go step by step through ordinary stores: 8 steps a
    block, 40 blocks a group, all of them one behind another, time and again."""
    gen = torch.Generator().manual_seed(7)
    g, n, k, blocks = 2, 272, 320, 80
    mi = (torch.arange(blocks) % g).repeat_interleave(128).int()
    first = torch.arange(blocks) * 128
    mi[torch.rand(mi.numel(), generator=gen) < 0.4] = -1
    mi[first] = (torch.arange(blocks) % g).int()
    dy, x = whole(gen, mi.numel(), n), whole(gen, mi.numel(), k)
    dy[mi < 0], x[mi < 0] = float("nan"), float("inf")
    want = torch.zeros(g, n, k, dtype=torch.float64)
    for e in range(g):
        r = mi == e
        want[e] = dy[r].double().T @ x[r].double()
    want = packed(want).float().to(DEV)
    args = dy.to(DEV), x.to(DEV), mi.to(DEV), g
    for _ in range(50):
        assert torch.equal(grouped_bf16_weight_grad(*args, dtype=F32, tile=tile), want)
    deepgemm.check_device_status()
