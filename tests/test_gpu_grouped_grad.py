"""Gradients of the contiguous BF16 grouped GEMM against plain 64-bit products.

Small whole numbers make every fp32 sum exact in any order, so those results are compared for
equality (after the one rounding to bf16).  Random values: a sum of L products in fp32, each
partial sum off by at most 2^-22 of it (the tensor cores may truncate), plus half a bf16 step."""
import pytest
import torch

import deepgemm
from deepgemm import grouped_bf16_input_grad, grouped_bf16_weight_grad

pytestmark = pytest.mark.gpu
DEV = "cuda"


def layout(counts, align, tail=0):
    """m_indices of groups with `counts` rows, each padded to `align`, and `tail` rows behind them."""
    parts = []
    for g, c in enumerate(counts):
        parts.append(torch.full((c,), g))
        parts.append(torch.full((-c % align,), -1))
    return torch.cat(parts + [torch.full((tail,), -1)]).int()


def whole(gen, *shape, lim=4):
    return torch.randint(-lim, lim + 1, shape, generator=gen).bfloat16()


def packed(w):  # [G, N, K] -> [G, K/64, N, 64]
    g, n, k = w.shape
    return w.view(g, n, k // 64, 64).transpose(1, 2).contiguous()


def plain(w_packed):
    g, kb, n, _ = w_packed.shape
    return w_packed.transpose(1, 2).reshape(g, n, kb * 64)


def plain_dw(dy, x, m_indices, g):
    out = torch.zeros(g, dy.shape[1], x.shape[1], dtype=torch.float64)
    for e in range(g):
        r = (m_indices == e).nonzero()[:, 0]
        out[e] = dy[r].double().T @ x[r].double()
    return out


LAYOUTS = {
    "one row": ([1], 128, 0),
    "ragged": ([0, 1, 63, 64, 65, 0, 127, 128, 129, 200, 0], 128, 128),
    "256": ([300, 0, 16, 17], 256, 0),
    "one group": ([515], 128, 0),
    "none": ([0, 0, 0], 128, 256),
    "many": ([(7 * i) % 40 for i in range(300)], 128, 0),
}
SIZES = [(16, 64), (48, 192), (336, 576), (512, 256), (264 - 8, 1024)]


@pytest.mark.parametrize("name", LAYOUTS)
@pytest.mark.parametrize("n,k", SIZES)
@pytest.mark.parametrize("block_n", [128, 256, 512, 0])
def test_input_grad_is_exact_on_whole_numbers(name, n, k, block_n):
    counts, align, tail = LAYOUTS[name]
    if name == "many" and (n, k) != (48, 192):
        pytest.skip("one size is enough for 300 groups")
    mi = layout(counts, align, tail)
    gen = torch.Generator().manual_seed(n + k)
    m, g = mi.numel(), len(counts)
    dy, w = whole(gen, m, n), whole(gen, g, n, k, lim=2)
    dy[mi < 0] = float("nan")
    buf = torch.full((m, k), 3.0, dtype=torch.bfloat16, device=DEV)
    wd, md = packed(w).to(DEV), mi.to(DEV)
    grouped_bf16_input_grad(dy.to(DEV), wd, md, buf, block_n=block_n)
    want = torch.full((m, k), 3.0, dtype=torch.bfloat16)
    for e in range(g):
        r = mi == e
        want[r] = (dy[r].double() @ w[e].double()).bfloat16()
    assert torch.equal(buf.cpu(), want)
    deepgemm.check_device_status()
    if block_n == 0:
        fresh = grouped_bf16_input_grad(dy.to(DEV), wd, md).cpu()
        want[mi < 0] = 0
        assert torch.equal(fresh, want)


@pytest.mark.parametrize("name", LAYOUTS)
@pytest.mark.parametrize("n,k", SIZES)
@pytest.mark.parametrize("tile", [128, 256, 0, 1])
@pytest.mark.parametrize("dtype,add", [(torch.bfloat16, False), (torch.float32, False), (torch.float32, True)])
def test_weight_grad_is_exact_on_whole_numbers(name, n, k, tile, dtype, add):
    counts, align, tail = LAYOUTS[name]
    if name == "many" and (n, k) != (48, 192):
        pytest.skip("one size is enough for 300 groups")
    mi = layout(counts, align, tail)
    gen = torch.Generator().manual_seed(n * k)
    m, g = mi.numel(), len(counts)
    dy, x = whole(gen, m, n), whole(gen, m, k)
    dy[mi < 0], x[mi < 0] = float("nan"), float("inf")
    start = torch.randint(-9, 10, (g, k // 64, n, 64), generator=gen).to(dtype)
    out = start.to(DEV)
    got = grouped_bf16_weight_grad(dy.to(DEV), x.to(DEV), mi.to(DEV), g, out=out, accumulate=add, tile=tile)
    assert got is out
    want = packed(plain_dw(dy, x, mi, g))
    if add:
        want = want + start.double()
    assert torch.equal(out.cpu(), want.to(dtype))
    deepgemm.check_device_status()


@pytest.mark.parametrize("tile", [128, 256, 1])
def test_weight_grad_of_any_order_of_blocks_and_stray_rows(tile):
    """A group's blocks need not lie together, a block may hold rows that stand for nothing between
    others, and rows of another group than its first row's count for nothing."""
    g, n, k = 5, 208, 320
    gen = torch.Generator().manual_seed(3)
    mi = torch.cat([torch.full((128,), e) for e in (3, 0, 3, 4, 0, 0, 1)]).int()
    mi[torch.rand(mi.numel(), generator=gen) < 0.3] = -1
    mi[::128] = torch.tensor([3, 0, 3, 4, 0, 0, 1]).int()
    mi[3 * 128 + 64:4 * 128] = -1                    # half a block without a row
    mi[700:710] = 4                                  # strays in a block of group 0
    mi = mi[:-40]                                    # the last block is cut short
    m = mi.numel()
    dy, x = whole(gen, m, n), whole(gen, m, k)
    counted = mi.clone()
    counted[700:710] = -1
    dy[counted < 0], x[counted < 0] = float("inf"), float("nan")
    out = grouped_bf16_weight_grad(dy.to(DEV), x.to(DEV), mi.to(DEV), g, dtype=torch.float32, tile=tile)
    assert torch.equal(out.cpu().double(), packed(plain_dw(dy, x, counted, g)))
    assert bool((out[2] == 0).all())


def test_groups_out_of_range_are_reported():
    mi = torch.tensor([0] * 128 + [7] * 128 + [1] * 128).int()
    gen = torch.Generator().manual_seed(0)
    dy, x, w = whole(gen, 384, 64), whole(gen, 384, 128), whole(gen, 2, 64, 128)
    deepgemm.check_device_status()
    out = grouped_bf16_weight_grad(dy.to(DEV), x.to(DEV), mi.to(DEV), 2, dtype=torch.float32)
    with pytest.raises(RuntimeError, match="expert index was outside"):
        deepgemm.check_device_status()
    assert torch.equal(out.cpu().double(), packed(plain_dw(dy, x, mi, 2)))
    grouped_bf16_input_grad(dy.to(DEV), packed(w).to(DEV), mi.to(DEV))
    with pytest.raises(RuntimeError, match="expert index was outside"):
        deepgemm.check_device_status()


@pytest.mark.parametrize("counts,n,k,tile", [([700, 50, 1300], 1024, 768, 256), ([700, 50, 1300], 304, 320, 128), ([7000, 50, 1300], 304, 320, 0), ([5000], 128, 64, 0)])
def test_random_values(counts, n, k, tile):
    mi = layout(counts, 128)
    gen = torch.Generator().manual_seed(1)
    m, g = mi.numel(), len(counts)
    dy, x = torch.randn(m, n, generator=gen).bfloat16(), torch.randn(m, k, generator=gen).bfloat16()
    w = torch.randn(g, n, k, generator=gen).bfloat16()
    want, size = plain_dw(dy, x, mi, g), plain_dw(dy.abs(), x.abs(), mi, g)
    length = torch.tensor(counts).view(-1, 1, 1)
    f32 = plain(grouped_bf16_weight_grad(dy.to(DEV), x.to(DEV), mi.to(DEV), g, dtype=torch.float32, tile=tile).cpu()).double()
    bf = plain(grouped_bf16_weight_grad(dy.to(DEV), x.to(DEV), mi.to(DEV), g, tile=tile).cpu())
    assert bool(((f32 - want).abs() <= length * 2.0 ** -22 * size).all())
    # bf16 results are one sum, fp32 ones are made of segments of 896 rows: not the same sums rounded
    assert bool(((bf.double() - want).abs() <= want.abs() * 2.0 ** -8 * 1.01 + length * 2.0 ** -22 * size).all())
    dx = grouped_bf16_input_grad(dy.to(DEV), packed(w).to(DEV), mi.to(DEV)).cpu().double()
    for e in range(g):
        r = mi == e
        want, size = dy[r].double() @ w[e].double(), dy[r].double().abs() @ w[e].double().abs()
        assert bool(((dx[r] - want).abs() <= want.abs() * 2.0 ** -8 * 1.01 + n * 2.0 ** -22 * size).all())


def test_both_follow_the_differences_of_the_forward_product():
    """The product is linear in x and in W: its differences, exact on whole numbers, are the gradients'."""
    counts, n, k = [130, 0, 77], 96, 128
    mi = layout(counts, 128).to(DEV)
    gen = torch.Generator().manual_seed(2)
    m = mi.numel()
    w, vw = whole(gen, 3, n, k, lim=1), whole(gen, 3, n, k, lim=1)
    x, vx, dy = whole(gen, m, k, lim=1), whole(gen, m, k, lim=1), whole(gen, m, n, lim=1)
    keep = (mi >= 0).cpu()

    def f(w, x):  # |sums| <= 128 * 4: exact in bf16 up to 256, rounded by one beyond; kept below by the draw
        y = torch.zeros(m, n, dtype=torch.bfloat16, device=DEV)
        deepgemm.m_grouped_bf16_gemm_nt_contiguous(x.to(DEV), packed(w).to(DEV), y, mi)
        assert float(y.abs().max()) <= 256
        return y.cpu().double()[keep]

    dx = grouped_bf16_input_grad(dy.to(DEV), packed(w).to(DEV), mi).cpu().double()
    dw = plain(grouped_bf16_weight_grad(dy.to(DEV), x.to(DEV), mi, 3, dtype=torch.float32).cpu()).double()
    assert float(dx.abs().max()) <= 256
    y = f(w, x)
    assert float(((f(w, x + vx) - y) * dy.double()[keep]).sum()) == float((dx * vx.double())[keep].sum())
    assert float(((f(w + vw, x) - y) * dy.double()[keep]).sum()) == float((dw * vw.double()).sum())


def test_captured_and_replayed_and_on_another_stream():
    counts, n, k = [100, 300, 0, 20], 256, 512
    mi = layout(counts, 128).to(DEV)
    gen = torch.Generator().manual_seed(4)
    dy, x = whole(gen, mi.numel(), n).to(DEV), whole(gen, mi.numel(), k).to(DEV)
    w = packed(whole(gen, 4, n, k)).to(DEV)
    grouped_bf16_weight_grad(dy, x, mi, 4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dx = grouped_bf16_input_grad(dy, w, mi)
        dw = grouped_bf16_weight_grad(dy, x, mi, 4, dtype=torch.float32)
        grouped_bf16_weight_grad(dy, x, mi, 4, out=dw, accumulate=True)
    dy.copy_(whole(gen, mi.numel(), n))
    mi.copy_(layout([0, 200, 130, 1], 128)[:mi.numel()] if layout([0, 200, 130, 1], 128).numel() >= mi.numel() else mi)
    graph.replay()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        dx2 = grouped_bf16_input_grad(dy, w, mi)
        dw2 = grouped_bf16_weight_grad(dy, x, mi, 4, dtype=torch.float32)
    side.synchronize()
    assert torch.equal(dx, dx2) and torch.equal(dw, 2 * dw2)


def test_the_same_bits_every_time():
    mi = layout([500, 3, 900], 128).to(DEV)
    gen = torch.Generator().manual_seed(6)
    dy, x = torch.randn(mi.numel(), 512, generator=gen).bfloat16().to(DEV), torch.randn(mi.numel(), 768, generator=gen).bfloat16().to(DEV)
    start = torch.randn(3, 12, 512, 64, generator=gen).to(DEV)
    one = grouped_bf16_weight_grad(dy, x, mi, 3, out=start.clone(), accumulate=True)
    for _ in range(5):
        assert torch.equal(one, grouped_bf16_weight_grad(dy, x, mi, 3, out=start.clone(), accumulate=True))


def test_refusals():
    mi = layout([100], 128).to(DEV)
    dy, x = torch.zeros(128, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(128, 128, dtype=torch.bfloat16, device=DEV)
    w = torch.zeros(1, 2, 64, 64, dtype=torch.bfloat16, device=DEV)
    f32 = torch.zeros(1, 2, 64, 64, device=DEV)
    bad = [
        (RuntimeError, lambda: grouped_bf16_input_grad(dy.half(), w, mi)),
        (RuntimeError, lambda: grouped_bf16_input_grad(dy[:, :32], w, mi)),
        (RuntimeError, lambda: grouped_bf16_input_grad(x, w, mi)),
        (RuntimeError, lambda: grouped_bf16_input_grad(dy, w, mi.long())),
        (RuntimeError, lambda: grouped_bf16_input_grad(dy, w, mi[:64])),
        (RuntimeError, lambda: grouped_bf16_input_grad(dy, w, mi, out=dy)),
        (ValueError, lambda: grouped_bf16_input_grad(dy, w[0], mi)),
        (RuntimeError, lambda: grouped_bf16_input_grad(dy, w, mi, block_n=64)),
        (RuntimeError, lambda: grouped_bf16_weight_grad(dy, x[:64], mi, 1)),
        (RuntimeError, lambda: grouped_bf16_weight_grad(dy, x.float(), mi, 1)),
        (RuntimeError, lambda: grouped_bf16_weight_grad(dy, x[:, :96].contiguous(), mi, 1)),
        (RuntimeError, lambda: grouped_bf16_weight_grad(dy[:, :24].contiguous(), x, mi, 1)),
        (RuntimeError, lambda: grouped_bf16_weight_grad(dy, x, mi.cpu(), 1)),
        (RuntimeError, lambda: grouped_bf16_weight_grad(dy, x, mi, 1, dtype=torch.float16)),
        (RuntimeError, lambda: grouped_bf16_weight_grad(dy, x, mi, 2, out=f32)),
        (RuntimeError, lambda: grouped_bf16_weight_grad(dy, x, mi, 1, tile=64)),
        (ValueError, lambda: grouped_bf16_weight_grad(dy, x, mi, 1, accumulate=True)),
        (ValueError, lambda: grouped_bf16_weight_grad(dy, x, mi, 1, out=w, accumulate=True)),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()


@pytest.mark.parametrize("tile", [128, 256, 1])
def test_the_most_rows_and_groups(tile):
    """4096 blocks of 128 rows, 1024 groups in a scattered order: the largest table."""
    m, g, n, k = 4096 * 128, 1024, 16, 64
    gen = torch.Generator().manual_seed(8)
    of_block = torch.randint(0, g, (4096,), generator=gen)
    count = torch.randint(1, 129, (4096,), generator=gen)
    mi = torch.where(torch.arange(128)[None] < count[:, None], of_block[:, None], -1).reshape(-1).int()
    dy, x = whole(gen, m, n, lim=1), whole(gen, m, k, lim=1)
    out = grouped_bf16_weight_grad(dy.to(DEV), x.to(DEV), mi.to(DEV), g, dtype=torch.float32, tile=tile)
    deepgemm.check_device_status()
    d, xx, key = dy.float().to(DEV), x.float().to(DEV), mi.to(DEV)
    pairs = (d[:, :, None] * xx[:, None, :4]).view(m, -1)    # whole numbers: any order of the sums is exact
    want = torch.zeros(g + 1, pairs.shape[1], device=DEV).index_add_(0, torch.where(key < 0, g, key).long(), pairs)[:g].view(g, n, 4)
    assert torch.equal(out[:, 0, :, :4], want)


@pytest.mark.parametrize("tile", [128, 256, 1, 0])
def test_long_sums_keep_their_precision(tile):
    """The tensor cores accumulate in fp32 rounding towards zero: half a 2^-23 a step on average.  fp32
    gradients add up segments of at most 896 rows (56 steps), whatever the number of rows: 56 * 2^-24 =
    3.3e-6 in the relative 2-norm."""
    gen = torch.Generator().manual_seed(12)
    mi = layout([8192, 700, 3000], 128).to(DEV)
    dy, x = torch.randn(mi.numel(), 144, generator=gen).bfloat16().to(DEV), torch.randn(mi.numel(), 192, generator=gen).bfloat16().to(DEV)
    start = torch.randn(3, 3, 144, 64, generator=gen).to(DEV)
    got = grouped_bf16_weight_grad(dy, x, mi, 3, dtype=torch.float32, tile=tile)
    added = grouped_bf16_weight_grad(dy, x, mi, 3, out=start.clone(), accumulate=True, tile=tile)
    for g in range(3):
        r = mi == g
        want = (dy[r].double().T @ x[r].double()).view(144, 3, 64).transpose(0, 1)
        assert float((got[g].double() - want).norm() / want.norm()) <= 3.3e-6
        want = want + start[g].double()
        assert float((added[g].double() - want).norm() / want.norm()) <= 3.3e-6
    for _ in range(3):
        assert torch.equal(got, grouped_bf16_weight_grad(dy, x, mi, 3, dtype=torch.float32, tile=tile))
        assert torch.equal(added, grouped_bf16_weight_grad(dy, x, mi, 3, out=start.clone(), accumulate=True, tile=tile))


def test_offsets_beyond_32_bits():
    """Results of more than 2^31 elements: their last group and rows, where 32-bit offsets have wrapped."""
    gen = torch.Generator().manual_seed(5)
    g, n, k = 80, 4096, 7168
    dy, x = whole(gen, 128, n, lim=2).to(DEV), whole(gen, 128, k, lim=2).to(DEV)
    mi = torch.full((128,), g - 1, dtype=torch.int32, device=DEV)
    out = grouped_bf16_weight_grad(dy, x, mi, g)
    assert out.numel() > 2 ** 31
    assert torch.equal(out[-1], grouped_bf16_weight_grad(dy, x, torch.zeros_like(mi), 1)[0])
    assert not bool(out[:-1].any())
    del out
    m, n = 2432 * 128, 16
    dy = whole(gen, m, n, lim=2).to(DEV)
    w = packed(whole(gen, 2, n, k, lim=2)).to(DEV)
    mi = (torch.arange(m, device=DEV) >= m // 2).int()
    dx = grouped_bf16_input_grad(dy, w, mi)
    assert dx.numel() > 2 ** 31
    assert torch.equal(dx[-256:], grouped_bf16_input_grad(dy[-256:].contiguous(), w, mi[-256:].contiguous()))
