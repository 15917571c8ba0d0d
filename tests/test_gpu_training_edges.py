"""Edges of the training operators on a GPU.  Whole numbers make every fp32 sum exact in any order, so
results on them are compared for equality after the one rounding."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

import deepgemm
from deepgemm import (_cabi, checkpoint_rows, clear_padding_rows, expert_mlp_bf16, grouped_bf16_input_grad, grouped_bf16_weight_grad,
                      grouped_grad, moe_forward_bf16, restore_rows, silu_mul, silu_mul_checkpoint, silu_mul_checkpoint_grad, sort_capacity,
                      sort_tokens, token_sort, unsort_tokens, unsort_tokens_grad)

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


@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_the_largest_values_stay_finite_in_the_backward_pass(dtype, kind):
    """A value beside the largest of its type may be held by a code beyond it (255 / 256 of a power of two);
    it counts as that largest value, so what is finite going forward is finite coming back."""
    top = torch.finfo(dtype).max
    x = torch.zeros(6, 2, 256, dtype=torch.float64)
    for r, (g, u) in enumerate(((top, 1.0), (1.0, top), (top, -1.0), (-1.0, top), (-top, 1.0), (top, 0.5))):
        x[r, 0, 130], x[r, 1, 130] = g, u
    x = x.view(6, 512).to(dtype).to(DEV)
    act, kept = silu_mul_checkpoint(x, kind=kind)
    dx, again = silu_mul_checkpoint_grad(kept, torch.ones(6, 256, dtype=dtype, device=DEV))
    assert bool(act.isfinite().all()) and bool(dx.isfinite().all()) and bool(again.isfinite().all())
    # within what eight bits hold of the two factors, 2^-4 each
    act, again = act.double(), again.double()
    assert bool(((again - act).abs() <= act.abs() * (2.0 ** -4 + 2.0 ** -4 + 2.0 ** -8)).all())


def unnamed_blocks(groups):
    """Blocks of 128 rows whose first entry names no group, with entries that do behind it."""
    mi = torch.full((7 * 128 + 40,), -1, dtype=torch.int32)
    for b, (first, others) in enumerate(((0, 0), (-1, 1), (1, 1), (groups, 0), (0, 0), (-1, 0), (2, 2), (-1, 1))):
        mi[b * 128 + 1:b * 128 + 100], mi[b * 128] = others, first
    named = ((mi[::128] >= 0) & (mi[::128] < groups)).repeat_interleave(128)[:mi.numel()]
    return mi, named & (mi >= 0)


def poison(*like):
    """Leaves NaN in the blocks that the allocator hands out next."""
    held = [torch.full(shape, float("nan"), dtype=dtype, device=DEV) for shape, dtype in like for _ in range(6)]
    del held


@pytest.mark.parametrize("block_n", [128, 256, 512, 0])
def test_input_grad_writes_every_row_of_its_own_result(block_n):
    gen = torch.Generator().manual_seed(1)
    g, n, k = 3, 96, 512
    mi, written = unnamed_blocks(g)
    dy, w = whole(gen, mi.numel(), n), whole(gen, g, n, k, lim=2)
    dyd, wd, md = dy.to(DEV), packed(w).to(DEV), mi.to(DEV)
    deepgemm.check_device_status()
    poison(((mi.numel(), k), BF))
    got = grouped_bf16_input_grad(dyd, wd, md, block_n=block_n).cpu()
    with pytest.raises(RuntimeError, match="expert index was outside"):
        deepgemm.check_device_status()
    want = torch.zeros(mi.numel(), k, dtype=BF)
    for e in range(g):
        r = written & (mi == e)
        want[r] = (dy[r].double() @ w[e].double()).bfloat16()
    assert torch.equal(got, want)
    # in a buffer of the caller's the same rows are left as they are
    buf = torch.full((mi.numel(), k), 3.0, dtype=BF, device=DEV)
    grouped_bf16_input_grad(dyd, wd, md, buf, block_n=block_n)
    want[~written] = 3.0
    assert torch.equal(buf.cpu(), want)
    with pytest.raises(RuntimeError):
        deepgemm.check_device_status()


def test_the_expert_part_writes_every_row_of_its_results():
    gen = torch.Generator().manual_seed(2)
    mi, written = unnamed_blocks(3)
    md, wd = mi.to(DEV), written.to(DEV)
    rows, g = torch.randn(mi.numel(), 128, generator=gen).bfloat16().to(DEV), torch.randn(mi.numel(), 128, generator=gen).bfloat16().to(DEV)
    w13, w2 = (torch.randn(3, 2, 256, 64, generator=gen) / 11).bfloat16().to(DEV), (torch.randn(3, 2, 128, 64, generator=gen) / 11).bfloat16().to(DEV)
    clean = torch.where(wd, md, -1)                  # the same, said in the entries themselves
    clean[::128] = torch.where(wd[::128], md[::128], -1)

    def run(m_indices):
        leaves = [t.clone().requires_grad_() for t in (rows, w13, w2)]
        poison((rows.shape, BF), ((mi.numel(), 256), BF), ((mi.numel(), 128), BF))
        y = expert_mlp_bf16(leaves[0], m_indices, *leaves[1:])
        poison((rows.shape, BF), ((mi.numel(), 256), BF), ((mi.numel(), 128), BF))
        return [y.detach(), *torch.autograd.grad(y, leaves, g)]

    want = run(clean)
    deepgemm.check_device_status()
    got = run(md)
    with pytest.raises(RuntimeError, match="expert index was outside"):
        deepgemm.check_device_status()
    assert bool((got[0][~wd] == 0).all()) and bool((got[1][~wd] == 0).all())
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_forward_mode_is_refused_and_not_passed_by():
    x = torch.randn(9, 64, device=DEV)
    ids = torch.randint(0, 3, (9, 2), device=DEV)
    rows, plan = sort_tokens(x, ids, 3)
    w = torch.rand(9, 2, device=DEV)
    with fwad.dual_level():
        dual = lambda t: fwad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                for call in (lambda: sort_tokens(dual(x), ids, 3), lambda: sort_tokens(dual(x), ids, 3, out=rows.clone()),
                             lambda: unsort_tokens(dual(rows), plan, w), lambda: unsort_tokens(rows, plan, dual(w)),
                             lambda: unsort_tokens(rows, plan, dual(w), out=x.clone()), lambda: silu_mul(dual(x))):
                    with pytest.raises((RuntimeError, NotImplementedError, ValueError), match="jvp|forward|out cannot be given"):
                        call()
        # tensors without a tangent are not concerned
        assert torch.equal(sort_tokens(x, ids, 3)[0], rows)
        assert unsort_tokens(rows, plan, w).shape == x.shape


@pytest.mark.parametrize("native", [True, False])
def test_the_arrays_of_a_plan_are_apart(native, monkeypatch):
    if not native:
        monkeypatch.setattr(token_sort, "_glue", None)
    x = torch.randn(20, 64, device=DEV).requires_grad_()
    ids = torch.randint(-1, 3, (20, 2), device=DEV)
    w = torch.rand(20, 2, device=DEV).requires_grad_()
    g = torch.randn(20, 64, device=DEV)
    rows, plan = sort_tokens(x, ids, 3)
    want = torch.autograd.grad(unsort_tokens(rows, plan, w), (x, w), g)
    rows, plan = sort_tokens(x, ids, 3)
    out = unsort_tokens(rows, plan, w)
    dest, m_indices = plan.dest.clone(), plan.m_indices.clone()
    plan.counts.zero_()
    plan.offsets.fill_(-5)
    plan.m_total.fill_(7)
    for a, b in zip(torch.autograd.grad(out, (x, w), g), want):
        assert torch.equal(a, b)
    assert torch.equal(plan.dest, dest) and torch.equal(plan.m_indices, m_indices)
    for t in plan:
        assert t.is_contiguous() and t.data_ptr() % 16 == 0


@pytest.mark.parametrize("weighted", [True, False])
def test_the_sorted_rows_are_kept_for_the_weights_alone(weighted):
    """Only the gradient of the weights reads the rows: without it they can go."""
    x = torch.randn(512, 1024, device=DEV)
    ids = torch.randint(0, 4, (512, 2), device=DEV)
    rows, plan = sort_tokens(x, ids, 4)
    leaf = rows.clone().requires_grad_()
    w = torch.rand(512, 2, device=DEV) if weighted else None
    g = torch.randn_like(x)
    want = unsort_tokens_grad(g, rows, plan, w)[0]
    del rows
    y = leaf * 2
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    out = unsort_tokens(y, plan, w)
    size = y.numel() * y.element_size()
    del y
    assert torch.cuda.memory_allocated() <= before + out.numel() * 4 - size + 4096
    assert torch.equal(torch.autograd.grad(out, leaf, g)[0], want * 2)


@pytest.mark.parametrize("native", [True, False])
def test_the_gradient_of_the_rows_without_the_rows(native, monkeypatch):
    if not native:
        monkeypatch.setattr(token_sort, "_glue", None)
    x = torch.randn(30, 96, device=DEV).bfloat16()
    ids = torch.randint(-1, 4, (30, 3), device=DEV)
    w = torch.rand(30, 3, device=DEV)
    rows, plan = sort_tokens(x, ids, 4, align=16)
    for weights in (w, None):
        want, _ = unsort_tokens_grad(x, rows, plan, weights)
        got, none = unsort_tokens_grad(x, None, plan, weights, need_dweights=False)
        assert none is None and torch.equal(got, want)
    for call in (lambda: unsort_tokens_grad(x, None, plan, w), lambda: unsort_tokens_grad(x[:7], None, plan, w, need_dweights=False),
                 lambda: unsort_tokens_grad(x, None, plan, w[:7], need_dweights=False)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("t,k", [(16384, 1), (16385, 1), (4096, 4), (5462, 3), (2048, 8), (2049, 8)])
@pytest.mark.parametrize("wide", [False, True])
def test_sort_on_both_sides_of_counting_ahead(t, k, wide):
    """Up to 16384 pairs every block counts them all, beyond that two launches count ahead."""
    gen = torch.Generator().manual_seed(t)
    e, h, align = 40, 16, 128
    ids = torch.randint(-1, e, (t, k), generator=gen)
    x = torch.randn(t, h, generator=gen).bfloat16().to(DEV)
    before = _cabi.query(_cabi.QUERY_LAUNCH_COUNT)
    rows, plan = sort_tokens(x, ids.to(DEV) if wide else ids.int().to(DEV), e, align=align)
    assert _cabi.query(_cabi.QUERY_LAUNCH_COUNT) - before == (1 if t * k <= 16384 else 3)
    flat = ids.reshape(-1)
    counts = torch.bincount(flat[flat >= 0], minlength=e)
    blocks = (counts + align - 1) // align * align
    offsets = blocks.cumsum(0) - blocks
    order = torch.sort(torch.where(flat < 0, e, flat), stable=True).indices[:int(counts.sum())]
    key = flat[order]
    dest = torch.full_like(flat, -1)
    dest[order] = offsets[key] + torch.arange(order.numel()) - (counts.cumsum(0) - counts)[key]
    m_indices = torch.full((sort_capacity(t * k, e, align),), -1)
    m_indices[dest[order]] = key
    assert torch.equal(plan.dest.cpu().long(), dest.view(t, k)) and torch.equal(plan.m_indices.cpu().long(), m_indices)
    assert torch.equal(plan.counts.cpu().long(), counts) and torch.equal(plan.offsets.cpu().long(), offsets)
    assert plan.m_total.item() == int(blocks.sum())
    want = torch.zeros(m_indices.numel(), h, dtype=BF, device=DEV)
    want[dest[order].to(DEV)] = x[(order // k).to(DEV)]
    assert torch.equal(rows, want)


@pytest.mark.parametrize("block_n", [128, 256, 512, 0])
@pytest.mark.parametrize("last", [1, 40, 64, 100, 128])
@pytest.mark.parametrize("n,k", [(16, 64), (336, 576), (256, 768)])
def test_input_grad_of_any_number_of_rows(block_n, last, n, k):
    """The last block cut short, in a result of its own (padding cleared) and in a given one."""
    gen = torch.Generator().manual_seed(last)
    counts = [130, 0, 128, 257, last]
    m, g = 6 * 128 + last, len(counts)
    mi = torch.cat([torch.cat([torch.full((c,), e), torch.full((-c % 128,), -1)]) for e, c in enumerate(counts)]).int()[:m]
    if last > 40:
        mi[-7:] = -1
    dy, w = whole(gen, m, n), whole(gen, g, n, k, lim=2)
    dy[mi < 0] = float("nan")
    want = torch.zeros(m, k, dtype=BF)
    for e in range(g):
        r = mi == e
        want[r] = (dy[r].double() @ w[e].double()).bfloat16()
    dyd, wd, md = dy.to(DEV), packed(w).to(DEV), mi.to(DEV)
    poison(((m, k), BF))
    assert torch.equal(grouped_bf16_input_grad(dyd, wd, md, block_n=block_n).cpu(), want)
    room = torch.full((m + 128, k), 3.0, dtype=BF, device=DEV)
    grouped_bf16_input_grad(dyd, wd, md, room[:m], block_n=block_n)
    want[mi < 0] = 3.0
    assert torch.equal(room[:m].cpu(), want) and bool((room[m:] == 3.0).all())
    deepgemm.check_device_status()


@pytest.mark.parametrize("t,gone", [(0, False), (50, True)])
@pytest.mark.parametrize("kind", ["fp8", "int8"])
def test_a_layer_without_a_row(t, gone, kind):
    """No tokens, or every pair at experts that live elsewhere: zeros, and gradients of zeros."""
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(t, 128, generator=gen).bfloat16().to(DEV)
    ids = torch.full((t, 2), -1, device=DEV) if gone else torch.zeros(t, 2, dtype=torch.long, device=DEV)
    w = torch.rand(t, 2, generator=gen).to(DEV)
    w13, w2 = torch.randn(3, 2, 256, 64, generator=gen).bfloat16().to(DEV), torch.randn(3, 2, 192, 64, generator=gen).bfloat16().to(DEV)
    leaves = [v.requires_grad_() for v in (x, w, w13, w2)]
    poison((w13.shape, BF), (w2.shape, BF), ((t, 192), BF), ((t, 128), BF))
    out = moe_forward_bf16(leaves[0], ids, *leaves[1:], checkpoint=kind)
    assert out.shape == (t, 192) and not bool(out.any())
    for v, d in zip(leaves, torch.autograd.grad(out, leaves, torch.ones_like(out))):
        assert d.shape == v.shape and d.dtype == v.dtype and bool((d == 0).all())
    with torch.no_grad():
        assert torch.equal(moe_forward_bf16(leaves[0], ids, *leaves[1:], checkpoint=kind), out)
    deepgemm.check_device_status()


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("m,h", [(0, 8), (1, 1), (130, 264), (300, 77), (5000, 16), (64, 2048)])
def test_clear_padding_rows_clears_those_and_no_others(dtype, m, h):
    gen = torch.Generator().manual_seed(m + h)
    rows = torch.randn(m, h, generator=gen).to(dtype)
    mi = torch.randint(-2, 3, (m,), generator=gen).int()
    room = torch.full((m + 2, h), 5.0, dtype=dtype, device=DEV)
    room[1:m + 1] = rows.to(DEV)
    room[1:m + 1][(mi < 0).to(DEV)] = float("nan")
    mid = room[1:m + 1]
    assert clear_padding_rows(mid, mi.to(DEV)) is mid
    rows[mi < 0] = 0
    assert torch.equal(mid.cpu(), rows) and bool((room[0] == 5.0).all()) and bool((room[-1] == 5.0).all())


@pytest.mark.parametrize("block_n,tile", [(128, 128), (512, 256)])
def test_entries_beside_the_first_of_a_block(block_n, tile):
    """What the documentation says of a block that holds entries of two groups: the product and the gradient
    of the rows take all of them with the first one's weights, the gradient of the weights leaves the
    others out."""
    gen = torch.Generator().manual_seed(4)
    g, n, k = 3, 128, 256
    mi = torch.full((256,), 1, dtype=torch.int32)
    mi[30:40], mi[200:256] = 2, -1
    dy, x, w = whole(gen, 256, n), whole(gen, 256, k), whole(gen, g, n, k, lim=2)
    dyd, wd, md = dy.to(DEV), packed(w).to(DEV), mi.to(DEV)
    y = torch.zeros(256, n, dtype=BF, device=DEV)
    deepgemm.m_grouped_bf16_gemm_nt_contiguous(x.to(DEV), wd, y, md)
    used = mi >= 0
    assert torch.equal(y.cpu()[used], (x.double() @ w[1].double().T).bfloat16()[used])
    dx = grouped_bf16_input_grad(dyd, wd, md, block_n=block_n).cpu()
    assert torch.equal(dx[used], (dy.double() @ w[1].double()).bfloat16()[used])
    dw = grouped_bf16_weight_grad(dyd, x.to(DEV), md, g, dtype=F32, tile=tile).cpu()
    one = mi == 1
    assert torch.equal(dw[1], packed((dy[one].double().T @ x[one].double())[None])[0].float())
    assert not bool(dw[0].any()) and not bool(dw[2].any())
    whole_blocks = grouped_bf16_weight_grad(dyd, x.to(DEV), md, g, dtype=F32, tile=tile, whole_blocks=True).cpu()
    assert torch.equal(whole_blocks[1], packed((dy[used].double().T @ x[used].double())[None])[0].float())
    assert not bool(whole_blocks[0].any()) and not bool(whole_blocks[2].any())


@pytest.mark.parametrize("native", [True, False])
def test_the_gradients_of_the_layer_are_those_of_its_result(native, monkeypatch):
    """Whatever the entries behind a block's first one name: the product takes the first's weights for all
    rows, and so do all three gradients."""
    if not native:
        monkeypatch.setattr(grouped_grad, "_glue", None)
    gen = torch.Generator().manual_seed(6)
    mi = torch.randint(-1, 3, (5 * 128 + 17,), generator=gen).int()
    mi[::128] = torch.tensor([2, 0, 2, 1, 1, 0]).int()
    rows, g = torch.randn(mi.numel(), 128, generator=gen).bfloat16().to(DEV), torch.randn(mi.numel(), 128, generator=gen).bfloat16().to(DEV)
    w13, w2 = (torch.randn(3, 2, 256, 64, generator=gen) / 11).bfloat16().to(DEV), (torch.randn(3, 2, 128, 64, generator=gen) / 11).bfloat16().to(DEV)
    first = mi[::128].repeat_interleave(128)[:mi.numel()]

    def run(m_indices):
        leaves = [t.clone().requires_grad_() for t in (rows, w13, w2)]
        y = expert_mlp_bf16(leaves[0], m_indices.to(DEV), *leaves[1:])
        return [y.detach(), *torch.autograd.grad(y, leaves, g)]

    for a, b in zip(run(mi), run(torch.where(mi < 0, mi, first))):
        assert torch.equal(a, b)
    deepgemm.check_device_status()


def test_results_that_lie_on_their_inputs_are_refused():
    x = torch.randn(256, 128, device=DEV).bfloat16()
    ids = torch.randint(0, 2, (128, 2), dtype=torch.int32, device=DEV)
    room = torch.randn(1024, 128, device=DEV).bfloat16()
    w = torch.rand(128, 2, device=DEV)
    rows, plan = sort_tokens(x[:128], ids, 2, align=1)
    mi = torch.zeros(256, dtype=torch.int32, device=DEV)
    square = torch.randn(1, 2, 128, 64, device=DEV).bfloat16()
    grad = torch.zeros(1, 2, 128, 64, dtype=BF, device=DEV)
    bad = [
        lambda: sort_tokens(room[100:228], ids, 2, align=1, out=room[:256]),
        lambda: unsort_tokens(room[:256], plan, w, out=room[255:383]),
        lambda: grouped_bf16_input_grad(x, square, mi, out=x),
        lambda: grouped_bf16_input_grad(room[:256], square, mi, out=room[255:511]),
        lambda: grouped_bf16_input_grad(x, room[:128].view(1, 2, 128, 64), mi, out=room[:256]),
        lambda: grouped_bf16_weight_grad(x, room[:256], mi, 1, out=room[:128].view(1, 2, 128, 64)),
        lambda: grouped_bf16_weight_grad(room[:256], x, mi, 1, out=room[200:328].view(1, 2, 128, 64)),
    ]
    before = room.clone()
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError), match="overlap"):
            call()
            print("accepted:", i)
    assert torch.equal(room, before)
    # neighbours in one buffer are not concerned
    assert torch.equal(sort_tokens(room[256:384], ids, 2, align=1, out=room[:256])[0], sort_tokens(room[256:384], ids, 2, align=1)[0])
    unsort_tokens(room[:256], plan, w, out=room[256:384])
    grouped_bf16_input_grad(room[:256], square, mi, out=room[256:512])
    grouped_bf16_weight_grad(room[:256], room[256:512], mi, 1, out=grad)
    deepgemm.check_device_status()


def test_where_codes_become_subnormal():
    """The bound on what e4m3 holds, on both sides of 2^-6 scales: 2^-4 of the value or 2^-10 scales,
    whichever is more.  Beside a block's 225 (scale 1) 7.5 / 512 is further off than 2^-4 of itself."""
    x = torch.zeros(3, 128, device=DEV)
    x[0, :2] = torch.tensor([225.0, 7.5 / 512])
    x[1] = torch.linspace(0, 2.0 ** -5, 128)
    x[1, 0] = 448.0
    x[2] = torch.exp2(torch.linspace(-16, 0, 128)) * 224.0
    c = checkpoint_rows(x)
    assert c.scale.flatten().tolist() == [1.0, 1.0, 0.5]
    off, v = (restore_rows(c).double() - x.double()).abs(), x.double().abs()
    assert float(off[0, 1]) > float(v[0, 1]) * 2.0 ** -4
    assert bool((off <= torch.maximum(v * 2.0 ** -4, c.scale.double() * 2.0 ** -10)).all())
