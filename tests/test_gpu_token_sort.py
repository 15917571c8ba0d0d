"""Tokens sorted by expert and back, with weights, and their gradients, against plain 64-bit forms.

Tolerances.  Sorting copies: equality.  A sum of k products in fp32, rounded once to a type with
relative half step e: |err| <= e |v| + k 2^-24 sum|terms| + the type's smallest step.  A product of
H terms summed in fp32: H 2^-24 sum|terms|."""
import pytest
import torch

import deepgemm
from deepgemm import TokenPlan, sort_capacity, sort_tokens, sort_tokens_grad, unsort_tokens, unsort_tokens_grad

pytestmark = pytest.mark.gpu
DEV = "cuda"
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}


def routing(t, k, e, seed, gone=0.0):
    gen = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(e, generator=gen)[:k] for _ in range(t)]) if t else torch.empty(0, k, dtype=torch.long)
    ids = torch.where(torch.rand(t, k, generator=gen) < gone, -1, ids)
    return ids, gen


def plain_plan(ids, e, align):
    t, k = ids.shape
    cap = sort_capacity(t * k, e, align)
    flat = ids.reshape(-1).tolist()
    counts = [sum(1 for v in flat if v == x) for x in range(e)] if e <= 64 else torch.bincount(
        torch.tensor([v for v in flat if 0 <= v < e] + [e]), minlength=e + 1)[:e].tolist()
    offsets, at = [], 0
    for c in counts:
        offsets.append(at)
        at += -(-c // align) * align
    nxt = list(offsets)
    dest, m_indices = [], [-1] * cap
    for v in flat:
        if 0 <= v < e:
            dest.append(nxt[v])
            m_indices[nxt[v]] = v
            nxt[v] += 1
        else:
            dest.append(-1)
    i32 = dict(dtype=torch.int32)
    return (torch.tensor(dest, **i32).view(t, k), torch.tensor(m_indices, **i32), torch.tensor(counts, **i32),
            torch.tensor(offsets, **i32), torch.tensor([at], **i32))


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


SHAPES = [  # tokens, top_k, experts, hidden, align, dtype, gone
    (1, 8, 256, 7168, 1, torch.bfloat16, 0.0),
    (1, 1, 1, 1, 1, torch.bfloat16, 0.0),
    (0, 2, 4, 64, 128, torch.bfloat16, 0.0),
    (3, 3, 4, 33, 16, torch.float16, 0.3),
    (67, 8, 256, 520, 1, torch.float16, 0.3),
    (129, 4, 32, 1000, 128, torch.bfloat16, 0.0),
    (513, 2, 3, 70, 256, torch.float32, 0.2),
    (1000, 8, 1024, 264, 1, torch.bfloat16, 0.0),
    (5, 2, 7, 2049, 128, torch.float32, 1.0),          # no pair has a row
    (9000, 8, 64, 24, 128, torch.bfloat16, 0.1),       # above 65536 pairs
    (70000, 1, 2, 8, 16, torch.float16, 0.0),
]


@pytest.mark.parametrize("t,k,e,h,align,dtype,gone", SHAPES)
@pytest.mark.parametrize("wide", [False, True])
def test_sort_places_every_pair(t, k, e, h, align, dtype, gone, wide):
    ids, gen = routing(t, k, e, t + e, gone)
    x = torch.randn(t, h + (3 if wide else 0), generator=gen).to(dtype)
    xd = x.to(DEV)[:, :h] if wide else x.to(DEV)
    x = x[:, :h]
    rows, plan = sort_tokens(xd, ids.to(DEV, torch.int64 if wide else torch.int32), e, align=align)
    want = plain_plan(ids, e, align)
    for got, w, name in zip(plan, want, TokenPlan._fields):
        assert got.dtype == torch.int32 and torch.equal(got.cpu(), w), name
    expect = torch.zeros(want[1].numel(), h, dtype=dtype)
    d = want[0].reshape(-1).long()
    token = torch.arange(t).repeat_interleave(k)
    expect[d[d >= 0]] = x[token[d >= 0]]
    assert torch.equal(rows.cpu(), expect)
    deepgemm.check_device_status()


def test_rows_of_a_given_buffer_stay_as_they_were():
    ids, gen = routing(37, 2, 5, 3, 0.2)
    x = torch.randn(37, 136, generator=gen).bfloat16().to(DEV)
    buf = torch.full((sort_capacity(74, 5, 128), 136), 7.0, dtype=torch.bfloat16, device=DEV)
    rows, plan = sort_tokens(x, ids.to(DEV), 5, out=buf)
    assert rows is buf and bool((rows[plan.m_indices < 0] == 7.0).all())
    fresh, _ = sort_tokens(x, ids.to(DEV), 5)
    used = plan.m_indices >= 0
    assert torch.equal(rows[used], fresh[used]) and bool((fresh[~used] == 0).all())


def test_the_same_expert_twice_and_ids_out_of_range():
    ids = torch.tensor([[1, 1, 1], [2, 9, -5], [1, 0, 2 ** 31 - 1]])
    x = torch.arange(3 * 16, dtype=torch.float32).view(3, 16).to(DEV)
    deepgemm.check_device_status()
    rows, plan = sort_tokens(x, ids.to(DEV), 3, align=1)
    with pytest.raises(RuntimeError, match="expert index was outside"):
        deepgemm.check_device_status()
    assert plan.dest.tolist() == [[1, 2, 3], [5, -1, -1], [4, 0, -1]]
    assert plan.counts.tolist() == [1, 4, 1] and plan.m_indices.tolist() == [0, 1, 1, 1, 1, 2, -1, -1, -1]
    rows64, plan64 = sort_tokens(x, torch.where(ids == 9, 2 ** 40, ids).to(DEV), 3, align=1)
    with pytest.raises(RuntimeError):
        deepgemm.check_device_status()
    assert torch.equal(rows, rows64) and torch.equal(plan.dest, plan64.dest)


@pytest.mark.parametrize("t,k,e,h,align,dtype,gone", SHAPES)
@pytest.mark.parametrize("weighted,wide", [(True, False), (True, True), (False, False)])
def test_back_and_gradients(t, k, e, h, align, dtype, gone, weighted, wide):
    ids, gen = routing(t, k, e, 2 * t + e, gone)
    plan_cpu = plain_plan(ids, e, align)
    plan = TokenPlan(*[v.to(DEV) for v in plan_cpu])
    cap = plan_cpu[1].numel()
    extra = 5 if wide else 0
    y = torch.randn(cap, h + extra, generator=gen).to(dtype)
    y[(plan_cpu[1] < 0)] = float("nan")                 # rows of no pair are never read
    dout = torch.randn(t, h + extra, generator=gen).to(dtype)
    w = torch.rand(t, k, generator=gen) if weighted else None
    if weighted:
        w[plan_cpu[0] < 0] = float("inf")               # nor is the weight of a pair without a row
    yd, dd = y.to(DEV)[:, :h], dout.to(DEV)[:, :h]
    y, dout = y[:, :h].double(), dout[:, :h].double()
    wd = w.to(DEV) if weighted else None
    out = unsort_tokens(yd, plan, wd)
    dy, dw = unsort_tokens_grad(dd, yd, plan, wd)
    dx = sort_tokens_grad(yd, plan)
    assert out.dtype == dy.dtype == dx.dtype == dtype and (dw is None) == (not weighted)

    dest = plan_cpu[0].long()
    here = dest >= 0
    ww = (w if weighted else torch.ones(t, k)).double()
    total, size = torch.zeros(t, h, dtype=torch.float64), torch.zeros(t, h, dtype=torch.float64)
    plainx, sizex = torch.zeros_like(total), torch.zeros_like(total)
    want_dy = torch.zeros(cap, h, dtype=torch.float64)
    want_dw, size_dw = torch.zeros(t, k, dtype=torch.float64), torch.zeros(t, k, dtype=torch.float64)
    for j in range(k):
        i = here[:, j].nonzero()[:, 0]
        r = dest[i, j]
        term = ww[i, j, None] * y[r]
        total[i] += term
        size[i] += term.abs()
        plainx[i] += y[r]
        sizex[i] += y[r].abs()
        want_dy[r] = ww[i, j, None] * dout[i]
        want_dw[i, j] = (dout[i] * y[r]).sum(1)
        size_dw[i, j] = (dout[i] * y[r]).abs().sum(1)
    e_half, tiny = half_step(dtype) * 1.01, TINY[dtype]
    assert bool(((out.cpu().double() - total).abs() <= e_half * total.abs() + k * 2.0 ** -24 * size * 1.01 + tiny).all())
    assert bool(((dx.cpu().double() - plainx).abs() <= e_half * plainx.abs() + k * 2.0 ** -24 * sizex * 1.01 + tiny).all())
    assert bool(((dy.cpu().double() - want_dy).abs() <= (e_half + 2.0 ** -23) * want_dy.abs() + tiny).all())
    if weighted:
        assert bool(((dw.cpu().double() - want_dw).abs() <= h * 2.0 ** -24 * size_dw * 1.01 + 1e-37).all())


def test_autograd_follows_the_differences():
    """There and back is linear in the tokens and in the weights: the gradient is the difference itself."""
    ids, gen = routing(19, 3, 6, 1, 0.2)
    x = torch.randn(19, 40, generator=gen).to(DEV).requires_grad_()
    w = torch.rand(19, 3, generator=gen).to(DEV).requires_grad_()
    g = torch.randn(19, 40, generator=gen).to(DEV)
    scale = torch.rand(40, generator=gen).to(DEV).requires_grad_()

    def f(x, w, scale):
        rows, plan = sort_tokens(x, ids.to(DEV), 6, align=16)
        return unsort_tokens(rows * scale, plan, w)

    out = f(x, w, scale)
    dx, dw, ds = torch.autograd.grad(out, (x, w, scale), g)
    with torch.no_grad():
        for at, grad in ((0, dx), (1, dw), (2, ds)):
            v = torch.randn((x, w, scale)[at].shape, generator=gen).to(DEV)
            args = [x, w, scale]
            args[at] = args[at] + v
            diff = ((f(*args) - out).double() * g.double()).sum()
            slope = (grad.double() * v.double()).sum()
            # 57 terms of 40 columns, each a difference of fp32 sums of up to three products
            assert abs(float(diff - slope)) <= 40 * 57 * 2.0 ** -22 * 4
    # a gradient that autograd hands over expanded
    f(x, w, scale).sum().backward()
    assert torch.allclose(x.grad, torch.autograd.grad(f(x, w, scale), x, torch.ones_like(g))[0])


def test_captured_and_replayed_with_other_inputs():
    ids, gen = routing(50, 4, 9, 8)
    x = torch.randn(50, 256, generator=gen).bfloat16().to(DEV)
    w = torch.rand(50, 4, generator=gen).to(DEV)
    ids_d = ids.to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sort_tokens(x, ids_d, 9)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rows, plan = sort_tokens(x, ids_d, 9)
        out = unsort_tokens(rows, plan, w)
        dy, dw = unsort_tokens_grad(x, rows, plan, w)
    for seed in (1, 2):
        ids2, gen2 = routing(50, 4, 9, seed)
        ids_d.copy_(ids2.to(DEV))
        x.copy_(torch.randn(50, 256, generator=gen2).bfloat16())
        graph.replay()
        rows2, plan2 = sort_tokens(x, ids_d, 9)
        assert torch.equal(rows, rows2) and all(torch.equal(a, b) for a, b in zip(plan, plan2))
        assert torch.equal(out, unsort_tokens(rows2, plan2, w))
        dy2, dw2 = unsort_tokens_grad(x, rows2, plan2, w)
        assert torch.equal(dy, dy2) and torch.equal(dw, dw2)


def test_offsets_beyond_32_bits():
    """2.3e9 elements of sorted rows: the last rows are where 32-bit element numbers have wrapped."""
    t, h = 20000, 7168
    ids = torch.arange(16, device=DEV, dtype=torch.int32).expand(t, 16).contiguous()
    x = torch.randn(t, h, device=DEV, dtype=torch.bfloat16)
    rows, plan = sort_tokens(x, ids, 16, align=1)
    assert rows.numel() > 2 ** 31
    assert torch.equal(rows[15 * t:], x) and torch.equal(rows[14 * t:15 * t], x)
    out = unsort_tokens(rows, plan, torch.full((t, 16), 2.0 ** -4, device=DEV))
    assert torch.equal(out, x)                          # 16 equal terms: every partial sum is exact
    dy, dw = unsort_tokens_grad(x, rows, plan, torch.ones(t, 16, device=DEV))
    assert torch.equal(dy[15 * t:], x) and torch.equal(dw[:, 15], dw[:, 0])
