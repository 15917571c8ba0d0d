"""Activation checkpoints in 8 bits against plain 64-bit forms.

Tolerances.  e4m3 codes and scales are compared for equality (the scale is a power of two, so x / s
is exact); int8 values come back within (0.5 + 2^-16) scales (two fp32 roundings on at most 127
steps).  The activation and its gradients: q * s is rounded by 2^-24, which moves exp(-g) by
|g| 2^-24 of itself, as does the rounding of g log2(e) inside the hardware's exp, with log2(e) itself
a little off (16-bit results); exp, sum, quotient and products add at most 8 half steps of fp32.
So with s = the sigmoid every result is within (|g| + 8) 2^-24 (fp32) or (|g| + 8) 2^-23 (16-bit
types) of its terms, and is then rounded once, by half a step."""
import pytest
import torch

import deepgemm
from deepgemm import Checkpoint, checkpoint_rows, restore_rows, silu_mul, silu_mul_checkpoint, silu_mul_checkpoint_grad

pytestmark = pytest.mark.gpu
DEV = "cuda"
CODE = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def values(m, h, dtype, seed, top=4.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(m, h, generator=gen) * torch.exp2(torch.randint(-3, 4, (m, 1), generator=gen).float())
    return x.clamp(-top * 8, top * 8).to(dtype), gen


def plain_checkpoint(x, kind):
    """codes (float64) and scales (float64), block by block."""
    m, h = x.shape
    n = -(-h // 128)
    q, s = torch.zeros(m, h, dtype=torch.float64), torch.ones(m, n, dtype=torch.float64)
    for b in range(n):
        v = x[:, 128 * b:128 * b + 128].double()
        top = v.abs().amax(1)
        if kind == "fp8":
            mant, exp = torch.frexp(top)                       # top = mant 2^exp, 448 = 0.875 * 2^9
            step = torch.exp2((exp - 9 + (mant > 0.875)).clamp_min(-126).double())
        else:
            step = (top.float() / 127).clamp_min(2.0 ** -126).double()
        step = torch.where(top == 0, 1.0, step)
        step = torch.where(top.isfinite(), step, float("nan"))
        s[:, b] = step
        r = v / step[:, None]
        q[:, 128 * b:128 * b + 128] = r.float().to(torch.float8_e4m3fn).double() if kind == "fp8" else r
    return q, s


ROWS = [(1, 1, BF), (1, 128, BF), (3, 129, HF), (37, 1000, BF), (130, 264, F32), (64, 7168, BF), (257, 77, HF), (0, 64, BF)]


@pytest.mark.parametrize("m,h,dtype", ROWS)
@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("wide", [False, True])
def test_rows_there_and_back(m, h, dtype, kind, wide):
    x, _ = values(m, h + (3 if wide else 0), dtype, m + h)
    c = checkpoint_rows(x.to(DEV)[:, :h], kind=kind)
    x = x[:, :h]
    assert c.q.dtype == CODE[kind] and c.dtype == dtype
    q, s = plain_checkpoint(x, kind)
    assert torch.equal(c.scale.cpu().double(), s)
    wide_s = s.repeat_interleave(128, 1)[:, :h]
    if kind == "fp8":
        assert torch.equal(c.q.cpu().double(), q)
    else:
        assert bool(((c.q.cpu().double() * wide_s - x.double()).abs() <= (0.5 + 2.0 ** -16) * wide_s).all())
    held = c.q.cpu().double() * wide_s
    back = restore_rows(c)
    assert back.dtype == dtype
    half = torch.finfo(dtype).eps / 2
    tiny = {BF: 2.0 ** -133, HF: 2.0 ** -24, F32: 2.0 ** -149}[dtype]
    assert bool(((back.cpu().double() - held).abs() <= (half + 2.0 ** -24) * held.abs() + tiny).all())
    if kind == "fp8" and dtype != HF:
        assert torch.equal(back.cpu().double(), held)


@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_zeros_tiny_huge_and_nonfinite_blocks(kind, dtype):
    top = torch.finfo(dtype).max
    x = torch.zeros(9, 256, dtype=torch.float64)
    x[1] = torch.linspace(-1, 1, 256) * top
    x[2, 5] = torch.finfo(dtype).smallest_normal / 4           # a subnormal alone
    x[3, 7], x[3, 200] = float("inf"), 1.0
    x[4, 130] = float("nan")
    x[5, :128] = 448.0
    x[6, :128] = 449.0 if dtype == F32 else 450.0 if dtype == BF else 448.5
    x[7] = torch.linspace(-3, 3, 256)
    x[8, 0] = -float("inf")
    x = x.to(dtype)
    c = checkpoint_rows(x.to(DEV), kind=kind)
    q, s = plain_checkpoint(x, kind)
    assert torch.equal(torch.nan_to_num(c.scale.cpu().double(), nan=-1.0), torch.nan_to_num(s, nan=-1.0))
    back = restore_rows(c).cpu().double()
    lost = torch.tensor([[(r, b) in ((3, 0), (4, 1), (8, 0)) for b in range(2)] for r in range(9)]).repeat_interleave(128, 1)
    assert bool(back[lost].isnan().all()) and bool(back[~lost].isfinite().all())
    step = s.repeat_interleave(128, 1)
    err = (back - x.double()).abs()
    half, tiny = torch.finfo(dtype).eps / 2, {BF: 2.0 ** -133, HF: 2.0 ** -24, F32: 2.0 ** -149}[dtype]
    if kind == "fp8":
        bound = torch.maximum(x.double().abs() * 2.0 ** -4, step * 2.0 ** -10)
    else:
        bound = step * (0.5 + 2.0 ** -16)
    bound = bound + half * x.double().abs() * 1.1 + tiny
    assert bool((err <= bound)[~lost].all())
    assert bool((back[0] == 0).all())


def plain_act(g, u):
    return g * torch.sigmoid(g) * u


def plain_grad(g, u, d):
    s = torch.sigmoid(g)
    return d * u * s * (1 + g * (1 - s)), d * g * s


ACTS = [(1, 1, BF), (1, 128, HF), (37, 1000, HF), (130, 264, F32), (100, 2048, BF), (257, 77, BF), (5, 130, F32), (0, 8, BF)]


@pytest.mark.parametrize("m,h,dtype", ACTS)
@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("masked,wide", [(False, False), (True, False), (True, True)])
def test_activation_forward_and_backward(m, h, dtype, kind, masked, wide):
    x, gen = values(m, 2 * h + (2 if wide else 0), dtype, m + h + masked)
    dact = torch.randn(m, h + (1 if wide else 0), generator=gen).to(dtype)
    mi = None
    keep = torch.ones(m, dtype=torch.bool)
    if masked:
        mi = torch.randint(0, 5, (m,), generator=gen).int()
        mi[torch.rand(m, generator=gen) < 0.4] = -1
        keep = mi >= 0
        x[~keep], dact[~keep] = float("nan"), float("inf")     # rows of no pair are not read
        mi = mi.to(DEV)
    act, c = silu_mul_checkpoint(x.to(DEV)[:, :2 * h], kind=kind, m_indices=mi)
    dx, again = silu_mul_checkpoint_grad(c, dact.to(DEV)[:, :h], m_indices=mi)
    assert act.dtype == dx.dtype == again.dtype == dtype
    x, dact = x[:, :2 * h], dact[:, :h]
    g, u = x[:, :h].double(), x[:, h:].double()
    half = torch.finfo(dtype).eps / 2
    tiny = {BF: 2.0 ** -132, HF: 2.0 ** -24, F32: 2.0 ** -126}[dtype]
    exact = (g.abs() + 8) * 2.0 ** (-23 if dtype != F32 else -24)
    want = plain_act(g, u)
    assert bool(((act.cpu().double() - want).abs() <= (half + exact) * want.abs() + tiny)[keep].all())
    assert bool((act.cpu()[~keep] == 0).all()) and bool((dx.cpu()[~keep] == 0).all()) and bool((again.cpu()[~keep] == 0).all())
    assert bool((c.q.cpu().float()[~keep] == 0).all())

    # the checkpoint is that of gate and of up
    n = -(-h // 128)
    q, s = c.q.cpu().double(), c.scale.cpu().double()
    for i, v in enumerate((x[:, :h], x[:, h:])):
        pq, ps = plain_checkpoint(v, kind)
        assert torch.equal(s[keep, n * i:n * i + n], ps[keep])
        if kind == "fp8":
            assert torch.equal(q[keep, h * i:h * i + h], pq[keep])
    held = q * torch.cat([s[:, :n].repeat_interleave(128, 1)[:, :h], s[:, n:].repeat_interleave(128, 1)[:, :h]], 1)
    g, u, d = held[:, :h], held[:, h:], dact.double()
    exact = (g.abs() + 8) * 2.0 ** (-23 if dtype != F32 else -24)
    dg, du = plain_grad(g, u, d)
    sig = torch.sigmoid(g)
    got = dx.cpu().double()
    size_g = (d * u * sig).abs() * (1 + g.abs())
    assert bool(((got[:, :h] - dg).abs() <= half * dg.abs() * 1.01 + exact * size_g + tiny)[keep].all())
    assert bool(((got[:, h:] - du).abs() <= (half * 1.01 + exact) * du.abs() + tiny)[keep].all())
    want = plain_act(g, u)
    assert bool(((again.cpu().double() - want).abs() <= (half * 1.01 + exact) * want.abs() + tiny)[keep].all())
    # without the activation: the same gradients
    dx2, none = silu_mul_checkpoint_grad(c, dact.to(DEV), m_indices=mi, need_act=False)
    assert none is None and torch.equal(dx2, dx)


def test_gradient_follows_the_differences():
    """Values that e4m3 holds exactly, so that the checkpoint is the input: the gradient against
    central differences of the fp32 forward pass.  Step 2^-7: |third derivative| of silu is below 1,
    which leaves 2^-14 / 6 |u d|; the forward pass is within 2^-21, over a step of 2^-6."""
    gen = torch.Generator().manual_seed(5)
    x = (torch.randint(-16, 17, (40, 256), generator=gen).float() / 8).to(DEV).requires_grad_()
    d = torch.randn(40, 128, generator=gen).to(DEV)
    grad, = torch.autograd.grad(silu_mul(x), x, d)
    eps = 2.0 ** -7
    with torch.no_grad():
        for half in (0, 1):
            step = torch.zeros_like(x)
            step[:, 128 * half:128 * half + 128] = eps
            slope = (silu_mul(x + step).double() - silu_mul(x - step).double()) / (2 * eps) * d.double()
            size = d.double().abs() * (2.0 ** -14 / 6 * 2 + 2.0 ** -21 * 4 / eps + 2.0 ** -18)
            assert bool(((grad[:, 128 * half:128 * half + 128].double() - slope).abs() <= size).all())


def test_memory_kept_is_a_byte_for_each_value():
    x = torch.randn(512, 2 * 2048, device=DEV, dtype=BF).requires_grad_()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    out = silu_mul(x)
    kept = torch.cuda.memory_allocated() - before - out.numel() * 2
    assert kept <= x.numel() * (1 + 4 / 128) + 4096
    out.backward(torch.ones_like(out))
    assert x.grad.shape == x.shape


def test_captured_and_replayed_with_other_inputs():
    x, _ = values(70, 512, BF, 1)
    x, d = x.to(DEV), torch.randn(70, 256, device=DEV).bfloat16()
    silu_mul_checkpoint(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        act, c = silu_mul_checkpoint(x)
        dx, again = silu_mul_checkpoint_grad(c, d)
        back = restore_rows(checkpoint_rows(x, kind="int8"))
    x.copy_(values(70, 512, BF, 2)[0])
    graph.replay()
    act2, c2 = silu_mul_checkpoint(x)
    dx2, again2 = silu_mul_checkpoint_grad(c2, d)
    for a, b in ((act, act2), (dx, dx2), (again, again2), (back, restore_rows(checkpoint_rows(x, kind="int8")))):
        assert torch.equal(a, b)


def test_offsets_beyond_32_bits():
    m, h = 160000, 7168
    x = torch.randn(m, 2 * h, device=DEV, dtype=BF)
    assert x.numel() > 2 ** 31
    act, c = silu_mul_checkpoint(x)
    dx, again = silu_mul_checkpoint_grad(c, act)
    tail, tc = silu_mul_checkpoint(x[-300:])
    dtail, atail = silu_mul_checkpoint_grad(tc, tail)
    assert torch.equal(act[-300:], tail) and torch.equal(dx[-300:], dtail) and torch.equal(again[-300:], atail)
    c = checkpoint_rows(x)
    assert torch.equal(restore_rows(c)[-300:], restore_rows(checkpoint_rows(x[-300:])))
