"""The training path of an MoE layer: the operators in a run, as a user runs them.

Reference: the same formulas in float64 on the CPU, with the gradient of the activation taken at the
values that the checkpoint holds (computed here from the definition) and bf16 rounding where the
layer stores bf16.  What remains is where a sum lies next to a rounding border: every stored value
is off by at most one rounding more or less.  A chain of at most six stored stages, each off by at
most 2^-8 of its size, gives a relative 2-norm below 6 * 2^-8; the bound is 2^-5."""
import pytest
import torch

import deepgemm
from deepgemm import _cabi, expert_mlp_bf16, moe_forward_bf16, sort_tokens, unsort_tokens

pytestmark = pytest.mark.gpu
DEV = "cuda"
BOUND = 2.0 ** -5


def packed(w):
    g, n, k = w.shape
    return w.view(g, n, k // 64, 64).transpose(1, 2).contiguous()


def plain(w):
    g, kb, n, _ = w.shape
    return w.transpose(1, 2).reshape(g, n, kb * 64)


def b16(x):
    return x.bfloat16().double()


def held(x, kind):
    """What an 8-bit checkpoint of x (float64) holds, in blocks of 128 columns."""
    out = torch.empty_like(x)
    for c in range(0, x.shape[1], 128):
        v = x[:, c:c + 128]
        top = v.abs().amax(1, keepdim=True)
        if kind == "fp8":
            m, e = torch.frexp(top)
            s = torch.where(top > 0, torch.exp2((e - 9 + (m > 0.875)).double()), 1.0)
            out[:, c:c + 128] = (v / s).float().to(torch.float8_e4m3fn).double() * s
        else:
            s = torch.where(top > 0, (top.float() / 127).double(), 1.0)
            out[:, c:c + 128] = (v / s).round() * s
    return out


def layer(hidden, ids, w, w13, w2, dout, kind):
    """out, dhidden, dw, dw13, dw2 in float64 (bf16 where the layer stores it)."""
    e, _, k = w13.shape
    out = torch.zeros(hidden.shape[0], w2.shape[1], dtype=torch.float64)
    dhidden, dw = torch.zeros_like(hidden), torch.zeros_like(w)
    dw13, dw2 = torch.zeros_like(w13), torch.zeros_like(w2)
    for x in range(e):
        t, j = (ids == x).nonzero(as_tuple=True)
        rows = hidden[t]
        h = b16(rows @ w13[x].T)
        g, u = h.chunk(2, 1)
        y = b16(b16(g * torch.sigmoid(g) * u) @ w2[x].T)
        out.index_add_(0, t, w[t, j, None] * y)
        dw[t, j] = (dout[t] * y).sum(1)
        dy = b16(w[t, j, None] * dout[t])
        dact = b16(dy @ w2[x])
        g, u = held(g, kind), held(u, kind)
        s = torch.sigmoid(g)
        dh = b16(torch.cat([dact * u * s * (1 + g * (1 - s)), dact * g * s], 1))
        dw2[x] = dy.T @ b16(g * s * u)
        dw13[x] = dh.T @ b16(held(rows, kind))
        dhidden.index_add_(0, t, b16(dh @ w13[x]))
    return out, dhidden, dw, dw13, dw2


def close(got, want, what):
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, what
    off = float((got - want).norm() / want.norm())
    assert off <= BOUND, f"{what}: relative difference {off:.2e}"


@pytest.mark.parametrize("t,k,e,hidden,inner,out,gone,kind", [
    (96, 2, 4, 128, 192, 128, 0.0, "fp8"),
    (1, 1, 1, 64, 64, 64, 0.0, "fp8"),
    (1, 4, 8, 256, 128, 80, 0.0, "int8"),
    (333, 3, 16, 320, 256, 320, 0.3, "int8"),
    (700, 2, 3, 512, 320, 512, 0.1, "fp8"),
])
def test_layer_and_all_its_gradients(t, k, e, hidden, inner, out, gone, kind):
    gen = torch.Generator().manual_seed(t + e)
    x = torch.randn(t, hidden, generator=gen).bfloat16()
    ids = torch.stack([torch.randperm(e, generator=gen)[:k] for _ in range(t)])
    ids = torch.where(torch.rand(t, k, generator=gen) < gone, -1, ids)
    w = torch.rand(t, k, generator=gen) + 0.1
    w13 = (torch.randn(e, 2 * inner, hidden, generator=gen) / hidden ** 0.5).bfloat16()
    w2 = (torch.randn(e, out, inner, generator=gen) / inner ** 0.5).bfloat16()
    dout = torch.randn(t, out, generator=gen).bfloat16()
    args = [x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_(), packed(w13).to(DEV).requires_grad_(), packed(w2).to(DEV).requires_grad_()]
    got = moe_forward_bf16(args[0], ids.to(DEV), *args[1:], checkpoint=kind)
    grads = torch.autograd.grad(got, args, dout.to(DEV))
    want = layer(x.double(), ids, w.double(), w13.double(), w2.double(), dout.double(), kind)
    close(got, want[0], "out")
    close(grads[0], want[1], "dhidden")
    close(grads[1], want[2], "dweights")
    close(plain(grads[2]), want[3], "dw13")
    close(plain(grads[3]), want[4], "dw2")
    for g, a in zip(grads, args):
        assert g.dtype == a.dtype and g.shape == a.shape
    # the same bits once more, and without a gradient
    again = moe_forward_bf16(args[0], ids.to(DEV), *args[1:], checkpoint=kind)
    assert torch.equal(got, again)
    for a, b in zip(grads, torch.autograd.grad(again, args, dout.to(DEV))):
        assert torch.equal(a, b)
    with torch.no_grad():
        assert torch.equal(got, moe_forward_bf16(args[0], ids.to(DEV), *args[1:], checkpoint=kind))
    deepgemm.check_device_status()


def test_only_some_gradients_are_wanted():
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(200, 128, generator=gen).bfloat16().to(DEV)
    ids = torch.randint(0, 4, (200, 2), generator=gen).to(DEV)
    w = torch.rand(200, 2, generator=gen).to(DEV)
    w13, w2 = (torch.randn(4, 2, 256, 64, generator=gen) / 11).bfloat16().to(DEV), (torch.randn(4, 2, 128, 64, generator=gen) / 11).bfloat16().to(DEV)
    g = torch.randn(200, 128, generator=gen).bfloat16().to(DEV)
    every = [t.clone().requires_grad_() for t in (x, w, w13, w2)]
    full = torch.autograd.grad(moe_forward_bf16(every[0], ids, *every[1:]), every, g)
    for i in range(4):
        some = [t.clone() for t in (x, w, w13, w2)]
        some[i].requires_grad_()
        one, = torch.autograd.grad(moe_forward_bf16(some[0], ids, *some[1:]), some[i], g)
        assert torch.equal(one, full[i])


def test_rows_of_no_pair_reach_nothing():
    """What lies in the padding, on the way in or in a gradient, changes no result."""
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(150, 128, generator=gen).bfloat16().to(DEV)
    ids = torch.randint(-1, 3, (150, 2), generator=gen).to(DEV)
    w13, w2 = (torch.randn(3, 2, 256, 64, generator=gen) / 11).bfloat16().to(DEV), (torch.randn(3, 2, 128, 64, generator=gen) / 11).bfloat16().to(DEV)
    rows, plan = sort_tokens(x, ids, 3)
    pad = plan.m_indices < 0
    g = torch.randn(rows.shape, generator=gen).bfloat16().to(DEV)
    clean = [rows.clone().requires_grad_(), w13.clone().requires_grad_(), w2.clone().requires_grad_()]
    y = expert_mlp_bf16(clean[0], plan.m_indices, *clean[1:])
    want = torch.autograd.grad(y, clean, g)
    dirty = [t.detach().clone() for t in clean]
    dirty[0][pad] = float("nan")
    for t in dirty:
        t.requires_grad_()
    g2 = g.clone()
    g2[pad] = float("inf")
    y2 = expert_mlp_bf16(dirty[0], plan.m_indices, *dirty[1:])
    assert torch.equal(y, y2) and bool((y[pad] == 0).all())
    for a, b in zip(want, torch.autograd.grad(y2, dirty, g2)):
        assert torch.equal(a, b)
    assert bool((want[0][pad] == 0).all())


def test_a_training_step_captured_into_a_graph():
    """Forward, backward and an update, replayed: the same weights as the eager steps give.  The
    eager step's graph is gone before the capture begins."""
    gen = torch.Generator().manual_seed(4)
    shape = dict(dtype=torch.bfloat16, device=DEV)
    x = torch.randn(128, 128, generator=gen).to(**shape)
    ids = torch.randint(0, 4, (128, 2), generator=gen).to(DEV)
    w = torch.rand(128, 2, generator=gen).to(DEV)
    g = torch.randn(128, 128, generator=gen).to(**shape)
    start = [(torch.randn(4, 2, 256, 64, generator=gen) / 11).to(**shape), (torch.randn(4, 2, 128, 64, generator=gen) / 11).to(**shape)]

    def step(weights):
        leaves = [t.detach().requires_grad_() for t in weights]
        grads = torch.autograd.grad(moe_forward_bf16(x, ids, w, *leaves), leaves, g)
        with torch.no_grad():
            for t, d in zip(weights, grads):
                t.sub_(d, alpha=2.0 ** -8)

    eager = [t.clone() for t in start]
    for _ in range(3):
        step(eager)
    captured = [t.clone() for t in start]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step([t.clone() for t in start])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(captured)
    for t, s in zip(captured, start):
        t.copy_(s)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(eager, captured):
        assert torch.equal(a, b)


def test_a_gradient_that_begins_anywhere():
    """The layer's result as a piece of a longer vector: its gradient is a contiguous piece of that
    vector's, six bytes behind a 16-byte boundary."""
    gen = torch.Generator().manual_seed(5)
    rows = torch.randn(128, 128, generator=gen).bfloat16().to(DEV)
    mi = torch.zeros(128, dtype=torch.int32, device=DEV)
    w13, w2 = (torch.randn(1, 2, 256, 64, generator=gen) / 11).bfloat16().to(DEV), (torch.randn(1, 2, 128, 64, generator=gen) / 11).bfloat16().to(DEV)
    lead, g = torch.zeros(3, dtype=torch.bfloat16, device=DEV), torch.randn(3 + 128 * 128, generator=gen).bfloat16().to(DEV)
    leaves = [t.requires_grad_() for t in (rows, w13, w2)]
    got = torch.autograd.grad(torch.cat([lead, expert_mlp_bf16(leaves[0], mi, *leaves[1:]).flatten()]), leaves, g)
    want = torch.autograd.grad(expert_mlp_bf16(leaves[0], mi, *leaves[1:]), leaves, g[3:].clone().view(128, 128))
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_without_a_gradient_no_rows_are_kept():
    rows = torch.ones(128, 128, dtype=torch.bfloat16, device=DEV)
    mi = torch.zeros(128, dtype=torch.int32, device=DEV)
    w13 = torch.ones(1, 2, 256, 64, dtype=torch.bfloat16, device=DEV).requires_grad_()
    w2 = torch.ones(1, 2, 128, 64, dtype=torch.bfloat16, device=DEV).requires_grad_()

    def launches(run):
        before = _cabi.query(_cabi.QUERY_LAUNCH_COUNT)
        with run:
            expert_mlp_bf16(rows, mi, w13, w2)
        return _cabi.query(_cabi.QUERY_LAUNCH_COUNT) - before

    assert launches(torch.enable_grad()) == launches(torch.no_grad()) + 1


def test_in_inference_mode_and_with_a_plan_copied():
    gen = torch.Generator().manual_seed(6)
    x = torch.randn(70, 128, generator=gen).bfloat16().to(DEV)
    ids = torch.randint(-1, 4, (70, 2), generator=gen).to(DEV)
    w = torch.rand(70, 2, generator=gen).to(DEV)
    w13, w2 = (torch.randn(4, 2, 256, 64, generator=gen) / 11).bfloat16().to(DEV), (torch.randn(4, 2, 128, 64, generator=gen) / 11).bfloat16().to(DEV)
    want = moe_forward_bf16(x, ids, w, w13, w2)
    with torch.inference_mode():
        assert torch.equal(moe_forward_bf16(x, ids, w, w13, w2), want)
    rows, plan = sort_tokens(x, ids, 4)
    copied = type(plan)(*[t.clone() for t in plan])
    for a, b in zip(plan, copied):
        assert a.is_contiguous() and a.data_ptr() % 16 == 0
    plan.counts.zero_()  # the plan's arrays are apart
    plan.offsets.fill_(-5)
    assert torch.equal(plan.dest, copied.dest) and torch.equal(plan.m_indices, copied.m_indices) and torch.equal(plan.m_total, copied.m_total)
    assert torch.equal(unsort_tokens(rows, plan, w), unsort_tokens(rows, copied, w))


def test_refusals():
    x = torch.zeros(128, 128, dtype=torch.bfloat16, device=DEV)
    mi = torch.zeros(128, dtype=torch.int32, device=DEV)
    w13, w2 = torch.zeros(2, 2, 256, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(2, 2, 128, 64, dtype=torch.bfloat16, device=DEV)
    for call in (lambda: expert_mlp_bf16(x.half(), mi, w13, w2), lambda: expert_mlp_bf16(x[:, :64], mi, w13, w2),
                 lambda: expert_mlp_bf16(x, mi, w13, w2[:1]), lambda: expert_mlp_bf16(x, mi, w2, w2),
                 lambda: expert_mlp_bf16(x, mi, w13, w2, checkpoint="none"), lambda: expert_mlp_bf16(x, mi, w13[0], w2)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        expert_mlp_bf16(x.cpu(), mi, w13, w2)
    with pytest.raises(RuntimeError):
        expert_mlp_bf16(x, mi[:64], w13, w2)
