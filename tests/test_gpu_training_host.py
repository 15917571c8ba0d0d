"""The training operators' host side on a GPU: both marshalling paths give the same bytes, refusals
carry messages, and tensors that lie elsewhere or oddly are refused or handled."""
import pytest
import torch

import deepgemm
from deepgemm import activation_checkpoint, grouped_grad, token_sort
from deepgemm import (Checkpoint, TokenPlan, checkpoint_rows, clear_padding_rows, grouped_bf16_input_grad, grouped_bf16_weight_grad,
                      restore_rows, silu_mul, silu_mul_checkpoint, silu_mul_checkpoint_grad, sort_tokens, sort_tokens_grad,
                      unsort_tokens, unsort_tokens_grad)

pytestmark = pytest.mark.gpu
DEV = "cuda"


def everything(seed):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen).bfloat16().to(DEV)  # noqa: E731
    x, ids = r(45, 256), torch.randint(-1, 6, (45, 3), generator=gen).to(DEV)
    w = torch.rand(45, 3, generator=gen).to(DEV)
    rows, plan = sort_tokens(x, ids, 6)
    m = rows.shape[0]
    out = unsort_tokens(rows, plan, w)
    dy, dw = unsort_tokens_grad(x, rows, plan, w)
    dx = sort_tokens_grad(rows, plan)
    h, weight = r(m, 512), r(6, 4, 512, 64)
    act, kept = silu_mul_checkpoint(h, m_indices=plan.m_indices)
    dh, again = silu_mul_checkpoint_grad(kept, act, m_indices=plan.m_indices)
    c = checkpoint_rows(x, kind="int8")
    got = [rows, *plan, out, dy, dw, dx, act, *kept[:2], dh, again, *c[:2], restore_rows(c),
           grouped_bf16_input_grad(h, weight, plan.m_indices), grouped_bf16_weight_grad(h, rows, plan.m_indices, 6),
           grouped_bf16_weight_grad(h, rows, plan.m_indices, 6, dtype=torch.float32)]
    return got


def test_both_marshalling_paths_give_the_same_bytes(monkeypatch):
    if token_sort._glue is None:
        pytest.skip("the host glue is not built")
    everything(0)                                    # the status words are known to the glue from here on
    before = token_sort._glue.stats()
    native = everything(1)
    after = token_sort._glue.stats()
    assert after[0] - before[0] == 11 and after[1] == before[1]
    for module in (token_sort, activation_checkpoint, grouped_grad):
        monkeypatch.setattr(module, "_glue", None)
    plain = everything(1)
    for a, b in zip(native, plain):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_refusals():
    x, ids = torch.zeros(8, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(8, 2, dtype=torch.int32, device=DEV)
    rows, plan = sort_tokens(x, ids, 4)
    w = torch.ones(8, 2, device=DEV)
    c = checkpoint_rows(x)
    act, kept = silu_mul_checkpoint(x)
    leaf = x.clone().requires_grad_()
    bad = [
        lambda: sort_tokens(x.int(), ids, 4), lambda: sort_tokens(x[0], ids, 4), lambda: sort_tokens(x.t(), ids, 4),
        lambda: sort_tokens(x.expand(8, 64)[:, :0], ids, 4), lambda: sort_tokens(x[:1].expand(8, 64), ids, 4),
        lambda: sort_tokens(x, ids.float(), 4), lambda: sort_tokens(x, ids[:4], 4), lambda: sort_tokens(x, ids.cpu(), 4),
        lambda: sort_tokens(x, ids, 0), lambda: sort_tokens(x, ids, 1025), lambda: sort_tokens(x, ids, 4, align=0),
        lambda: sort_tokens(x, ids.repeat(1, 65), 4), lambda: sort_tokens(x, ids, 4, out=rows[:-1]), lambda: sort_tokens(x, ids, 4, out=rows.half()),
        lambda: sort_tokens(leaf, ids, 4, out=rows),
        lambda: unsort_tokens(rows[:-1], plan), lambda: unsort_tokens(rows, plan, w.half()), lambda: unsort_tokens(rows, plan, w[:4]),
        lambda: unsort_tokens(rows, plan, w, out=rows), lambda: unsort_tokens(rows, TokenPlan(plan.dest.long(), *plan[1:])),
        lambda: unsort_tokens_grad(x.float(), rows, plan, w), lambda: unsort_tokens_grad(x[:4], rows, plan, w),
        lambda: sort_tokens_grad(rows[:, :32], TokenPlan(plan.dest[0], *plan[1:])), lambda: clear_padding_rows(rows, ids[:, 0]),
        lambda: checkpoint_rows(x, kind="fp4"), lambda: checkpoint_rows(x.double()), lambda: restore_rows(Checkpoint(c.q, c.scale[:4], c.dtype)),
        lambda: restore_rows(Checkpoint(c.q, c.scale, torch.int8)), lambda: restore_rows(Checkpoint(x, c.scale, c.dtype)),
        lambda: silu_mul_checkpoint(x[:, :63]), lambda: silu_mul_checkpoint(x, m_indices=ids[:, 0].long()),
        lambda: silu_mul_checkpoint_grad(kept, act.half()), lambda: silu_mul_checkpoint_grad(kept, act[:4]),
        lambda: silu_mul_checkpoint_grad(kept, act, m_indices=ids[:4, 0]), lambda: silu_mul(x, checkpoint="bf16"),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print("accepted:", i)
    torch.cuda.synchronize()
    deepgemm.check_device_status()


def test_gradients_that_autograd_hands_over_laid_out_oddly():
    x = torch.randn(30, 64, device=DEV).requires_grad_()
    ids = torch.randint(0, 4, (30, 2), device=DEV)
    w = torch.rand(30, 2, device=DEV)
    g = torch.randn(64, 30, device=DEV)

    def f(x):
        rows, plan = sort_tokens(x, ids, 4, align=16)
        return unsort_tokens(silu_mul(rows.repeat(1, 2), m_indices=plan.m_indices), plan, w)

    a, = torch.autograd.grad(f(x), x, g.t())                   # transposed
    b, = torch.autograd.grad(f(x), x, g.t().contiguous())
    assert torch.equal(a, b)
    a, = torch.autograd.grad(f(x), x, torch.ones(1, 1, device=DEV).expand(30, 64))
    b, = torch.autograd.grad(f(x), x, torch.ones(30, 64, device=DEV))
    assert torch.equal(a, b)
    # only one of the two wants a gradient
    rows, plan = sort_tokens(x.detach(), ids, 4)
    ww = w.clone().requires_grad_()
    assert torch.autograd.grad(unsort_tokens(rows, plan, ww).sum(), ww)[0].shape == w.shape
    yy = rows.clone().requires_grad_()
    assert torch.autograd.grad(unsort_tokens(yy, plan, w).sum(), yy)[0].shape == rows.shape
    with torch.no_grad():
        assert not unsort_tokens(yy, plan, ww).requires_grad


def test_two_streams_at_once():
    x = torch.randn(3000, 512, device=DEV).bfloat16()
    ids = torch.randint(0, 32, (3000, 4), device=DEV)
    want = sort_tokens(x, ids, 32)
    wanta, wantc = silu_mul_checkpoint(x)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            for _ in range(3):
                got.append((sort_tokens(x, ids, 32), silu_mul_checkpoint(x)))
    torch.cuda.synchronize()
    for (rows, plan), (act, c) in got:
        assert torch.equal(rows, want[0]) and torch.equal(plan.dest, want[1].dest)
        assert torch.equal(act, wanta) and torch.equal(c.scale, wantc.scale)
