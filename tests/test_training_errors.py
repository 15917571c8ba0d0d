"""Refusals of the training operators, on the CPU: the C ABI's argument checks (made before any
device is touched) and those of the Python functions that need no device."""
import ctypes
import os
import re

import pytest
import torch

import deepgemm
from deepgemm import _cabi

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"dg_input_grad_args": _cabi.InputGradArgs, "dg_weight_grad_args": _cabi.WeightGradArgs,
           "dg_token_sort_args": _cabi.TokenSortArgs, "dg_token_unsort_args": _cabi.TokenUnsortArgs,
           "dg_token_unsort_grad_args": _cabi.TokenUnsortGradArgs, "dg_clear_rows_args": _cabi.ClearRowsArgs,
           "dg_checkpoint_args": _cabi.CheckpointArgs, "dg_act_checkpoint_args": _cabi.ActCheckpointArgs}


@pytest.mark.parametrize("name", STRUCTS)
def test_struct_layouts_match_the_header(name):
    text = open(os.path.join(REPO, "include", "deepgemm_b200.h")).read()
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    assert re.findall(r"(\w+)\s*;", body) == [f[0] for f in STRUCTS[name]._fields_]
    sizes = {"int32_t": 4, "int64_t": 8, "size_t": 8}
    types = re.findall(r"(\w+)(\*?)\s+\w+\s*;", body)
    assert len(types) == len(STRUCTS[name]._fields_)
    for (ctype, star), field in zip(types, STRUCTS[name]._fields_):
        assert ctypes.sizeof(field[1]) == (8 if star else sizes[ctype]), field


def call(entry, args):
    return getattr(_cabi.lib, entry)(ctypes.byref(args) if args is not None else None, None)


def sort_args(**over):
    base = dict(elem_bytes=2, num_tokens=4, top_k=2, num_groups=3, hidden=64, align=1, cap=8, x_stride=64, x=4096, ids=4096,
                rows=4096, dest=4096, m_indices=4096, counts=4096, offsets=4096, m_total=4096)
    return _cabi.TokenSortArgs(**{**base, **over})


@pytest.mark.parametrize("over,code", [
    (dict(elem_bytes=1), -9), (dict(elem_bytes=8), -9), (dict(num_tokens=-1), -3), (dict(top_k=0), -3), (dict(num_groups=0), -3),
    (dict(hidden=0), -3), (dict(align=0), -3), (dict(num_groups=1025), -8), (dict(top_k=129), -8), (dict(num_tokens=2 ** 30, top_k=4), -8),
    (dict(cap=7), -3), (dict(align=128), -3), (dict(x=None), -1), (dict(ids=None), -1), (dict(rows=None), -1), (dict(dest=None), -1),
    (dict(m_indices=None), -1), (dict(counts=None), -1), (dict(offsets=None), -1), (dict(m_total=None), -1), (dict(x_stride=63), -3),
    (dict(num_tokens=65537, top_k=1, cap=65537), -9), (dict(x=4097), -4), (dict(rows=4097), -4), (dict(ids=4098), -4),
    (dict(ids=4100, ids64=1), -4), (dict(elem_bytes=4, x=4098), -4),
])
def test_sort_refuses(over, code):
    assert call("dg_token_sort", sort_args(**over)) == code


def test_null_arguments():
    for name in ("dg_grouped_input_grad", "dg_grouped_weight_grad", "dg_token_sort", "dg_token_unsort", "dg_token_unsort_grad", "dg_clear_padding_rows", "dg_checkpoint_rows",
                 "dg_restore_rows", "dg_act_checkpoint", "dg_act_checkpoint_grad"):
        assert call(name, None) == -1


def test_the_way_back_refuses():
    u = dict(elem=0, num_tokens=4, top_k=2, hidden=64, num_rows=8, y_stride=64, y=4096, dest=4096, out=4096)
    for over, code in ((dict(elem=3), -2), (dict(top_k=0), -3), (dict(hidden=0), -3), (dict(num_rows=-1), -3), (dict(y_stride=10), -3),
                       (dict(y=None), -1), (dict(dest=None), -1), (dict(out=None), -1), (dict(out=4097), -4),
                       (dict(num_tokens=2 ** 30, top_k=8), -8)):
        assert call("dg_token_unsort", _cabi.TokenUnsortArgs(**{**u, **over})) == code, over
    assert call("dg_token_unsort", _cabi.TokenUnsortArgs(**{**u, "num_tokens": 0, "out": None})) == 0
    g = dict(elem=1, num_tokens=4, top_k=2, hidden=64, num_rows=8, y_stride=64, dout_stride=64, dout=4096, y=4096, dest=4096, dy=4096,
             dw=4096, clear=1, m_indices=4096)
    for over, code in ((dict(elem=-1), -2), (dict(dout_stride=63), -3), (dict(y=None), -1), (dict(dy=None), -1), (dict(m_indices=None), -1),
                       (dict(dout=None), -1), (dict(dy=4097), -4)):
        assert call("dg_token_unsort_grad", _cabi.TokenUnsortGradArgs(**{**g, **over})) == code, over
    c = dict(elem=0, num_rows=8, hidden=64, rows=4096, m_indices=4096)
    for over, code in ((dict(elem=9), -2), (dict(hidden=0), -3), (dict(rows=None), -1), (dict(m_indices=None), -1), (dict(rows=4097), -4)):
        assert call("dg_clear_padding_rows", _cabi.ClearRowsArgs(**{**c, **over})) == code, over


def test_checkpoints_refuse():
    c = dict(elem=0, kind=1, num_rows=8, hidden=64, x_stride=64, x=4096, q=4096, scale=4096)
    for over, code in ((dict(kind=2), -2), (dict(kind=3), -2), (dict(elem=3), -2), (dict(hidden=0), -3), (dict(x_stride=63), -3),
                       (dict(x=None), -1), (dict(q=None), -1), (dict(scale=None), -1), (dict(x=4097), -4), (dict(scale=4098), -4)):
        for entry in ("dg_checkpoint_rows", "dg_restore_rows"):
            assert call(entry, _cabi.CheckpointArgs(**{**c, **over})) == code, (entry, over)
    assert call("dg_restore_rows", _cabi.CheckpointArgs(**{**c, "x_stride": 65})) == -3
    a = dict(elem=0, kind=0, num_rows=8, hidden=64, x_stride=128, dact_stride=64, x=4096, dact=4096, q=4096, scale=4096, act=4096, dx=4096)
    for over, code, entries in ((dict(kind=2), -2, "fb"), (dict(hidden=0), -3, "fb"), (dict(x_stride=127), -3, "f"), (dict(dact_stride=63), -3, "b"),
                                (dict(x=None), -1, "f"), (dict(act=None), -1, "f"), (dict(dact=None), -1, "b"), (dict(dx=None), -1, "b"),
                                (dict(q=None), -1, "fb"), (dict(act=4097), -4, "fb")):
        for e in entries:
            entry = "dg_act_checkpoint" if e == "f" else "dg_act_checkpoint_grad"
            assert call(entry, _cabi.ActCheckpointArgs(**{**a, **over})) == code, (entry, over)


def test_gradients_of_the_product_refuse():
    i = dict(dy=4096, w_packed=4096, dx=4096, m_indices=4096, num_groups=2, m_total=128, n=64, k=128)
    for over, code in ((dict(n=8), -3), (dict(n=72), -3), (dict(k=96), -3), (dict(k=0), -3), (dict(num_groups=0), -3), (dict(m_total=-1), -3),
                       (dict(num_groups=1025), -8), (dict(m_total=4096 * 128 + 1), -8), (dict(block_n=64), -9), (dict(dy=None), -1),
                       (dict(w_packed=None), -1), (dict(dx=None), -1), (dict(m_indices=None), -1), (dict(dy=4104), -4), (dict(dx=4098), -4)):
        assert call("dg_grouped_input_grad", _cabi.InputGradArgs(**{**i, **over})) == code, over
    assert call("dg_grouped_input_grad", _cabi.InputGradArgs(**{**i, "m_total": 0})) == 0
    w = dict(dy=4096, x=4096, dw=4096, m_indices=4096, num_groups=2, m_total=128, n=64, k=128)
    for over, code in ((dict(n=8), -3), (dict(n=72), -3), (dict(k=96), -3), (dict(num_groups=0), -3), (dict(num_groups=1025), -8),
                       (dict(m_total=4096 * 128 + 1), -8), (dict(tile=64), -9), (dict(out_kind=1), -9), (dict(accumulate=1), -9),
                       (dict(dy=None), -1), (dict(x=None), -1), (dict(dw=None), -1), (dict(m_indices=None), -1), (dict(x=4104), -4)):
        assert call("dg_grouped_weight_grad", _cabi.WeightGradArgs(**{**w, **over})) == code, over
    assert call("dg_grouped_weight_grad", _cabi.WeightGradArgs(**{**w, "m_total": 0, "out_kind": 2, "accumulate": 1})) == 0


def test_capacity():
    for pairs, experts, align in ((0, 4, 128), (1, 4, 128), (8, 256, 1), (8, 256, 128), (1000, 3, 16), (7, 7, 5)):
        got = deepgemm.sort_capacity(pairs, experts, align)
        assert got == _cabi.lib.dg_token_sort_capacity(pairs, experts, align)
        # the worst routing: as many experts in use as there can be, each but one with a single pair
        used = min(pairs, experts)
        worst = (used - 1) * align + -(-(pairs - used + 1) // align) * align if used else 0
        assert worst <= got and got % align == 0 and got - worst < align * max(used, 1)
    with pytest.raises(ValueError):
        deepgemm.sort_capacity(-1, 4)
    assert _cabi.lib.dg_token_sort_capacity(-1, 4, 1) == -1


def test_python_functions_refuse_cpu_tensors():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    ids = torch.zeros(4, 2, dtype=torch.int32)
    plan = deepgemm.TokenPlan(ids, torch.zeros(8, dtype=torch.int32), None, None, None)
    c = deepgemm.Checkpoint(torch.zeros(4, 64, dtype=torch.int8), torch.ones(4, 1), torch.bfloat16)
    w = torch.zeros(1, 1, 64, 64, dtype=torch.bfloat16)
    for f in (lambda: deepgemm.grouped_bf16_input_grad(x, w, ids[:, 0]), lambda: deepgemm.grouped_bf16_weight_grad(x, x, ids[:, 0], 1),
              lambda: deepgemm.sort_tokens(x, ids, 4), lambda: deepgemm.unsort_tokens(x, plan), lambda: deepgemm.sort_tokens_grad(x, plan),
              lambda: deepgemm.unsort_tokens_grad(x, x, plan), lambda: deepgemm.clear_padding_rows(x, ids[:, 0]),
              lambda: deepgemm.checkpoint_rows(x), lambda: deepgemm.restore_rows(c), lambda: deepgemm.silu_mul_checkpoint(x),
              lambda: deepgemm.silu_mul_checkpoint_grad(c, x), lambda: deepgemm.silu_mul(x)):
        with pytest.raises(RuntimeError, match="no CPU implementation"):
            f()
