"""Edges of the training operators that need no GPU: what the kernel sources and the host code promise."""
import ctypes
import glob
import os
import re

import pytest
import torch

import deepgemm
from deepgemm import _cabi

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def sources():
    return {os.path.basename(p): open(p).read() for p in glob.glob(os.path.join(REPO, "deepgemm-das_b200", "csrc", "*.c*"))}


def test_posted_counts_are_acquired():
    """A count that one warp posts in shared memory for another is stored with release and read with
    acquire, in one place: a volatile read would order nothing behind it."""
    text = sources()
    assert not [n for n, t in text.items() if re.search(r'asm volatile\(\s*"[^"]*ld\.volatile', t)]
    assert [n for n, t in text.items() if "st.release.cta.shared" in t] == ["dg_ptx.cuh"]
    assert [n for n, t in text.items() if "ld.acquire.cta.shared" in t] == ["dg_ptx.cuh"]
    for n, t in text.items():
        assert ("post_count(" in t) == ("poll_above(" in t), n


def test_clearing_refuses_a_number_of_groups_that_is_none():
    args = dict(elem=0, num_rows=8, hidden=64, rows=4096, m_indices=4096)
    assert _cabi.lib.dg_clear_padding_rows(ctypes.byref(_cabi.ClearRowsArgs(**args, num_groups=-1)), None) == -3
    rows, mi = torch.zeros(8, 64), torch.zeros(8, dtype=torch.int32)
    for groups in (-1, 1025):
        with pytest.raises(ValueError, match="num_groups"):
            deepgemm.clear_padding_rows(rows, mi, groups)


def test_the_header_says_where_scratch_begins():
    text = open(os.path.join(REPO, "include", "deepgemm_b200.h")).read()
    most = int(re.search(r"dg_token_sort needs: 0 up to (\d+) pairs", text).group(1))
    for top_k in (1, 3, 8, 128):
        tokens = most // top_k
        assert _cabi.lib.dg_token_sort_scratch_bytes(tokens, top_k, 32) == 0
        assert _cabi.lib.dg_token_sort_scratch_bytes(tokens + 1, top_k, 32) > 0
    args = dict(elem_bytes=2, top_k=1, num_groups=3, hidden=64, align=1, x_stride=64, x=4096, ids=4096, rows=4096, dest=4096,
                m_indices=4096, counts=4096, offsets=4096, m_total=4096)
    beyond = _cabi.TokenSortArgs(**args, num_tokens=most + 1, cap=most + 1)
    assert _cabi.lib.dg_token_sort(ctypes.byref(beyond), None) == -9
    beyond.scratch, beyond.scratch_bytes = 4096, _cabi.lib.dg_token_sort_scratch_bytes(most + 1, 1, 3) - 1
    assert _cabi.lib.dg_token_sort(ctypes.byref(beyond), None) == -9


def test_results_on_their_inputs_are_refused():
    """Buffers are compared by address, before any device is touched."""
    def code(entry, cls, **args):
        return getattr(_cabi.lib, entry)(ctypes.byref(cls(**args)), None)

    base = 1 << 20
    sort = dict(elem_bytes=2, num_tokens=4, top_k=2, num_groups=3, hidden=64, align=1, cap=8, x_stride=80, x=base, ids=base + 4096,
                dest=base + 8192, m_indices=base + 8192, counts=base + 8192, offsets=base + 8192, m_total=base + 8192)
    x_end = base + (3 * 80 + 64) * 2
    for rows in (base, x_end - 2, base - 8 * 128 + 2, base + 4096 + 30, base + 4096 - 8 * 128 + 2):
        assert code("dg_token_sort", _cabi.TokenSortArgs, **sort, rows=rows) == -9, rows - base
    back = dict(elem=0, num_tokens=4, top_k=2, hidden=64, num_rows=8, y_stride=64, y=base, dest=base + 4096, weights=base + 8192)
    for out in (base, base + 8 * 128 - 2, base - 4 * 128 + 2, base + 4096 + 30, base + 8192 - 2):
        assert code("dg_token_unsort", _cabi.TokenUnsortArgs, **back, out=out) == -9, out - base
    grad = dict(elem=0, num_tokens=4, top_k=2, hidden=64, num_rows=8, y_stride=64, dout_stride=64, dout=base, y=base + 4096, dest=base + 8192,
                dw=base + 8192, m_indices=base + 8192, clear=1)
    for dy in (base + 510, base - 1022, base + 4096 + 1022):
        assert code("dg_token_unsort_grad", _cabi.TokenUnsortGradArgs, **grad, dy=dy) == -9, dy - base
    rows = dict(m_indices=base - 4096, num_groups=2, m_total=128, n=64, k=128)
    wide, deep = 128 * 128 * 2, 128 * 64 * 2
    for dx in (base, base + deep - 16, base - wide + 16, base + (1 << 20), base + (1 << 20) + 2 * 64 * 128 * 2 - 16, base - 4096):
        assert code("dg_grouped_input_grad", _cabi.InputGradArgs, **rows, dy=base, w_packed=base + (1 << 20), dx=dx) == -9, dx - base
    for kind, size in ((0, 2), (2, 4)):
        for dw in (base, base + deep - 16, base + (1 << 20) + wide - 16, base + (1 << 20) - 2 * 64 * 128 * size + 16, base - 4096):
            assert code("dg_grouped_weight_grad", _cabi.WeightGradArgs, **rows, dy=base, x=base + (1 << 20), dw=dw, out_kind=kind) == -9, dw - base


def test_neighbours_in_a_buffer_are_apart():
    room = torch.zeros(64, 16)
    core = deepgemm._core
    core._apart(room[:8], "f", x=room[8:], y=None, z=room[8:8])
    core._apart(room[8:8], "f", x=room)
    for out, x in ((room[:8], room[7:]), (room[7:], room[:8]), (room[3:4], room), (room[8:16], room[:32, :4][::4])):
        with pytest.raises(ValueError, match="overlap x"):
            core._apart(out, "f", x=x)
