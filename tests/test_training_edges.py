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
