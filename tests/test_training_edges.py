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
