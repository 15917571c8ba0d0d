"""Edges of the training operators that need no GPU: what the kernel sources and the host code promise."""
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
