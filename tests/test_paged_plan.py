"""The paged cache's host arithmetic (qwenscriber_amd/csrc/paged_plan.h) on the
CPU: qwenscriber_amd/sanitize/paged_check.cpp, built with g++ and its
sanitizers (Makefile `paged_check`, no device code), holds the entry points'
refusals and runs thousands of sets of page copies (forks, chains, swaps,
cycles longer than a launch) step by step as the kernel does, against all
sources read before any destination is written. And what the binding itself
refuses."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

import qwenscriber_amd as qa
from qwenscriber_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CHECK = os.path.join(ROOT, "qwenscriber_amd", "build", "paged_check")


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host C++ compiler")
def test_refusals_and_copy_order():
    subprocess.run(["make", "-s", "-C", os.path.join(ROOT, "qwenscriber_amd"), "paged_check"], check=True)
    run = subprocess.run([CHECK], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout[-3000:] + run.stderr[-2000:]
    assert " 0 failures" in run.stdout, run.stdout


def test_null_context_is_refused_without_a_device():
    lib = qa.load()
    cache, batch = qa.PagedCache(), qa.PagedBatch()
    assert lib.qwh_paged_append(None, cache, 0, batch, None, 0, 1, None, None, 1e-6, None, None, 0, None, 0) == -1
    assert lib.qwh_paged_attention(None, cache, 0, batch, None, None, 0, 1) == -1
    assert lib.qwh_paged_copy(None, cache, None, None, 1) == -1
    assert lib.qwh_rope_tables(None, 64, 1, 1e6, None, None) == -1
    assert lib.qwh_sample_rows(None, None, 1, 1, None, None, None) == -1
    assert lib.qwh_decoder_sample(None, None, None, None) == -1


@pytest.mark.parametrize("pages", [[2**32 + 1], [-1], np.array([3, 2**40], np.int64), np.array([-2**31], np.int32), [1.5], np.ones(2),
                                   [2**70], ["1"], [None], [True]])
def test_what_is_no_page_number_is_refused(pages):
    """Not taken as the page that its low 32 bits or its whole part name."""
    with pytest.raises(ValueError):
        _lib._page_numbers(pages)


@pytest.mark.parametrize("pages", [[], [0, 5, 2**32 - 1], (1, 2), np.arange(6)[::-2], np.arange(4, dtype=np.uint8),
                                   np.array([7, 2**32 - 1], np.uint32), np.array([2**31], np.uint64)])
def test_page_numbers_of_any_whole_type(pages):
    got = _lib._page_numbers(pages)
    assert got.dtype == np.uint32 and got.flags.c_contiguous and got.tolist() == [int(p) for p in pages]


def test_descriptors_have_the_header_s_layout():
    # Five 32-bit fields, padding, four pointers; three fields, padding, three
    # pointers; four 32-bit fields.
    assert ctypes.sizeof(qa.PagedCache) == 24 + 32 and qa.PagedCache.k_scales.offset == 24
    assert ctypes.sizeof(qa.PagedBatch) == 16 + 24 and qa.PagedBatch.row_starts.offset == 16
    assert ctypes.sizeof(qa.Sampling) == 16 and qa.Sampling.min_p.offset == 12
    assert qa.PAGE_NONE == np.uint32(0xFFFFFFFF)
