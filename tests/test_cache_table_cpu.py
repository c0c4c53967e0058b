"""What the cache kernels read of a sequence's table of pages, on the host from the kernels' own
header, and which kernel the full tables of tests/test_cache_edges_gpu.py take."""
import ctypes

import numpy as np
import pytest

from tests.cache_host import library

SOURCE = """
#include "cache.hpp"
extern "C" int page_of(const int32_t* table, int64_t pages, int M, int b, int i) {
  tpo::Cache c;
  c.table = table;
  c.pages = pages;
  c.M = M;
  return c.page_of(b, i);
}
"""


@pytest.fixture(scope="module")
def page_of(tmp_path_factory):
    lib = library(SOURCE, tmp_path_factory.mktemp("table"))
    lib.page_of.argtypes = [ctypes.c_void_p, ctypes.c_int64] + [ctypes.c_int] * 3
    return lib.page_of


def test_entries_of_other_sequences_are_not_read(page_of):
    """A sequence has M entries: what lies behind them, another's or nobody's, is no page of it."""
    B, M = 3, 5
    table = np.arange(B * M + 4, dtype=np.int32)  # (the last four are behind the table)
    table[7], table[8] = -1, 100
    for b in range(B):
        for i in range(-2, M + 4):
            inside = 0 <= i < M and b * M + i not in (7, 8)
            if b * M + i < 0:
                continue
            assert page_of(table.ctypes.data, 50, M, b, i) == (b * M + i if inside else -1), (b, i)


def test_full_tables_take_the_kernel_of_128_rows(tpo):
    from tests import test_cache_edges_gpu as t
    from torch_point_ops import _native

    rows = ctypes.CDLL(_native.HIP_LIB).tpo_cache_attention_rows
    rows.argtypes = [ctypes.c_int] + [ctypes.c_int64] * 7
    for page, M in t.FULL:
        assert page // 32 * M % 2 == 1
        for dtype in (2, 3):
            assert rows(dtype, len(t.FULL_NEW), sum(t.FULL_NEW), 2 * t.FULL_HEADS, t.FULL_HEADS,
                        t.FULL_D, page, M) == 128
