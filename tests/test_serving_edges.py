"""Edges of the serving-step operators beyond the sizes of test_serving_ops.py: limits, large batches, shared pages, values that
are not finite. Exact where integers are compared; tolerances elsewhere are those of test_serving_ops.py.
"""
import ctypes

import pytest
import torch

from fgw_b200 import _native

MAX_ENTRIES = 2 ** 31 - 2 ** 16


def page_params(**values):
    p = _native.PageParams()
    for key, value in {**dict(block_table=256, cache_seqlens=512, parents=256, table_out=1024, seqlens_out=2048, status=256,
                              batch=2, table_width=2, page_size=1, num_pages=9), **values}.items():
        setattr(p, key, value)
    return p


def test_page_operators_refuse_tables_past_their_loops():
    """The plan's loops step past the last entry in 32 bits; larger tables are refused before any CUDA call."""
    lib = _native.library()
    for batch, width in ((2 ** 31 - 1, 1), (1, 2 ** 31 - 1), (2 ** 15, 2 ** 16 - 1), (MAX_ENTRIES // 5 + 1, 5)):
        p = page_params(batch=batch, table_width=width)
        assert lib.fgw_page_fork(ctypes.byref(p), 256, 16, None) == 1, (batch, width)
        assert lib.fgw_page_compact(ctypes.byref(p), 256, 16, None) == 1, (batch, width)
    for batch, width in ((MAX_ENTRIES, 1), (1, MAX_ENTRIES), (2 ** 15 - 1, 2 ** 16)):
        p = page_params(batch=batch, table_width=width)
        assert lib.fgw_page_fork(ctypes.byref(p), 256, 16, None) == _native.ERR_WORKSPACE_TOO_SMALL, (batch, width)


@pytest.mark.gpu
def test_page_operators_refuse_tables_past_their_loops_from_python():
    from fgw_b200.operators.mha.page_ops import compact_pages, fork_pages
    pool = [torch.zeros(16, 8, dtype=torch.bfloat16, device="cuda")]
    one = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    table, lens = one.expand(2 ** 15, 2 ** 16 - 1), one[0].expand(2 ** 15)
    with pytest.raises(ValueError, match="table entries"):
        fork_pages(pool, table, lens, lens, 1)
    with pytest.raises(ValueError, match="table entries"):
        compact_pages(pool, table, lens, 1)
