"""Chunk attention when loads get lost: every wait gives up in time, the status says so, and the next call is right.

``fgw_chunk_selftest_wait`` runs the call with K's or V's boxes half as high as the kernels wait for: barriers that nothing
completes, without a fault.
"""
import ctypes
import time

import pytest
import torch

from fgw_b200 import _native
from test_serving_ops import attend_case, check_attention, on_gpu

pytestmark = pytest.mark.gpu

# (new tokens, held, heads, kv heads, dim, page, causal): decode kernel alone, items of 16, 32 and 64 rows
TOKENS = [
    ([1] * 40, [300 + 17 * i for i in range(40)], 8, 2, 128, 16, True),
    ([1] * 5, [4000, 1, 77, 2000, 900], 4, 4, 64, 64, True),
    ([7] * 12, [7 + 113 * i for i in range(12)], 8, 2, 128, 32, True),
    ([8, 5, 1, 7] * 3, [8 + 113 * i for i in range(12)], 8, 1, 256, 48, False),
    ([2] * 6, [500 + 100 * i for i in range(6)], 8, 1, 176, 16, True),
]

# chunks (tensor kernel), and chunks among single tokens (both kernels): items cut, whole, of one tile and two
CHUNKS = [
    ([600], [1600], 8, 2, 128, 64, True),
    ([70, 1, 300, 128, 1], [170, 3000, 310, 128, 700], 16, 16, 128, 128, True),
    ([400, 30, 1, 130, 257, 1], [500, 3000, 1200, 130, 2000, 1], 24, 8, 64, 32, True),
    ([100, 33, 1, 200], [1100, 33, 400, 600], 6, 2, 176, 48, True),
    ([140, 1, 90], [300, 2000, 1000], 4, 2, 256, 64, False),
]


def native_call(case, dtype=torch.bfloat16, budget_ms=20):
    """(params, workspace, guarded output, inputs) of one call by the C ABI."""
    new, held, heads, kv_heads, dim, page, causal = case
    inputs = attend_case(("x", new, held, heads, kv_heads, dim, page, causal), dtype, seed=31)
    q, k, v, table, lens, cu = inputs
    gpu = [q.cuda(), k.cuda(), v.cuda(), *on_gpu(table, lens, cu)]
    room = torch.full((q.shape[0] + 2, heads, dim), 7.0, dtype=dtype, device="cuda")
    p = _native.ChunkParams()
    for name, t in zip(("q", "k_cache", "v_cache", "block_table", "cache_seqlens", "cu_seqlens_q", "out"),
                       (*gpu, room[1:-1])):
        setattr(p, name, t.data_ptr())
    for name, value in dict(tokens=q.shape[0], pool_rows=k.shape[0], q_stride=heads * dim, out_stride=heads * dim,
                            batch=len(new), heads=heads, kv_heads=kv_heads, head_dim=dim, table_width=table.shape[1],
                            page_size=page, dtype=_native.DTYPE_BFLOAT16, causal=int(causal), softmax_scale=dim ** -0.5,
                            wait_budget_ms=budget_ms).items():
        setattr(p, name, value)
    size = ctypes.c_size_t()
    assert _native.library().fgw_chunk_workspace_size(ctypes.byref(p), ctypes.byref(size)) == 0
    workspace = torch.full((size.value,), 255, dtype=torch.uint8, device="cuda")
    return p, workspace, room, inputs, gpu


def run_case(case, short, sites):
    lib, stream = _native.library(), torch.cuda.current_stream().cuda_stream
    p, workspace, room, inputs, gpu = native_call(case)
    args = (workspace.data_ptr(), workspace.numel(), stream)
    started = time.perf_counter()
    assert lib.fgw_chunk_selftest_wait(ctypes.byref(p), short, *args) == 0
    status, site = _native.read_error(workspace.data_ptr(), stream)
    assert status == _native.ERR_DEVICE_TIMEOUT and site in sites, site
    # a CTA's roles give up within a few budgets and wait at most 0.1 s for each of up to eight stages of either ring
    assert time.perf_counter() - started < 5.0
    assert (room[0] == 7).all() and (room[-1] == 7).all()
    assert lib.fgw_chunk_attention(ctypes.byref(p), *args) == 0
    assert _native.read_error(workspace.data_ptr(), stream) == (_native.OK, 0)
    new, held, heads, kv_heads, dim, page, causal = case
    check_attention(room[1:-1], *inputs, page, causal, dim ** -0.5)


@pytest.mark.parametrize("short", [1, 2, 3])
@pytest.mark.parametrize("case", TOKENS, ids=range(len(TOKENS)))
def test_decode_kernel_gives_up_on_lost_loads(case, short):
    run_case(case, short, sites=(70, 71))


@pytest.mark.parametrize("short", [1, 2, 3])
@pytest.mark.parametrize("case", CHUNKS, ids=range(len(CHUNKS)))
def test_tensor_kernel_gives_up_on_lost_loads(case, short):
    run_case(case, short, sites=(70, 71, *range(80, 94)))


def test_selftest_refuses():
    p, workspace, *_ = native_call(TOKENS[1])
    for short in (-1, 4):
        assert _native.library().fgw_chunk_selftest_wait(ctypes.byref(p), short, workspace.data_ptr(), workspace.numel(),
                                                         None) == 1


def test_a_lost_load_is_reported_to_python_once():
    """The Python call's workspace is gone when it returns: the status stays readable, for each device, until it is read."""
    from fgw_b200.operators.mha.chunk_attention import paged_chunk_attention, read_error
    lib, stream = _native.library(), torch.cuda.current_stream().cuda_stream
    read_error()
    for case in (TOKENS[2], CHUNKS[2]):
        p, workspace, room, inputs, gpu = native_call(case)
        args = (workspace.data_ptr(), workspace.numel(), stream)
        assert lib.fgw_chunk_selftest_wait(ctypes.byref(p), 1, *args) == 0
        first = _native.read_error(workspace.data_ptr(), stream)
        assert lib.fgw_chunk_attention(ctypes.byref(p), *args) == 0  # a later good call does not cover it
        new, held, heads, kv_heads, dim, page, causal = case
        paged_chunk_attention(*gpu, page, is_causal=causal)
        assert first[0] == _native.ERR_DEVICE_TIMEOUT
        assert read_error() == first
        assert read_error(0) == (_native.OK, 0)
        check_attention(paged_chunk_attention(*gpu, page, is_causal=causal), *inputs, page, causal, dim ** -0.5)
        assert read_error(torch.device("cuda", 0)) == (_native.OK, 0)
