"""Page-table operators of a paged KV cache (``fgw_page_*`` of ``libfgw_mha.so``): fork, free, reserve, compact, copy.

The table and the lengths alone say which pages are live: row b holds the pages of its first ``cache_seqlens[b]`` tokens,
and a page that no row holds is free. So there is no free list or count to keep in step; whoever keeps pages outside
the batch (a prefix cache) keeps them as rows of the table. Everything stays on the device: the calls read no length
on the host, and give new tables, so that a step in flight can go on reading the old ones.

``pools`` are the K and V caches of every layer, tensors of one shape [num_pages * page_size, ...] and type.
"""
import array
import operator
import struct

import torch

from fgw_b200 import _native
from fgw_b200.operators.mha.chunk_attention import on_device
from fgw_b200.operators.mha.kernels.mha_paged_fwd_sm100 import _current_stream

_PACK = struct.Struct(_native.struct_format(_native.PageParams)).pack
_kind_of = operator.attrgetter("shape", "dtype", "device")
_is_contiguous = operator.methodcaller("is_contiguous")
_data_ptr = operator.methodcaller("data_ptr")


def _check_pools(pools, page_size):
    """(data pointers, bytes of a row, number of pages, device index) of the pools."""
    if not pools:
        raise ValueError("at least one pool required")
    first = pools[0]
    shape, _, device = kind = _kind_of(first)
    rows = shape[0] if len(shape) >= 2 else 0
    if page_size <= 0 or rows <= 0 or rows % page_size:
        raise ValueError("pools must be [num_pages * page_size, ...] with a positive page size")
    if any([k != kind for k in map(_kind_of, pools)]):
        raise ValueError("pools must have one shape, type and device")
    row_bytes = first.numel() // rows * first.element_size()
    if row_bytes <= 0 or row_bytes % 16:
        raise ValueError("a pool row must be a multiple of 16 bytes")
    if rows // page_size > 1 << 30:
        raise ValueError("at most 2^30 pages")
    if device.type != "cuda":
        raise ValueError("every tensor must be on the same CUDA device")
    pointers = tuple(map(_data_ptr, pools))
    if not all(map(_is_contiguous, pools)) or any([p & 15 for p in pointers]):
        raise ValueError("pools must be contiguous and 16-byte aligned")
    return pointers, row_bytes, rows // page_size, first.get_device()


def _check_table(block_table, cache_seqlens, page_size, device):
    if block_table.dim() != 2 or cache_seqlens.shape != block_table.shape[:1] or not block_table.numel():
        raise ValueError("metadata shape mismatch")
    if block_table.shape[1] * page_size > (1 << 31) - 1 or block_table.numel() > (1 << 31) - 1:
        raise ValueError("requires logical positions and table entries to fit int32")
    _check_rows((block_table, cache_seqlens), device)


def _check_rows(tensors, device):
    for t in tensors:
        if t.dtype != torch.int32:
            raise ValueError("page table, lengths and page lists must be int32")
        if t.get_device() != device:
            raise ValueError("every tensor must be on the same CUDA device")
        if not t.is_contiguous():
            raise ValueError("kernel inputs must be contiguous")


def _run(call, size_key, pools, page_size, device, *pointers):
    """Pack the parameters and make the call on the current stream of the pools' device. ``size_key`` is (batch, table
    width, copies); ``pointers`` the tables' and lists' data pointers in the order of ``fgw_page_params``."""
    at, row_bytes, pages, _ = pools
    batch, width, copies = size_key
    addresses = array.array("Q", at)  # host memory that outlives the call
    params = _PACK(addresses.buffer_info()[0], *pointers, row_bytes, len(at), batch, width, page_size, pages, copies,
                   0, 0)
    nbytes = _native.page_workspace_bytes(batch, pages, copies)
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
    on_device(device, call, params, workspace.data_ptr(), nbytes, _current_stream(device))


def fork_pages(pools, block_table, cache_seqlens, parents, page_size, reserve_seqlens=None):
    """The state in which row i is a fork of row ``parents[i]``; returns (table, seqlens, status), all new tensors.

    ``parents`` [B] int32 reads the rows as they were: a row's own index keeps it, an index outside [0, B) frees it, and
    a beam step's choice is passed as it is. Full pages are shared. A partly filled last page stays with the first row
    that has its parent; the others get a page of their own with the filled tokens copied in every pool. Then row i has
    pages for ``reserve_seqlens[i]`` tokens (at least its own; at most the table's width). New pages are the lowest
    free ones. ``status`` [2] int32 is (pages needed, pages free): when the first is larger, the state is returned as
    it was and nothing is copied.
    """
    checked = _check_pools(pools, page_size)
    device = checked[3]
    _check_table(block_table, cache_seqlens, page_size, device)
    rows = (parents,) if reserve_seqlens is None else (parents, reserve_seqlens)
    if any([t.shape != cache_seqlens.shape for t in rows]):
        raise ValueError("metadata shape mismatch")
    _check_rows(rows, device)
    table = torch.empty_like(block_table)
    seqlens = torch.empty_like(cache_seqlens)
    status = cache_seqlens.new_empty(2)
    _run(_native.page_fork, (*block_table.shape, 0), checked, page_size, device, block_table.data_ptr(),
         cache_seqlens.data_ptr(), parents.data_ptr(), 0 if reserve_seqlens is None else reserve_seqlens.data_ptr(),
         table.data_ptr(), seqlens.data_ptr(), status.data_ptr(), 0, 0)
    return table, seqlens, status


def compact_pages(pools, block_table, cache_seqlens, page_size):
    """Move the live pages into the lowest ids, in every pool; returns (table, status), new tensors.

    With ``live`` pages held, the k-th held page from id ``live`` on goes to the k-th free page below it; afterwards the
    pools hold nothing from page ``live`` on. Pages that were reserved but hold no token yet are not live: pass the
    lengths the rows hold pages for. ``status`` [2] int32 is (live, pages moved).
    """
    checked = _check_pools(pools, page_size)
    device = checked[3]
    _check_table(block_table, cache_seqlens, page_size, device)
    table = torch.empty_like(block_table)
    status = cache_seqlens.new_empty(2)
    _run(_native.page_compact, (*block_table.shape, 0), checked, page_size, device, block_table.data_ptr(),
         cache_seqlens.data_ptr(), 0, 0, table.data_ptr(), 0, status.data_ptr(), 0, 0)
    return table, status


def copy_pages(pools, src_pages, dst_pages, page_size):
    """Copy page ``src_pages[i]`` to page ``dst_pages[i]`` in every pool (both [n] int32 on the device).

    No destination may be a source or occur twice; pairs with a page outside the pool are skipped.
    """
    checked = _check_pools(pools, page_size)
    if src_pages.dim() != 1 or dst_pages.shape != src_pages.shape or src_pages.numel() > (1 << 31) - 1:
        raise ValueError("metadata shape mismatch")
    _check_rows((src_pages, dst_pages), checked[3])
    if src_pages.numel():
        _run(_native.page_copy, (0, 0, src_pages.numel()), checked, page_size, checked[3], 0, 0, 0, 0, 0, 0, 0,
             src_pages.data_ptr(), dst_pages.data_ptr())
