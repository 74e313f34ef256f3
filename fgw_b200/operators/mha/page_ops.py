"""Page-table operators of a paged KV cache (``fgw_page_*`` of ``libfgw_mha.so``): fork, free, reserve, compact, copy.

The table and the lengths alone say which pages are live: row b holds the pages of its first ``cache_seqlens[b]`` tokens,
and a page that no row holds is free. So there is no free list or count to keep in step; whoever keeps pages outside
the batch (a prefix cache) keeps them as rows of the table. Everything stays on the device: the calls read no length
on the host, and give new tables, so that a step launched before on the same stream reads the old ones. A step on another
stream has to be waited for: pages that a fork frees may be given out and written by the same call.

``pools`` are the K and V caches of every layer, a list of tensors of one shape [num_pages * page_size, ...] and type
whose rows are multiples of 16 bytes. Arguments that do not fit raise ValueError before any launch.
"""
from fgw_b200 import _native


def fork_pages(pools, block_table, cache_seqlens, parents, page_size, reserve_seqlens=None):
    """The state in which row i is a fork of row ``parents[i]``; returns (table, seqlens, status), all new tensors.

    ``parents`` [B] int32 reads the rows as they were: a row's own index keeps it, an index outside [0, B) frees it, and
    a beam step's choice is passed as it is. Full pages are shared. A partly filled last page stays with the first row
    that has its parent; the others get a page of their own with the filled tokens copied in every pool. So does the first
    where another parent's row holds that page too, as after a length was lowered: afterwards the page that a row's next
    token goes to is the row's own (so a lowered row passes through here before it is appended to). Then row i has pages
    for ``reserve_seqlens[i]`` tokens (at least its own; at most the table's width). New pages are the lowest free ones.
    ``status`` [2] int32 is (pages needed, pages free): when the first is larger, the state is returned as it was and
    nothing is copied.
    """
    return _native.torch_binding().fork_pages(pools, block_table, cache_seqlens, parents, page_size, reserve_seqlens)


def compact_pages(pools, block_table, cache_seqlens, page_size):
    """Move the live pages into the lowest ids, in every pool; returns (table, status), new tensors.

    With ``live`` pages held, the k-th held page from id ``live`` on goes to the k-th free page below it; afterwards the
    pools hold nothing from page ``live`` on. Pages that were reserved but hold no token yet are not live: pass the
    lengths the rows hold pages for. ``status`` [2] int32 is (live, pages moved).
    """
    return _native.torch_binding().compact_pages(pools, block_table, cache_seqlens, page_size)


def copy_pages(pools, src_pages, dst_pages, page_size):
    """Copy page ``src_pages[i]`` to page ``dst_pages[i]`` in every pool (both [n] int32 on the device).

    No destination may be a source or occur twice; pairs with a page outside the pool are skipped.
    """
    _native.torch_binding().copy_pages(pools, src_pages, dst_pages, page_size)
