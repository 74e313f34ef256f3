"""Attention of a ragged batch of new tokens over a paged KV cache (``fgw_chunk_attention`` of ``libfgw_mha.so``).

FGW's ``mha_paged_decode`` takes one query length for the whole batch and as many key heads as query heads. A serving
step brings single tokens and prompt chunks together, grouped heads, and lengths that live on the device;
``paged_chunk_attention`` takes those as they are: query head h reads key head h // (heads // kv_heads), request b's
new tokens are rows ``cu_seqlens_q[b]`` to ``cu_seqlens_q[b + 1]``, and nothing is copied to the host.
"""
import torch

from fgw_b200 import _native


def paged_chunk_attention(q, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens_q, page_size, is_causal=True,
                          softmax_scale=None, out=None):
    """Attention of the new tokens over everything cached; returns ``out`` [T, H, D].

    ``q`` is [T, H, D] (each token's heads contiguous, any token stride that is a multiple of 8: a slice of a fused
    projection serves as it is), ``k_cache`` / ``v_cache`` [pool_rows, Hkv, D], ``block_table`` [B, W] int32,
    ``cache_seqlens`` [B] int32 (tokens in the cache with the new ones), ``cu_seqlens_q`` [B + 1] int32. Causal: the
    i-th of a request's n new tokens sees the first ``cache_seqlens - n + i + 1`` cached ones. Rows that see nothing (or
    only scores of -inf) and rows of no request are exact zeros; a score that is NaN or +inf makes its row NaN. Cached
    values have to be finite: one that is not reaches rows of its request whose mask hides it too. ``softmax_scale``
    defaults to 1 / sqrt(D). At most 128 query heads may share a key head. Raises ValueError for tensors that do not fit this, before any launch. Waits on
    the device give up after two seconds; ``read_error`` reports it, and the output is then undefined.
    """
    return _native.torch_binding().paged_chunk_attention(q, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens_q,
                                                         page_size, is_causal, softmax_scale, out)


def read_error(device=None):
    """Device-side status of the calls on ``device`` (the current one by default) since it was last read.

    Waits for the device's current stream and returns (status, wait site): ``(_native.OK, 0)``, or
    ``_native.ERR_DEVICE_TIMEOUT`` with the site of the first wait that gave up, and clears it. Not during a capture.
    """
    with torch.cuda.device(device):
        return _native.chunk_read_error(torch.cuda.current_stream().cuda_stream)
