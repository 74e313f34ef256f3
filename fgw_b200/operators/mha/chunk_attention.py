"""Attention of a ragged batch of new tokens over a paged KV cache (``fgw_chunk_attention`` of ``libfgw_mha.so``).

FGW's ``mha_paged_decode`` takes one query length for the whole batch and as many key heads as query heads. A serving
step brings single tokens and prompt chunks together, grouped heads, and lengths that live on the device;
``paged_chunk_attention`` takes those as they are: query head h reads key head h // (heads // kv_heads), request b's
new tokens are rows ``cu_seqlens_q[b]`` to ``cu_seqlens_q[b + 1]``, and nothing is copied to the host.
"""
import functools
import struct

import torch

from fgw_b200 import _native
from fgw_b200.operators.mha.kernels.mha_paged_fwd_sm100 import _KEPT, _KEPT_WORKSPACE_BYTES, _current_stream

_DTYPES = {torch.float16: _native.DTYPE_FLOAT16, torch.bfloat16: _native.DTYPE_BFLOAT16}
MAX_GROUP = 128  # query heads that may share a key head
_PACK = struct.Struct(_native.struct_format(_native.ChunkParams)).pack  # one call instead of a store per field


def check_ragged(q, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens_q, page_size):
    """Checks shared by the operators over a ragged batch and a paged cache; returns (tokens, heads, dim, kv_heads,
    pool_rows, batch, width)."""
    pool = k_cache.shape
    if q.dim() != 3 or len(pool) != 3 or v_cache.shape != pool:
        raise ValueError("Expected q[T,H,D] and K/V[N,Hkv,D]")
    tokens, heads, dim = q.shape
    rows, kv_heads, pool_dim = pool
    if pool_dim != dim or kv_heads <= 0 or heads <= 0 or heads % kv_heads:
        raise ValueError("K/V heads must divide the query heads and share their dimension")
    dtype = q.dtype
    if dtype not in _DTYPES or k_cache.dtype != dtype or v_cache.dtype != dtype:
        raise ValueError("FP16 or BF16 required, the same for every tensor")
    if dim < 16 or dim > 256 or dim % 16:
        raise ValueError("D must be in [16, 256] and divisible by 16")
    if page_size <= 0 or page_size % 16 or rows <= 0 or rows % page_size:
        raise ValueError("page_size must be a positive multiple of 16 and divide the pool's rows")
    if block_table.dim() != 2:
        raise ValueError("metadata shape mismatch")
    batch, width = block_table.shape
    if batch <= 0 or width <= 0 or cache_seqlens.shape != (batch,) or cu_seqlens_q.shape != (batch + 1,):
        raise ValueError("metadata shape mismatch")
    if not block_table.dtype == cache_seqlens.dtype == cu_seqlens_q.dtype == torch.int32:
        raise ValueError("page table, lengths and offsets must be int32")
    if width * page_size > (1 << 31) - 1 or tokens > (1 << 31) - 1 or rows > (1 << 31) - 1:
        raise ValueError("requires logical positions, tokens and pool rows to fit int32")
    device = q.get_device()  # -1 on the CPU
    if (device < 0 or k_cache.get_device() != device or v_cache.get_device() != device
            or block_table.get_device() != device or cache_seqlens.get_device() != device
            or cu_seqlens_q.get_device() != device):
        raise ValueError("every tensor must be on the same CUDA device")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous() and block_table.is_contiguous()
            and cache_seqlens.is_contiguous() and cu_seqlens_q.is_contiguous()):
        raise ValueError("kernel inputs must be contiguous")
    return tokens, heads, dim, kv_heads, rows, batch, width


def token_stride(x, name):
    """Elements from one token's row to the next of ``x`` [tokens, heads, dim]; each row itself is contiguous."""
    tokens, heads, dim = x.shape
    stride, head_stride, one = x.stride()
    if one != 1 or (head_stride != dim and heads > 1):
        raise ValueError(f"{name}: a token's heads must be contiguous")
    if tokens <= 1:
        return heads * dim
    if stride < heads * dim or stride % 8:
        raise ValueError(f"{name}: the token stride must be a multiple of 8 and cover the heads")
    return stride


def aligned(*tensors):
    """The data pointers; 16-byte aligned as the kernels' vector accesses and TMA need them."""
    pointers = [t.data_ptr() for t in tensors]
    if any([p & 15 for p in pointers]):
        raise ValueError("tensors must be 16-byte aligned")
    return pointers


def output_like(q, out):
    """``out``, or a new contiguous tensor of q's shape, and its token stride."""
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        return out, q.shape[1] * q.shape[2]
    if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
        raise ValueError("out must match q")
    return out, token_stride(out, "out")


def on_device(device, call, *args):
    """``call(*args)`` with CUDA device index ``device`` current."""
    if torch._C._cuda_getDevice() == device:
        return call(*args)
    with torch.cuda.device(device):
        return call(*args)


@functools.lru_cache(maxsize=256)
def _workspace_bytes(tokens, batch, heads, kv_heads, dim, page_size):
    p = _native.ChunkParams()
    p.tokens, p.batch, p.heads, p.kv_heads, p.head_dim = tokens, batch, heads, kv_heads, dim
    p.pool_rows = p.page_size = page_size
    p.table_width = 1
    p.q_stride = p.out_stride = heads * dim
    p.softmax_scale = 1.0
    return _native.chunk_workspace_size(p)


def _launch(params, nbytes, device):
    stream = _current_stream(device)
    # a graph keeps what it allocates while it is captured, and would outlive a kept workspace
    if nbytes > _KEPT_WORKSPACE_BYTES or torch.cuda.is_current_stream_capturing():
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
        _native.chunk_attention(params, workspace.data_ptr(), nbytes, stream)
        return
    with _KEPT.lock:
        workspace = _KEPT.get(("chunk", nbytes, device, stream), nbytes,
                              lambda: torch.empty(nbytes, dtype=torch.uint8, device=device))
        _native.chunk_attention(params, workspace.data_ptr(), nbytes, stream)


def paged_chunk_attention(q, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens_q, page_size, is_causal=True,
                          softmax_scale=None, out=None):
    """Attention of the new tokens over everything cached; returns ``out`` [T, H, D].

    ``q`` is [T, H, D] (each token's heads contiguous, any token stride that is a multiple of 8: a slice of a fused
    projection serves as it is), ``k_cache`` / ``v_cache`` [pool_rows, Hkv, D], ``block_table`` [B, W] int32,
    ``cache_seqlens`` [B] int32 (tokens in the cache with the new ones), ``cu_seqlens_q`` [B + 1] int32. Causal: the
    i-th of a request's n new tokens sees the first ``cache_seqlens - n + i + 1`` cached ones. Rows that see nothing and
    rows of no request are exact zeros. ``softmax_scale`` defaults to 1 / sqrt(D).
    """
    tokens, heads, dim, kv_heads, rows, batch, width = check_ragged(q, k_cache, v_cache, block_table, cache_seqlens,
                                                                    cu_seqlens_q, page_size)
    if heads > MAX_GROUP * kv_heads:
        raise ValueError(f"at most {MAX_GROUP} query heads per key head")
    scale = dim ** -0.5 if softmax_scale is None else float(softmax_scale)
    if not 0.0 < scale <= 1e30:
        raise ValueError("softmax_scale must be positive and finite")
    out, out_stride = output_like(q, out)
    q_stride = token_stride(q, "q")
    if not tokens:
        return out
    q_at, k_at, v_at, out_at = aligned(q, k_cache, v_cache, out)
    params = _PACK(q_at, k_at, v_at, block_table.data_ptr(), cache_seqlens.data_ptr(), cu_seqlens_q.data_ptr(), out_at,
                   tokens, rows, q_stride, out_stride, batch, heads, kv_heads, dim, width, page_size, _DTYPES[q.dtype],
                   1 if is_causal else 0, scale, 0, 0, 0)
    nbytes = _workspace_bytes(tokens, batch, heads, kv_heads, dim, page_size)
    on_device(q.get_device(), _launch, params, nbytes, q.get_device())
    return out
