"""Attention of a ragged batch of new tokens over a paged KV cache (``fgw_chunk_attention`` of ``libfgw_mha.so``).

FGW's ``mha_paged_decode`` takes one query length for the whole batch and as many key heads as query heads. A serving
step brings single tokens and prompt chunks together, grouped heads, and lengths that live on the device;
``paged_chunk_attention`` takes those as they are: query head h reads key head h // (heads // kv_heads), request b's
new tokens are rows ``cu_seqlens_q[b]`` to ``cu_seqlens_q[b + 1]``, and nothing is copied to the host.
"""
import torch

from fgw_b200 import _native
from fgw_b200.operators.mha.kernels.mha_paged_fwd_sm100 import _KEPT, _KEPT_WORKSPACE_BYTES, _current_stream

_DTYPES = {torch.float16: _native.DTYPE_FLOAT16, torch.bfloat16: _native.DTYPE_BFLOAT16}
MAX_GROUP = 128  # query heads that may share a key head


def check_ragged(q, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens_q, page_size):
    """Checks shared by the operators over a ragged batch and a paged cache; returns (tokens, heads, dim, kv_heads)."""
    if q.dim() != 3 or k_cache.dim() != 3 or v_cache.shape != k_cache.shape:
        raise ValueError("Expected q[T,H,D] and K/V[N,Hkv,D]")
    tokens, heads, dim = q.shape
    kv_heads = k_cache.shape[1]
    if k_cache.shape[2] != dim or kv_heads <= 0 or heads % kv_heads:
        raise ValueError("K/V heads must divide the query heads and share their dimension")
    if q.dtype not in _DTYPES or k_cache.dtype != q.dtype or v_cache.dtype != q.dtype:
        raise ValueError("FP16 or BF16 required, the same for every tensor")
    if dim < 16 or dim > 256 or dim % 16:
        raise ValueError("D must be in [16, 256] and divisible by 16")
    if page_size <= 0 or page_size % 16 or k_cache.shape[0] <= 0 or k_cache.shape[0] % page_size:
        raise ValueError("page_size must be a positive multiple of 16 and divide the pool's rows")
    batch = cache_seqlens.shape[0] if cache_seqlens.dim() == 1 else 0
    if (batch <= 0 or block_table.dim() != 2 or block_table.shape[0] != batch or block_table.shape[1] <= 0
            or cu_seqlens_q.shape != (batch + 1,)):
        raise ValueError("metadata shape mismatch")
    if not block_table.dtype == cache_seqlens.dtype == cu_seqlens_q.dtype == torch.int32:
        raise ValueError("page table, lengths and offsets must be int32")
    if block_table.shape[1] * page_size > (1 << 31) - 1:
        raise ValueError("requires logical positions to fit int32")
    device = q.device
    if not q.is_cuda or any(t.device != device for t in (k_cache, v_cache, block_table, cache_seqlens, cu_seqlens_q)):
        raise ValueError("every tensor must be on the same CUDA device")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous() and block_table.is_contiguous()
            and cache_seqlens.is_contiguous() and cu_seqlens_q.is_contiguous()):
        raise ValueError("kernel inputs must be contiguous")
    return tokens, heads, dim, kv_heads


def token_stride(x, name):
    """Elements from one token's row to the next of ``x`` [tokens, heads, dim]; each row itself is contiguous."""
    tokens, heads, dim = x.shape
    stride, head_stride, one = x.stride()
    if (one != 1 and dim > 1) or (head_stride != dim and heads > 1):
        raise ValueError(f"{name}: a token's heads must be contiguous")
    if tokens <= 1:
        return heads * dim
    if stride < heads * dim or stride % 8:
        raise ValueError(f"{name}: the token stride must be a multiple of 8 and cover the heads")
    return stride


def aligned(x, name):
    """The data pointer of ``x``; 16-byte aligned as the kernels' vector accesses and TMA need it."""
    at = x.data_ptr()
    if at % 16:
        raise ValueError(f"{name} must be 16-byte aligned")
    return at


def paged_chunk_attention(q, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens_q, page_size, is_causal=True,
                          softmax_scale=None, out=None):
    """Attention of the new tokens over everything cached; returns ``out`` [T, H, D].

    ``q`` is [T, H, D] (each token's heads contiguous, any token stride that is a multiple of 8: a slice of a fused
    projection serves as it is), ``k_cache`` / ``v_cache`` [pool_rows, Hkv, D], ``block_table`` [B, W] int32,
    ``cache_seqlens`` [B] int32 (tokens in the cache with the new ones), ``cu_seqlens_q`` [B + 1] int32. Causal: the
    i-th of a request's n new tokens sees the first ``cache_seqlens - n + i + 1`` cached ones. Rows that see nothing and
    rows of no request are exact zeros. ``softmax_scale`` defaults to 1 / sqrt(D).
    """
    tokens, heads, dim, kv_heads = check_ragged(q, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens_q,
                                                page_size)
    if heads // kv_heads > MAX_GROUP:
        raise ValueError(f"at most {MAX_GROUP} query heads per key head")
    scale = dim ** -0.5 if softmax_scale is None else float(softmax_scale)
    if not 0.0 < scale <= 1e30:
        raise ValueError("softmax_scale must be positive and finite")
    if out is None:
        out = torch.empty((tokens, heads, dim), dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
        raise ValueError("out must match q")
    if not tokens:
        return out
    p = _native.ChunkParams()
    p.q, p.k_cache, p.v_cache, p.out = (aligned(q, "q"), aligned(k_cache, "k_cache"), aligned(v_cache, "v_cache"),
                                        aligned(out, "out"))
    p.block_table, p.cache_seqlens = block_table.data_ptr(), cache_seqlens.data_ptr()
    p.cu_seqlens_q = cu_seqlens_q.data_ptr()
    p.tokens, p.pool_rows = tokens, k_cache.shape[0]
    p.q_stride, p.out_stride = token_stride(q, "q"), token_stride(out, "out")
    p.batch, p.heads, p.kv_heads, p.head_dim = cache_seqlens.shape[0], heads, kv_heads, dim
    p.table_width, p.page_size = block_table.shape[1], page_size
    p.dtype, p.causal, p.softmax_scale = _DTYPES[q.dtype], 1 if is_causal else 0, scale
    device = q.device.index
    nbytes = _native.chunk_workspace_size(p)
    with torch.cuda.device(device):
        stream = _current_stream(device)
        # a graph keeps what it allocates while it is captured, and would outlive a kept workspace
        if nbytes > _KEPT_WORKSPACE_BYTES or torch.cuda.is_current_stream_capturing():
            workspace = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
            _native.chunk_attention(p, workspace.data_ptr(), nbytes, stream)
        else:
            with _KEPT.lock:
                workspace = _KEPT.get(("chunk", nbytes, device, stream), nbytes,
                                      lambda: torch.empty(nbytes, dtype=torch.uint8, device=q.device))
                _native.chunk_attention(p, workspace.data_ptr(), nbytes, stream)
    return out
