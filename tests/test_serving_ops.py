"""Chunk attention, rotary append and the page-table operators against plain 64-bit restatements (oracle/serving.py).

Tolerances follow from the arithmetic. u is the type's unit roundoff (2^-8 BF16, 2^-11 FP16). Attention rounds each
softmax weight once to the type before it multiplies V (relative error u, the weights' sum taken over the rounded ones)
and the result once: |error| <= u (2 |out| + sum p |v|), plus 2^-25 per key and value for FP16 weights below its
normal range, plus FP32 terms (2^-16 relative is ample for dots of up to 256 products and 2^x). Rotation in FP32
rounds once: u |out| + 2^-22 (|x| + |y|). Tables, lengths and copied bytes are exact.
"""
import math

import numpy as np
import pytest
import torch

from oracle import serving

ROUNDOFF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def ragged(new, held, page, seed, spare_pages=3, spare_width=1):
    """(table, lens, cu) with every request's pages at random places of the pool; dead entries are -1."""
    rng = np.random.default_rng(seed)
    counts = [-(-n // page) for n in held]
    pages = sum(counts) + spare_pages
    ids = rng.permutation(pages)
    table = np.full((len(held), max(max(counts), 1) + spare_width), -1, dtype=np.int32)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = ids[at:at + c]
        at += c
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    return table, np.array(held, dtype=np.int32), cu, pages


def values(shape, dtype, seed, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * scale).to(dtype)


def wide(x):
    return x.double().cpu().numpy()


# --- chunk attention ------------------------------------------------------------------------------------------------
# (name, new tokens, tokens held with them, heads, kv heads, dim, page, causal)
ATTEND = [
    ("one_token", [1], [1], 2, 2, 64, 16, True),
    ("one_token_long", [1], [700], 8, 1, 128, 64, True),
    ("tokens", [1, 1, 1, 1, 1], [129, 128, 127, 1, 260], 8, 2, 128, 16, True),
    ("empty_requests", [0, 3, 0, 5, 0], [40, 3, 0, 300, 5], 4, 4, 64, 32, True),
    ("rows_without_keys", [9, 4, 40], [5, 0, 33], 4, 2, 128, 16, True),
    ("group_of_three", [70, 1, 131], [70, 200, 389], 6, 2, 64, 48, True),
    ("group_of_seven", [37, 2], [300, 257], 7, 1, 96, 16, True),
    ("no_group", [130, 64], [513, 64], 3, 3, 128, 128, True),
    ("wide_head", [33, 1, 5], [150, 259, 64], 4, 1, 256, 64, True),
    ("wide_head_odd", [140], [300], 2, 2, 208, 16, True),
    ("narrow_head", [129, 7], [400, 64], 4, 2, 16, 16, True),
    ("unmasked", [7, 1, 20], [129, 0, 256], 8, 2, 128, 32, False),
    ("unmasked_wide", [6, 3], [101, 64], 8, 1, 256, 48, False),
    ("big_group", [2, 3], [65, 200], 64, 1, 64, 16, True),
    ("group_of_128", [3], [140], 128, 1, 32, 16, True),
    ("long_cache", [2, 1], [4099, 2500], 4, 1, 128, 256, True),
    ("many_rows", [1] * 70, list(range(1, 71)), 4, 2, 64, 16, True),
    ("long_chunk", [600], [600], 4, 2, 64, 128, True),
]


def attend_case(case, dtype, seed=1, scale_k=1.0):
    _, new, held, heads, kv_heads, dim, page, _ = case
    table, lens, cu, pages = ragged(new, held, page, seed)
    q = values((sum(new), heads, dim), dtype, seed + 1)
    k = values((pages * page, kv_heads, dim), dtype, seed + 2, scale_k)
    v = values((pages * page, kv_heads, dim), dtype, seed + 3)
    return q, k, v, table, lens, cu


def dead_rows(table, lens, page, rows):
    """Pool rows that hold no token of any request."""
    live = {int(table[b, p // page]) * page + p % page for b in range(len(lens)) for p in range(int(lens[b]))}
    return [r for r in range(rows) if r not in live]


def on_gpu(*arrays):
    return [torch.as_tensor(a, device="cuda") for a in arrays]


def check_attention(got, q, k, v, table, lens, cu, page, causal, scale):
    want, spread = serving.chunk_attention(wide(q), wide(k), wide(v), table, lens, cu, page, causal, scale)
    u = ROUNDOFF[q.dtype]
    bound = u * (2 * np.abs(want) + spread) + 2.0 ** -16 * spread + 1e-6
    if q.dtype == torch.float16:
        bound = bound + 2.0 ** -25 * max(int(lens.max()), 1) * float(np.nanmax(np.abs(wide(v))))
    err = np.abs(wide(got) - want)
    assert np.isfinite(wide(got)).all()
    assert (err <= bound).all(), (float((err / bound).max()), float(err.max()))
    empty = spread.sum(-1) == 0
    assert (wide(got)[empty] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("case", ATTEND, ids=[c[0] for c in ATTEND])
def test_chunk_attention(case, dtype):
    from fgw_b200.operators.mha.chunk_attention import paged_chunk_attention
    _, _, _, _, _, dim, page, causal = case
    q, k, v, table, lens, cu = attend_case(case, dtype)
    dead = dead_rows(table, lens, page, k.shape[0])
    k_nan, v_nan = k.clone(), v.clone()
    k_nan[dead], v_nan[dead] = float("nan"), float("inf")  # what no request holds may be anything
    out = torch.full(q.shape, float("nan"), dtype=dtype, device="cuda")
    got = paged_chunk_attention(q.cuda(), k_nan.cuda(), v_nan.cuda(), *on_gpu(table, lens, cu), page, is_causal=causal,
                                out=out)
    assert got is out
    k[dead], v[dead] = 0, 0
    check_attention(got, q, k, v, table, lens, cu, page, causal, dim ** -0.5)


def torch_attention(q, k, v, table, lens, cu, page, causal):
    """(out, spread) as oracle/serving.py gives them, in 64 bits with torch on the GPU, for the larger shapes."""
    q, k, v = q.double(), k.double(), v.double()
    out, spread = torch.zeros_like(q), torch.zeros_like(q)
    group = q.shape[1] // k.shape[1]
    for b, length in enumerate(lens.tolist()):
        first, n = int(cu[b]), int(cu[b + 1] - cu[b])
        at = torch.arange(length, device="cuda")
        rows = torch.as_tensor(table[b], device="cuda").long()[at // page] * page + at % page
        seen = (length - n + 1 + torch.arange(n, device="cuda")) if causal else torch.full((n,), length, device="cuda")
        hidden = at >= seen[:, None]
        for h in range(q.shape[1]):
            keys, values = k[rows, h // group], v[rows, h // group]
            s = (q[first:first + n, h] @ keys.T * q.shape[2] ** -0.5).masked_fill(hidden, -math.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0)  # rows without keys
            out[first:first + n, h], spread[first:first + n, h] = p @ values, p @ values.abs()
    return out, spread


# batches with several items per CTA: chunks that need one tile and two, requests of both kernels, items cut and whole
LARGE = [
    # (name, new tokens, held, heads, kv heads, dim, page, causal)
    ("prompts", [70, 300, 1, 128, 257, 1000, 20, 129, 511, 64], [170, 310, 900, 128, 700, 1300, 20, 1129, 600, 64],
     16, 16, 128, 128, True),
    ("narrow", [400, 30, 1, 130, 257, 1, 90, 333, 9], [500, 3000, 1200, 130, 2000, 1, 90, 1500, 700], 24, 8, 64, 32, True),
    ("wide", [100, 33, 1, 200, 65, 31], [1100, 33, 400, 600, 900, 1000], 8, 2, 256, 64, True),
    ("wide_odd", [100, 33, 1, 200, 65, 31], [1100, 33, 400, 600, 900, 1000], 6, 2, 176, 48, True),
    ("one_long", [1500], [6000], 8, 2, 128, 64, True),
    ("tiles_of_one", [40] * 60, [40 + 37 * i % 700 for i in range(60)], 8, 4, 64, 16, True),
    ("tiles_of_one_128", [40] * 60, [40 + 37 * i % 700 for i in range(60)], 8, 4, 128, 16, True),
    ("unmasked", [77, 300, 5, 150], [1000, 300, 700, 2222], 8, 4, 96, 32, False),
    ("decode_32_rows", [7] * 30, [7 + 113 * i % 2000 for i in range(30)], 8, 2, 128, 64, True),
    ("decode_64_rows", [5, 1, 3, 5, 2] * 6, [5 + 113 * i % 2000 for i in range(30)], 24, 2, 80, 64, True),
    ("decode_wide_32_rows", [3] * 20, [3 + 113 * i % 2000 for i in range(20)], 8, 1, 256, 48, False),
    ("decode_wide_64_rows", [8, 5, 1, 7] * 6, [8 + 113 * i % 2000 for i in range(24)], 8, 1, 256, 48, False),
    ("decode_wide_odd_64_rows", [5, 8, 2] * 7, [8 + 113 * i % 1500 for i in range(21)], 16, 2, 176, 16, True),
    ("rounds_by_load", [90 + 53 * i % 400 for i in range(40)], [500 + 211 * i % 1700 for i in range(40)], 8, 8, 128, 64, True),
    ("rounds_by_load_narrow", [30 + 53 * i % 300 for i in range(40)], [400 + 211 * i % 1700 for i in range(40)], 6, 6, 48, 32,
     True),
    ("group_over_decode", [1, 2, 1, 30, 1], [900, 40, 3000, 600, 1], 160, 2, 64, 32, True),
    ("long_among_tokens", [1] * 40 + [37], [50 + 97 * i % 3000 for i in range(40)] + [2000], 8, 2, 128, 16, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("case", LARGE, ids=[c[0] for c in LARGE])
def test_chunk_attention_many_items(case, dtype):
    from fgw_b200.operators.mha.chunk_attention import paged_chunk_attention
    _, new, held, _, _, _, page, causal = case
    held = [max(h, n) for h, n in zip(held, new)]
    q, k, v, table, lens, cu = attend_case((*case[:2], held, *case[3:]), dtype, seed=21)
    args = [q.cuda(), k.cuda(), v.cuda()]
    got = [paged_chunk_attention(*args, *on_gpu(table, lens, cu), page, is_causal=causal) for _ in range(3)]
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    want, spread = torch_attention(*args, table, lens, cu, page, causal)
    bound = ROUNDOFF[dtype] * (2 * want.abs() + spread) + 2.0 ** -16 * spread + 1e-6
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25 * max(held) * float(v.abs().max())
    err = (got[0].double() - want).abs()
    assert bool((err <= bound).all()), (float((err / bound).max()), float(err.max()))


@pytest.mark.gpu
def test_chunk_attention_reports_no_device_error_and_zeroes_rows_of_no_request():
    import ctypes

    from fgw_b200 import _native
    q, k, v, table, lens, cu = attend_case(("x", [40, 1, 300], [400, 20, 600], 4, 2, 128, 16, True), torch.bfloat16)
    q = torch.cat([q[:3], q, q[:5]])  # three rows before the first request, five after the last
    args = [q.cuda(), k.cuda(), v.cuda(), *on_gpu(table, lens, cu + 3)]
    out = torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda")
    p = _native.ChunkParams()  # by the C ABI, whose caller has the workspace to read the status from
    for name, t in zip(("q", "k_cache", "v_cache", "block_table", "cache_seqlens", "cu_seqlens_q", "out"), (*args, out)):
        setattr(p, name, t.data_ptr())
    for name, value in dict(tokens=q.shape[0], pool_rows=k.shape[0], q_stride=512, out_stride=512, batch=3, heads=4,
                            kv_heads=2, head_dim=128, table_width=table.shape[1], page_size=16,
                            dtype=_native.DTYPE_BFLOAT16, causal=1, softmax_scale=128 ** -0.5).items():
        setattr(p, name, value)
    size = ctypes.c_size_t()
    lib, stream = _native.library(), torch.cuda.current_stream().cuda_stream
    assert lib.fgw_chunk_workspace_size(ctypes.byref(p), ctypes.byref(size)) == 0
    workspace = torch.full((size.value,), 255, dtype=torch.uint8, device="cuda")  # whatever it holds
    assert lib.fgw_chunk_attention(ctypes.byref(p), workspace.data_ptr(), size.value, stream) == 0
    assert _native.read_error(workspace.data_ptr(), stream) == (_native.OK, 0)
    assert not out[:3].any() and not out[-5:].any()
    check_attention(out[3:-5], q[3:-5], k, v, table, lens, cu, 16, True, 128 ** -0.5)


@pytest.mark.gpu
def test_chunk_attention_over_a_pool_past_32_bits():
    """Cache rows whose element and byte offsets need more than 32 bits."""
    from fgw_b200.operators.mha.chunk_attention import paged_chunk_attention
    page, kv_heads, dim = 64, 8, 128
    pages = (5 << 30) // (page * kv_heads * dim)  # 5 G elements
    k = torch.zeros((pages * page, kv_heads, dim), dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    q, small_k, small_v, table, lens, cu = attend_case(("x", [1, 200], [300, 500], 8, kv_heads, dim, page, True),
                                                       torch.bfloat16)
    rows = small_k.shape[0]
    k[-rows:], v[-rows:] = small_k.cuda(), small_v.cuda()
    moved = np.where(table >= 0, table + pages - rows // page, -1).astype(np.int32)
    got = paged_chunk_attention(q.cuda(), k, v, *on_gpu(moved, lens, cu), page)
    want = paged_chunk_attention(q.cuda(), small_k.cuda(), small_v.cuda(), *on_gpu(table, lens, cu), page)
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_chunk_attention_peaked_and_scaled():
    """Scores far apart (weights underflow, the running maximum jumps) and another softmax scale."""
    from fgw_b200.operators.mha.chunk_attention import paged_chunk_attention
    case = ("peaked", [90, 1, 3], [700, 640, 131], 8, 2, 128, 32, True)
    for scale in (0.3, 1e-4):
        q, k, v, table, lens, cu = attend_case(case, torch.bfloat16, seed=5, scale_k=8.0)
        got = paged_chunk_attention(*(x.cuda() for x in (q, k, v)), *on_gpu(table, lens, cu), 32, softmax_scale=scale)
        # at scores of a few hundred, FP32 leaves 2^-16 of them in the exponent
        want, spread = serving.chunk_attention(wide(q), wide(k), wide(v), table, lens, cu, 32, True, scale)
        size = scale * float(np.abs(wide(q)).sum(-1).max()) * 40
        bound = 2.0 ** -8 * (2 * np.abs(want) + spread) + (2.0 ** -16 + size * 2.0 ** -22) * spread + 1e-6
        assert (np.abs(wide(got) - want) <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (4, 4, 64), (4, 1, 256)])
def test_chunk_attention_strides_streams_and_repeats(heads, kv_heads, dim):
    """A slice of a fused projection, an output slice, another stream than the default, and the same bits each time."""
    from fgw_b200.operators.mha.chunk_attention import paged_chunk_attention
    new, held, page = [150, 1, 0, 33], [1500, 4000, 9, 33], 64
    q, k, v, table, lens, cu = attend_case(("x", new, held, heads, kv_heads, dim, page, True), torch.bfloat16, seed=9)
    fused = torch.full((sum(new), heads + 2 * kv_heads, dim), float("nan"), dtype=q.dtype, device="cuda")
    fused[:, kv_heads:kv_heads + heads] = q.cuda()
    args = [k.cuda(), v.cuda(), *on_gpu(table, lens, cu), page]
    first = paged_chunk_attention(q.cuda(), *args)
    check_attention(first, q, k, v, table, lens, cu, page, True, dim ** -0.5)
    room = torch.zeros((sum(new), heads + 1, dim), dtype=q.dtype, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = paged_chunk_attention(fused[:, kv_heads:kv_heads + heads], *args, out=room[:, :heads])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, second) and not room[:, heads:].any()
    for _ in range(5):
        assert torch.equal(first, paged_chunk_attention(q.cuda(), *args))


@pytest.mark.gpu
def test_chunk_attention_in_a_graph_with_other_lengths():
    """Lengths are device data: a captured call serves other lengths of the same shapes."""
    from fgw_b200.operators.mha.chunk_attention import paged_chunk_attention
    case = ("graph", [1, 1, 60], [500, 20, 300], 8, 2, 128, 16, True)
    q, k, v, table, lens, cu = attend_case(case, torch.bfloat16, seed=12)
    args = [q.cuda(), k.cuda(), v.cuda(), *on_gpu(table, lens, cu)]
    out = torch.empty_like(args[0])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        paged_chunk_attention(*args, 16, out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            paged_chunk_attention(*args, 16, out=out)
    for other in ([500, 20, 300], [1, 17, 60], [33, 0, 10]):
        lens2 = np.array(other, dtype=np.int32)
        args[4].copy_(torch.from_numpy(lens2))
        graph.replay()
        torch.cuda.synchronize()
        check_attention(out, q, k, v, table, lens2, cu, 16, True, 128 ** -0.5)


# --- rotary append --------------------------------------------------------------------------------------------------
ROTARY = [
    # (name, new, held, heads, kv heads, dim, rotary, interleaved, page)
    ("tokens", [1, 1, 1], [1, 70, 300], 8, 2, 128, 128, False, 16),
    ("tokens_interleaved", [1, 1, 1], [1, 70, 300], 8, 2, 128, 128, True, 16),
    ("chunk", [130, 0, 17, 1], [200, 9, 17, 40], 4, 4, 64, 64, False, 32),
    ("part", [40, 3], [90, 3], 6, 3, 128, 32, False, 48),
    ("part_interleaved", [40, 3], [90, 3], 6, 3, 80, 26, True, 48),
    ("odd_half", [25, 1], [99, 5], 4, 1, 256, 46, False, 64),
    ("pair", [25, 1], [99, 5], 4, 1, 16, 2, True, 64),
    ("many_requests", [1] * 200 + [3], list(range(1, 201)) + [64], 2, 1, 64, 64, False, 16),
    ("many_tokens", [3000, 2500], [3000, 2600], 2, 1, 128, 64, True, 128),
    ("tokens_before_the_cache", [12, 5], [7, 5], 4, 2, 64, 64, False, 16),
    ("positions_past_the_angles", [12, 5], [400, 5], 4, 2, 64, 32, True, 16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("case", ROTARY, ids=[c[0] for c in ROTARY])
def test_rotary_append(case, dtype):
    from fgw_b200.operators.mha.rotary_append import rotary_append, rotary_table
    name, new, held, heads, kv_heads, dim, rotary, interleaved, page = case
    table, lens, cu, pages = ragged(new, held, page, 3)
    fused = values((sum(new) + 3, heads + 2 * kv_heads, dim), dtype, 4)  # three rows of no request
    kc, vc = values((pages * page, kv_heads, dim), dtype, 5), values((pages * page, kv_heads, dim), dtype, 6)
    cos_sin = rotary_table(395 if name.startswith("positions") else max(held), rotary, device="cpu")
    q, k, v = fused[:, :heads], fused[:, heads:heads + kv_heads], fused[:, heads + kv_heads:]
    want = serving.rotary_append(wide(q), wide(k), wide(v), wide(kc), wide(vc), table, lens, cu, cos_sin.numpy(), page,
                                 interleaved)
    gpu, kg, vg = fused.cuda(), kc.cuda(), vc.cuda()
    views = gpu[:, :heads], gpu[:, heads:heads + kv_heads], gpu[:, heads + kv_heads:]
    got = rotary_append(*views, kg, vg, *on_gpu(table, lens, cu), cos_sin.cuda(), page, interleaved=interleaved)
    largest = float(fused.float().abs().max())
    for x, w in zip((got, kg, vg), want):
        bound = ROUNDOFF[dtype] * np.abs(w) + 2.0 ** -21 * largest
        assert (np.abs(wide(x) - w) <= bound).all()
    assert torch.equal(gpu, fused.cuda())  # the projection is not written
    assert torch.equal(vg.cpu(), torch.from_numpy(want[2]).to(dtype))
    # into the queries' own memory, the same bits
    kg2, vg2 = kc.cuda(), vc.cuda()
    again = rotary_append(*views, kg2, vg2, *on_gpu(table, lens, cu), cos_sin.cuda(), page, interleaved=interleaved,
                          out=views[0])
    assert again.data_ptr() == gpu.data_ptr()
    assert torch.equal(again, got) and torch.equal(kg, kg2) and torch.equal(vg, vg2)


@pytest.mark.gpu
def test_rotary_append_skips_pages_outside_the_pool():
    from fgw_b200.operators.mha.rotary_append import rotary_append, rotary_table
    new, held, page = [6, 4], [6, 20], 16
    table, lens, cu, pages = ragged(new, held, page, 3)
    table[0, 0], table[1, 1] = pages, -1
    x = values((10, 6, 64), torch.float16, 4).cuda()
    kc, vc = values((pages * page, 2, 64), torch.float16, 5).cuda(), values((pages * page, 2, 64), torch.float16, 6).cuda()
    before = kc.clone(), vc.clone()
    cos_sin = rotary_table(20, 64)
    got = rotary_append(x[:, :2], x[:, 2:4], x[:, 4:], kc, vc, *on_gpu(table, lens, cu), cos_sin, page)
    assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])
    assert got.abs().sum(-1).min() > 0  # the queries turn all the same


def test_rotary_table_scalings():
    plain = _table(64, 32)
    pairs = np.arange(16)
    angle = np.arange(64)[:, None] * 10000.0 ** (-pairs / 16.0)
    assert np.allclose(plain, np.concatenate([np.cos(angle), np.sin(angle)], 1), atol=2e-7)
    # linear: position 2 p of the scaled table is position p of the plain one
    assert np.array_equal(_table(64, 32, scaling="linear", factor=2.0)[::2], plain[:32])
    # ntk: the fastest pair stays, the slowest slows by the factor
    ntk = _table(64, 32, scaling="ntk", factor=4.0)
    assert np.array_equal(ntk[:, 0], plain[:, 0])
    slowest = 10000.0 ** (-15 / 16.0)
    assert np.allclose(ntk[:, 31], np.sin(np.arange(64) * slowest / 4.0), atol=1e-6)
    # yarn: fast pairs stay, slow ones are divided, all grow by the attention factor
    yarn = _table(64, 32, scaling="yarn", factor=4.0, original_positions=4096)
    size = 0.1 * math.log(4.0) + 1.0
    assert np.allclose(yarn[:, 0], plain[:, 0] * size, atol=1e-6)
    assert np.allclose(yarn[:, 31], np.sin(np.arange(64) * slowest / 4.0) * size, atol=1e-6)
    assert np.allclose(_table(64, 32, scaling="yarn", factor=4.0, original_positions=4096, attention_factor=1.0)[:, 0],
                       plain[:, 0], atol=1e-6)


def _table(*args, **kwargs):
    from fgw_b200.operators.mha.rotary_append import rotary_table
    return rotary_table(*args, device="cpu", **kwargs).numpy().astype(np.float64)


# --- page operators -------------------------------------------------------------------------------------------------
def page_state(held, page, seed, spare, row=(2, 16), pools=3, dtype=torch.float16):
    table, lens, _, pages = ragged([0] * len(held), held, page, seed, spare_pages=spare, spare_width=2)
    stores = [values((pages * page, *row), dtype, seed + 10 + i) for i in range(pools)]
    return table, lens, pages, stores


FORKS = [
    # (name, held, parents, reserve (None: none), page, spare pages)
    ("keep", [5, 16, 0, 33], [0, 1, 2, 3], None, 16, 4),
    ("beam", [5, 40, 0, 33, 16], [1, 1, 3, 1, 4], [41, 49, 40, 41, 17], 16, 20),
    ("swap", [20, 40], [1, 0], None, 16, 0),
    ("free_all", [20, 40, 1], [-1, -1, -1], [5, 5, 5], 16, 0),
    ("free_and_reserve", [20, 40, 1], [-1, 7, 2], [50, 50, 48], 16, 0),
    ("reuse_the_freed", [64, 64], [1, 1], [80, 65], 16, 0),
    ("whole_pages", [32, 48], [1, 1], None, 16, 0),
    ("too_few", [20, 40, 1], [1, 1, 1], [60, 60, 64], 16, 1),
    ("empty_parents", [0, 0, 7], [0, 0, 1], [1, 0, 33], 16, 8),
    ("past_the_width", [20, 4], [0, 1], [500, 5], 16, 8),
    ("shorter_than_held", [20, 40], [0, 0], [1, 1], 16, 8),
    ("one_row", [31], [0], [32], 16, 1),
    ("odd_page", [100, 7, 50], [0, 0, 2], [111, 1, 51], 7, 9),
    ("many_rows", [17 * i % 90 for i in range(300)], [i * i % 301 - 1 for i in range(300)],
     [17 * i % 100 for i in range(300)], 16, 1500),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", FORKS, ids=[c[0] for c in FORKS])
def test_fork_pages(case):
    from fgw_b200.operators.mha.page_ops import fork_pages
    _, held, parents, reserve, page, spare = case
    table, lens, pages, stores = page_state(held, page, 2, spare)
    parents = np.array(parents, dtype=np.int32)
    reserve = None if reserve is None else np.array(reserve, dtype=np.int32)
    want_table, want_lens, want_status, copies = serving.fork_pages(table, lens, parents, reserve, page, pages)
    pools = [s.cuda() for s in stores]
    args = on_gpu(table, lens, parents)
    got = fork_pages(pools, *args, page, reserve_seqlens=None if reserve is None else torch.from_numpy(reserve).cuda())
    assert tuple(got[2].tolist()) == want_status
    assert np.array_equal(got[0].cpu().numpy(), want_table)
    assert np.array_equal(got[1].cpu().numpy(), want_lens)
    for pool, store in zip(pools, stores):
        assert torch.equal(pool.cpu(), torch.from_numpy(serving.copy_rows(store.numpy(), copies, page)))
    assert np.array_equal(args[0].cpu().numpy(), table) and np.array_equal(args[1].cpu().numpy(), lens)


@pytest.mark.gpu
def test_fork_pages_shares_pages_outside_the_pool_untouched():
    from fgw_b200.operators.mha.page_ops import fork_pages
    table, lens, pages, stores = page_state([20, 40], 16, 2, 6)
    table[0, 1], table[1, 0] = pages + 3, -5
    parents = np.array([0, 0], dtype=np.int32)
    want = serving.fork_pages(table, lens, parents, None, 16, pages)
    pools = [s.cuda() for s in stores]
    got = fork_pages(pools, *on_gpu(table, lens, parents), 16)
    assert np.array_equal(got[0].cpu().numpy(), want[0]) and tuple(got[2].tolist()) == want[2]
    assert all(torch.equal(p.cpu(), s) for p, s in zip(pools, stores))  # the only copy's source is outside


COMPACTS = [
    ("empty", [0, 0], 16, 5, 1), ("one", [3], 16, 9, 3), ("full", [40, 70], 16, 0, 2), ("sparse", [40, 70, 0, 9], 16, 40, 2),
    ("odd_page", [40, 70, 0, 9], 7, 40, 3), ("block_edges", [16 * 40, 16 * 31, 5], 16, 1200, 1),
    ("many", [37 * i % 200 for i in range(150)], 16, 3000, 2),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", COMPACTS, ids=[c[0] for c in COMPACTS])
def test_compact_pages(case):
    from fgw_b200.operators.mha.page_ops import compact_pages
    _, held, page, spare, pools = case
    table, lens, pages, stores = page_state(held, page, 8, spare, pools=pools)
    if len(held) > 2:
        table[2, :1] = table[1, :1]  # a shared page
        lens[2] = max(int(lens[2]), 1)
    want_table, want_status, copies = serving.compact_pages(table, lens, page, pages)
    gpu = [s.cuda() for s in stores]
    got_table, status = compact_pages(gpu, *on_gpu(table, lens), page)
    assert tuple(status.tolist()) == want_status
    assert np.array_equal(got_table.cpu().numpy(), want_table)
    for pool, store in zip(gpu, stores):
        assert torch.equal(pool.cpu(), torch.from_numpy(serving.copy_rows(store.numpy(), copies, page)))


@pytest.mark.gpu
@pytest.mark.parametrize("pools,row", [(1, (8,)), (300, (1, 16)), (2, (8, 128))])
def test_copy_pages(pools, row):
    from fgw_b200.operators.mha.page_ops import copy_pages
    page, pages = 5, 40
    stores = [values((pages * page, *row), torch.bfloat16, i) for i in range(pools)]
    src = np.array([3, 39, 0, 40, -1, 7], dtype=np.int32)
    dst = np.array([10, 11, 38, 12, 13, 400], dtype=np.int32)
    gpu = [s.cuda() for s in stores]
    copy_pages(gpu, *on_gpu(src, dst), page)
    copies = [(3, 10, page), (39, 11, page), (0, 38, page)]
    for pool, store in zip(gpu, stores):
        want = serving.copy_rows(store.view(torch.int16).numpy(), copies, page)
        assert np.array_equal(pool.cpu().view(torch.int16).numpy(), want)
    copy_pages(gpu, *on_gpu(src[:0], dst[:0]), page)


@pytest.mark.gpu
def test_copies_past_32_bits_of_bytes():
    """Pages whose byte offsets need more than 32 bits."""
    from fgw_b200.operators.mha.page_ops import copy_pages
    page, row = 64, 8 * 128
    pages = (9 << 30) // (page * row * 2)
    pool = torch.zeros((pages * page, row), dtype=torch.bfloat16, device="cuda")
    pool[-page:] = 3.0
    copy_pages([pool], *on_gpu(np.array([pages - 1], dtype=np.int32), np.array([pages // 2], dtype=np.int32)), page)
    assert (pool[pages // 2 * page:(pages // 2 + 1) * page] == 3.0).all()
    assert pool.float().sum().item() == 2 * 3.0 * page * row


# --- one step, end to end -------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_a_serving_step():
    """fork -> append -> attend -> compact -> attend: the second attention reads the moved pages."""
    from fgw_b200.operators.mha.chunk_attention import paged_chunk_attention
    from fgw_b200.operators.mha.page_ops import compact_pages, fork_pages
    from fgw_b200.operators.mha.rotary_append import rotary_append, rotary_table
    page, heads, kv_heads, dim = 16, 4, 2, 64
    held, new = [40, 33, 16, 0], [1, 1, 5, 0]
    table, lens, _, pages = ragged([0] * 4, held, page, 2, spare_pages=12, spare_width=2)
    kc, vc = (values((pages * page, kv_heads, dim), torch.bfloat16, s) for s in (3, 4))
    parents = np.array([0, 0, 2, -1], dtype=np.int32)
    after = np.array([41, 41, 21, 0], dtype=np.int32)
    pools = [kc.cuda(), vc.cuda()]
    table2, lens2, status = fork_pages(pools, *on_gpu(table, lens, parents), page, reserve_seqlens=on_gpu(after)[0])
    assert status[0] <= status[1]
    lens2 += torch.tensor(new, dtype=torch.int32, device="cuda")
    assert lens2.tolist() == after.tolist()
    x = values((sum(new), heads + 2 * kv_heads, dim), torch.bfloat16, 6).cuda()
    cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda")
    cos_sin = rotary_table(64, dim)
    q = rotary_append(x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:], *pools, table2, lens2, cu,
                      cos_sin, page)
    out = paged_chunk_attention(q, *pools, table2, lens2, cu, page)
    check_attention(out, q, *pools, table2.cpu().numpy(), after, cu.cpu().numpy(), page, True, dim ** -0.5)
    table3, status = compact_pages(pools, table2, lens2, page)
    assert int(table3.max()) < int(status[0])
    assert torch.equal(out, paged_chunk_attention(q, *pools, table3, lens2, cu, page))


# --- refusals -------------------------------------------------------------------------------------------------------
def _attend_args(device="cpu"):
    return dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16, device=device),
                k_cache=torch.zeros(64, 2, 64, dtype=torch.bfloat16, device=device),
                v_cache=torch.zeros(64, 2, 64, dtype=torch.bfloat16, device=device),
                block_table=torch.zeros(2, 2, dtype=torch.int32, device=device),
                cache_seqlens=torch.zeros(2, dtype=torch.int32, device=device),
                cu_seqlens_q=torch.zeros(3, dtype=torch.int32, device=device), page_size=16)


REFUSED = [
    dict(q=torch.zeros(3, 4, 64)), dict(q=torch.zeros(3, 256, dtype=torch.bfloat16)),
    dict(q=torch.zeros(3, 3, 64, dtype=torch.bfloat16)), dict(q=torch.zeros(3, 4, 72, dtype=torch.bfloat16)),
    dict(k_cache=torch.zeros(64, 2, 64, dtype=torch.float16)), dict(v_cache=torch.zeros(48, 2, 64, dtype=torch.bfloat16)),
    dict(page_size=24), dict(page_size=0), dict(page_size=128), dict(block_table=torch.zeros(3, 2, dtype=torch.int32)),
    dict(block_table=torch.zeros(2, 2, dtype=torch.int64)), dict(cache_seqlens=torch.zeros(3, dtype=torch.int32)),
    dict(cu_seqlens_q=torch.zeros(2, dtype=torch.int32)), dict(),  # the last: not on a CUDA device
]


@pytest.mark.parametrize("override", REFUSED, ids=range(len(REFUSED)))
def test_ragged_operators_refuse(override):
    from fgw_b200.operators.mha.chunk_attention import paged_chunk_attention
    from fgw_b200.operators.mha.rotary_append import rotary_append
    args = {**_attend_args(), **override}
    with pytest.raises(ValueError):
        paged_chunk_attention(**args)
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        rotary_append(k=k, v=k, cos_sin=torch.zeros(9, 64), **args)


@pytest.mark.gpu
def test_ragged_operators_refuse_on_the_gpu():
    from fgw_b200.operators.mha.chunk_attention import paged_chunk_attention
    from fgw_b200.operators.mha.rotary_append import rotary_append
    args = _attend_args("cuda")
    paged_chunk_attention(**args)
    flat = torch.zeros(3 * 4 * 64 + 8, dtype=torch.bfloat16, device="cuda")
    for bad in (dict(q=flat[4:4 + 768].view(3, 4, 64)), dict(q=flat[:768].view(3, 64, 4).transpose(1, 2)),
                dict(softmax_scale=0.0), dict(softmax_scale=math.inf), dict(softmax_scale=math.nan),
                dict(out=torch.zeros(3, 4, 64, device="cuda")), dict(k_cache=args["k_cache"].cpu()),
                dict(q=torch.zeros(3, 258, 64, dtype=torch.bfloat16, device="cuda")),
                dict(q=torch.zeros(3, 260, dtype=torch.bfloat16, device="cuda")[:, :256].view(3, 4, 64))):
        with pytest.raises(ValueError):
            paged_chunk_attention(**{**args, **bad})
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device="cuda")
    angles = torch.zeros(9, 64, device="cuda")
    rotary_append(k=k, v=k, cos_sin=angles, **args)
    for bad in (dict(k=k[:2]), dict(v=k.half()), dict(cos_sin=angles[:, :33]), dict(cos_sin=angles.double()),
                dict(cos_sin=torch.zeros(9, 66, device="cuda")), dict(cos_sin=angles.cpu())):
        with pytest.raises(ValueError):
            rotary_append(**{**dict(k=k, v=k, cos_sin=angles), **args, **bad})


def test_rotary_table_refuses():
    from fgw_b200.operators.mha.rotary_append import rotary_table
    for bad in (dict(positions=0), dict(rotary_dim=7), dict(rotary_dim=0), dict(scaling="other"), dict(base=1.0),
                dict(factor=2.0), dict(scaling="linear", factor=0.5), dict(scaling="yarn", factor=2.0),
                dict(attention_factor=1.0)):
        with pytest.raises(ValueError):
            rotary_table(**{**dict(positions=4, rotary_dim=8, device="cpu"), **bad})


def test_page_operators_refuse():
    from fgw_b200.operators.mha.page_ops import compact_pages, copy_pages, fork_pages
    table, lens = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    pool = torch.zeros(64, 2, 16, dtype=torch.bfloat16)
    for pools, page in (([], 16), ([pool], 0), ([pool], 48), ([pool, pool[:32]], 16), ([pool[:, :1, :4]], 16),
                        ([pool], 16)):  # the last: not on a CUDA device
        with pytest.raises(ValueError):
            fork_pages(pools, table, lens, lens, page)
        with pytest.raises(ValueError):
            compact_pages(pools, table, lens, page)
        with pytest.raises(ValueError):
            copy_pages(pools, lens, lens, page)


@pytest.mark.gpu
def test_page_operators_refuse_on_the_gpu():
    from fgw_b200.operators.mha.page_ops import compact_pages, copy_pages, fork_pages
    pool = [torch.zeros(64, 2, 16, dtype=torch.bfloat16, device="cuda")]
    table, lens = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in ((table, lens[:1], lens), (table.long(), lens, lens), (table, lens, lens.long()), (table, lens, lens[:1]),
                (table.cpu(), lens, lens), (table.T, lens, lens)):
        with pytest.raises(ValueError):
            fork_pages(pool, *bad, 16)
    for bad in ((table[:0], lens[:0]), (table, lens.float()), (table[0], lens)):
        with pytest.raises(ValueError):
            compact_pages(pool, *bad, 16)
    with pytest.raises(ValueError):
        copy_pages(pool, lens, lens[:1], 16)


def test_native_entries_refuse():
    """Every bad argument is an error code before any CUDA call."""
    import ctypes

    from fgw_b200 import _native
    lib = _native.library()

    def made(kind, good, **override):
        p = kind()
        for key, value in {**good, **override}.items():
            setattr(p, key, value)
        return ctypes.byref(p)

    chunk = dict(q=256, k_cache=256, v_cache=256, block_table=256, cache_seqlens=256, cu_seqlens_q=256, out=256, tokens=4,
                 pool_rows=64, q_stride=256, out_stride=256, batch=2, heads=4, kv_heads=2, head_dim=64, table_width=2,
                 page_size=16, dtype=1, causal=1, softmax_scale=0.1)
    for bad in (dict(q=0), dict(q=264), dict(out=0), dict(block_table=0), dict(tokens=-1), dict(pool_rows=60),
                dict(q_stride=128), dict(q_stride=257), dict(out_stride=100), dict(batch=0), dict(heads=5), dict(kv_heads=0),
                dict(head_dim=72), dict(head_dim=272), dict(table_width=0), dict(page_size=24), dict(dtype=2),
                dict(causal=2), dict(softmax_scale=0.0), dict(softmax_scale=math.nan), dict(wait_budget_ms=-1),
                dict(reserved=(ctypes.c_int32 * 2)(1, 0))):
        assert lib.fgw_chunk_attention(made(_native.ChunkParams, chunk, **bad), 256, 1 << 40, None) == 1, bad
    many = made(_native.ChunkParams, chunk, heads=258, kv_heads=2, q_stride=258 * 64, out_stride=258 * 64)
    assert lib.fgw_chunk_attention(many, 256, 1 << 40, None) == _native.ERR_UNSUPPORTED
    assert lib.fgw_chunk_attention(made(_native.ChunkParams, chunk), 100, 1 << 40, None) == 1
    assert lib.fgw_chunk_attention(made(_native.ChunkParams, chunk), 256, 16, None) == _native.ERR_WORKSPACE_TOO_SMALL
    assert lib.fgw_chunk_attention(made(_native.ChunkParams, chunk, tokens=0), None, 0, None) == 0
    assert lib.fgw_chunk_attention(None, None, 0, None) == 1

    rotary = dict(q=256, k=256, v=256, q_out=256, k_cache=256, v_cache=256, block_table=256, cache_seqlens=256,
                  cu_seqlens_q=256, cos_sin=256, tokens=4, pool_rows=64, q_stride=256, k_stride=128, v_stride=128,
                  q_out_stride=256, batch=2, heads=4, kv_heads=2, head_dim=64, rotary_dim=64, positions=9, table_width=2,
                  page_size=16, dtype=1)
    for bad in (dict(q=0), dict(k=8), dict(v_cache=0), dict(cos_sin=0), dict(tokens=-1), dict(pool_rows=0),
                dict(k_stride=64), dict(v_stride=130), dict(heads=3), dict(rotary_dim=0), dict(rotary_dim=65),
                dict(rotary_dim=66), dict(positions=0), dict(dtype=2), dict(interleaved=2), dict(batch=0)):
        assert lib.fgw_rotary_append(made(_native.RotaryParams, rotary, **bad), None) == 1, bad

    pools = (ctypes.c_void_p * 2)(256, 512)
    pages = dict(pools=ctypes.addressof(pools), pool_count=2, block_table=256, cache_seqlens=512, parents=256, table_out=1024,
                 seqlens_out=2048, status=256, row_bytes=64, batch=2, table_width=2, page_size=16, num_pages=9)
    for bad in (dict(pools=0), dict(row_bytes=24), dict(row_bytes=0), dict(table_out=256), dict(seqlens_out=512),
                dict(parents=0), dict(status=0), dict(batch=0), dict(table_width=0), dict(page_size=0), dict(num_pages=0),
                dict(num_pages=(1 << 30) + 1), dict(table_width=1 << 28)):
        assert lib.fgw_page_fork(made(_native.PageParams, pages, **bad), 256, 1 << 40, None) == 1, bad
    assert lib.fgw_page_compact(made(_native.PageParams, pages), 256, 16, None) == _native.ERR_WORKSPACE_TOO_SMALL
    assert lib.fgw_page_copy(made(_native.PageParams, pages, copy_count=3), 256, 1 << 40, None) == 1
