"""Edges of the serving-step operators beyond the sizes of test_serving_ops.py: limits, large batches, shared pages, values that
are not finite. Exact where integers are compared; tolerances elsewhere are those of test_serving_ops.py.
"""
import ctypes
import math
import subprocess

import numpy as np
import pytest
import torch

from fgw_b200 import _native
from oracle import serving
from test_serving_ops import attend_case, on_gpu, ragged, torch_attention, values

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


HOST_DRIVER = r"""
#include "fgw_chunk.cuh"

namespace fgw {  // what the host side calls on its way; nothing is launched
cudaError_t prepare_kernel(const void*, int, int, int*) { return cudaErrorNotSupported; }
CUresult encode_tiled_cached(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill) {
  return CUDA_ERROR_NOT_SUPPORTED;
}
cudaError_t launch_chunk_decode(const fgw_chunk_params&, ChunkArgs, int, cudaStream_t) { return cudaErrorNotSupported; }
cudaError_t launch_chunk_tensor(const fgw_chunk_params&, ChunkArgs, const ChunkList&, int, cudaStream_t) {
  return cudaErrorNotSupported;
}
}  // namespace fgw

int main() {
  for (int group = 1; group <= fgw::kMaxGroup; ++group) {
    for (int tokens = 1; tokens <= 300; tokens += 13) {
      for (int dim = 64; dim <= 256; dim += 64) {
        fgw_chunk_params p = {};
        p.tokens = tokens;
        p.batch = 3;
        p.heads = group;
        p.kv_heads = 1;
        p.head_dim = dim;
        p.page_size = p.pool_rows = 16;
        p.table_width = 1;
        p.q_stride = p.out_stride = group * dim;
        p.dtype = FGW_DTYPE_BFLOAT16;
        p.softmax_scale = 1.f;
        if (fgw::chunk_validate(p) != FGW_OK) return 1;
        if (fgw::launch_chunk(p, 0, nullptr, 148, 0, nullptr) != cudaErrorNotSupported) return 2;
      }
    }
  }
  return 0;
}
"""


def test_the_host_side_of_chunk_attention_is_defined_for_every_group(tmp_path):
    """The host code for up to 128 heads per key head, unoptimised and checked: no division by zero, no overflow."""
    from fgw_b200 import build
    driver = tmp_path / "driver.cu"
    driver.write_text(HOST_DRIVER)
    checks = "-fsanitize=undefined,-fno-sanitize-recover=all"
    command = [build.nvcc(), *build.ARCH, "-std=c++17", "-O0", "-Xcompiler", checks, "--expt-relaxed-constexpr",
               f"-I{build.INCLUDE}", f"-I{build.CSRC}", str(driver), str(build.CSRC / "fgw_chunk.cu"), "-o",
               str(tmp_path / "driver")]
    made = subprocess.run(command, capture_output=True, text=True)
    assert made.returncode == 0, made.stderr
    ran = subprocess.run([str(tmp_path / "driver")], capture_output=True, text=True)
    assert ran.returncode == 0, (ran.returncode, ran.stderr)


# --- pages that several rows hold -----------------------------------------------------------------------------------
# (name, pages of each row, held, parents, reserve, spare pages); pages of 16 tokens. Rows come to hold the same partly
# filled page when a length is lowered, as for a cached prefix of which only a part fits the new text.
SHARED = [
    ("part_of_a_prefix", [[3, 5, 7], [3, 5, 7]], [48, 40], [0, 1], None, 4),
    ("part_of_a_prefix_forked", [[3, 5, 7], [3, 5, 7], []], [48, 40, 0], [1, 0, 1], [41, 48, 41], 4),
    ("inner_page", [[3, 5, 7], [3, 5]], [48, 20], [0, 1], [49, 21], 4),
    ("two_parts", [[3, 5], [3, 5]], [20, 30], [0, 1], [21, 31], 4),
    ("three_parts", [[3, 5], [3, 5], [3, 5]], [20, 30, 17], [2, 1, 0], None, 4),
    ("forks_of_two_parts", [[3, 5], [3, 5], [], []], [20, 30, 0, 0], [0, 1, 0, 1], [33, 31, 21, 31], 9),
    ("the_other_leaves", [[3, 5, 7], [3, 5, 7]], [48, 40], [-1, 1], [0, 41], 4),
    ("whole_pages_stay_shared", [[3, 5, 7], [3, 5, 7]], [48, 32], [0, 1], [49, 33], 4),
    ("twice_in_a_row", [[3, 3]], [20], [0], [21], 4),
    ("too_few_for_the_copy", [[0, 1, 2], [0, 1, 2]], [48, 40], [0, 1], None, 0),
    ("empty", [[3, 5], [3, 5]], [0, 20], [0, 1], [1, 21], 4),
]


def shared_state(rows, held, spare):
    width = max(max(map(len, rows)), 1) + 3
    table = np.full((len(rows), width), -1, dtype=np.int32)
    for b, row in enumerate(rows):
        table[b, :len(row)] = row
    return table, np.array(held, dtype=np.int32), int(table.max()) + 1 + spare


@pytest.mark.gpu
@pytest.mark.parametrize("case", SHARED, ids=[c[0] for c in SHARED])
def test_fork_copies_a_partly_filled_page_that_another_row_holds(case):
    """After a fork the page that a row's next token goes to is the row's own."""
    from fgw_b200.operators.mha.page_ops import fork_pages
    name, rows, held, parents, reserve, spare = case
    page = 16
    table, lens, pages = shared_state(rows, held, spare)
    parents = np.array(parents, dtype=np.int32)
    reserve = None if reserve is None else np.array(reserve, dtype=np.int32)
    want_table, want_lens, want_status, copies = serving.fork_pages(table, lens, parents, reserve, page, pages)
    store = values((pages * page, 2, 16), torch.bfloat16, 3)
    pool = store.cuda()
    got = fork_pages([pool], *on_gpu(table, lens, parents), page,
                     reserve_seqlens=None if reserve is None else on_gpu(reserve)[0])
    assert tuple(got[2].tolist()) == want_status
    assert np.array_equal(got[0].cpu().numpy(), want_table)
    assert np.array_equal(got[1].cpu().numpy(), want_lens)
    assert torch.equal(pool.cpu().view(torch.int16),
                       torch.from_numpy(serving.copy_rows(store.view(torch.int16).numpy(), copies, page)))
    if want_status[0] > want_status[1]:
        return
    table2, lens2 = got[0].cpu().numpy(), got[1].cpu().numpy()
    entries = [table2[b, :-(-n // page)].tolist() for b, n in enumerate(lens2)]
    for b, n in enumerate(lens2):
        if n % page:
            assert sum(row.count(entries[b][-1]) for row in entries) == 1, (b, entries)
        # and the row still has its parent's tokens
        if parents[b] >= 0:
            before = [int(table[parents[b], t // page]) * page + t % page for t in range(n)]
            after = [entries[b][t // page] * page + t % page for t in range(n)]
            assert torch.equal(pool[after].cpu(), store[before])


# --- YaRN angles ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("base,dim,trained,factor", [
    (10000.0, 128, 131072, 4.0), (10000.0, 128, 4096, 16.0), (500.0, 64, 8192, 8.0), (1e6, 96, 32768, 2.0),
    (10000.0, 32, 100, 4.0),
])
def test_yarn_blends_by_the_turns_of_every_pair(base, dim, trained, factor):
    """Every pair, the middle of the blend and pairs past which it would run included, against the published ramp: over the
    pair index from floor(pair of beta_fast turns), at least 0, to ceil(pair of beta_slow turns), at most dim - 1."""
    from fgw_b200.operators.mha.rotary_append import rotary_table
    got = rotary_table(2, dim, base=base, scaling="yarn", factor=factor, original_positions=trained, attention_factor=1.0,
                       device="cpu").double()
    low = max(math.floor(dim * math.log(trained / (32.0 * 2 * math.pi)) / (2 * math.log(base))), 0)
    high = min(math.ceil(dim * math.log(trained / (1.0 * 2 * math.pi)) / (2 * math.log(base))), dim - 1)
    partly = 0
    for pair in range(dim // 2):
        plain = base ** (-2.0 * pair / dim)
        slow = min(max((pair - low) / max(high - low, 1e-3), 0.0), 1.0)
        partly += 0.0 < slow < 1.0
        freq = plain * (1.0 - slow) + plain / factor * slow
        assert abs(got[1, pair] - math.cos(freq)) <= 2.0 ** -24 + 1e-12  # one rounding to FP32
        assert abs(got[1, dim // 2 + pair] - math.sin(freq)) <= 2.0 ** -24 + 1e-12
        if trained * plain / (2 * math.pi) > 1.0 + 1e-6:  # more than beta_slow turns: not fully divided
            assert slow < 1.0
    assert partly > 3


# --- scores that are not finite -------------------------------------------------------------------------------------
NOT_FINITE = [
    # (name, new, held, heads, kv heads, dim, page, causal): pieces and whole items of both kernels
    ("tokens", [1] * 9, [5, 300, 64, 1, 2000, 77, 128, 129, 31], 8, 2, 128, 16, True),
    ("drafts", [7, 3, 5], [400, 90, 5], 8, 1, 256, 16, True),
    ("chunk", [200], [900], 4, 2, 128, 32, True),
    ("chunk_narrow", [200, 1, 70], [500, 40, 70], 4, 2, 64, 32, True),
    ("chunk_wide", [150, 2], [1200, 30], 2, 1, 192, 64, False),
    ("whole_items", [40 + 7 * i % 60 for i in range(40)], [140 + 211 * i % 700 for i in range(40)], 8, 8, 128, 64, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")], ids=["nan", "inf", "minus_inf"])
@pytest.mark.parametrize("case", NOT_FINITE, ids=[c[0] for c in NOT_FINITE])
def test_attention_of_scores_that_are_not_finite(case, bad):
    """A query or a key that is not finite makes the outputs of the rows that see it what the formula gives (NaN, not
    zeros, where a score is NaN or +inf; zeros where all are -inf), and leaves all other rows alone."""
    from fgw_b200.operators.mha.chunk_attention import paged_chunk_attention
    _, new, held, heads, kv_heads, dim, page, causal = case
    q, k, v, table, lens, cu = attend_case(case, torch.bfloat16, seed=41)
    q[len(q) // 2, heads - 1, dim // 3] = bad
    for b in range(0, len(new), 3):  # a key in the middle, and (where it is a chunk) one among the new tokens
        for at in {held[b] // 2, held[b] - (new[b] + 1) // 2}:
            k[int(table[b, at // page]) * page + at % page, 0, 1] = bad
    with np.errstate(invalid="ignore", over="ignore"):
        want, spread = serving.chunk_attention(*(x.double().numpy() for x in (q, k, v)), table, lens, cu, page, causal,
                                               dim ** -0.5)
    got = paged_chunk_attention(*(x.cuda() for x in (q, k, v)), *on_gpu(table, lens, cu), page, is_causal=causal)
    got = got.double().cpu().numpy()
    lost = np.isnan(want)
    assert lost.any() and not lost.all()
    assert np.array_equal(np.isnan(got), lost)
    bound = 2.0 ** -8 * (2 * np.abs(want) + spread) + 2.0 ** -16 * spread + 1e-6
    assert (np.abs(got - want)[~lost] <= bound[~lost]).all()


# --- lengths near 2^31 ----------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 200], ids=["token", "chunk"])
def test_attention_over_as_many_tokens_as_a_table_can_hold(new):
    """2^31 - 16 cached tokens, over pages that repeat. The keys are zeros, so every weight is one and every sum a whole
    number below 2^24 per CTA: the outputs are the values' shares, rounded once."""
    from fgw_b200.operators.mha.chunk_attention import paged_chunk_attention
    page, dim, pages = 16, 16, 8
    width = 2 ** 27 - 1
    table = (torch.arange(width, device="cuda", dtype=torch.int32) % pages).view(1, width)
    lens = torch.tensor([width * page], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, new], dtype=torch.int32, device="cuda")
    k = torch.zeros(pages * page, 1, dim, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    v[:, :, 0] = 1  # every token
    v[:page, :, 1] = 1  # every eighth page
    v[3::page, :, 2] = 1  # one token of every page
    v[5 * page + 7, :, 3] = 1
    q = torch.randn(new, 1, dim, device="cuda").to(torch.bfloat16)
    got = paged_chunk_attention(q, k, v, table, lens, cu, page).float()
    for at, share in enumerate((1.0, 1 / 8, 1 / 16, 1 / 128)):
        assert ((got[:, 0, at] - share).abs() <= share * 2.0 ** -8).all(), (at, got[:, 0, at])
    assert not got[:, 0, 4:].any()


# --- sizes at which the kernels take their other paths ----------------------------------------------------------------
BIG_STATES = [
    # (name, held, page, spare pages): more than 4096 rows, 32768 table entries, 131072 pages; the last has just as many
    ("rows", [(7 * i) % 33 for i in range(5000)], 4, 30000),
    ("entries", [37 * i % 1200 for i in range(1, 65)], 2, 3000),
    ("pages", [100 * i for i in range(9)], 4, 140000),
    ("below", [5 * i % 28 for i in range(4096)], 4, 131072 - 15354),
]


def big_state(case, row=(8,)):
    name, held, page, spare = case
    table, lens, _, pages = ragged([0] * len(held), held, page, 7, spare_pages=spare, spare_width=1)
    return table, lens, pages, page, values((pages * page, *row), torch.float16, 5)


@pytest.mark.gpu
@pytest.mark.parametrize("case", BIG_STATES, ids=[c[0] for c in BIG_STATES])
def test_fork_of_large_tables(case):
    from fgw_b200.operators.mha.page_ops import fork_pages
    table, lens, pages, page, store = big_state(case)
    rng = np.random.default_rng(3)
    rows = len(lens)
    parents = np.where(rng.random(rows) < 0.5, np.arange(rows), rng.integers(-1, rows, rows)).astype(np.int32)
    lens[1::7] -= np.minimum(lens[1::7], 1)  # ends that are not where the tables were filled to
    table[2::11] = table[1::11][:len(table[2::11])]  # rows that hold their neighbours' pages, also with other lengths
    lens[2::11] = np.minimum(lens[2::11], lens[1::11][:len(lens[2::11])])
    held = np.where(parents >= 0, lens[np.maximum(parents, 0)], 0)
    reserve = (held + rng.integers(0, 3, rows)).astype(np.int32)
    want_table, want_lens, want_status, copies = serving.fork_pages(table, lens, parents, reserve, page, pages)
    assert want_status[0] <= want_status[1] and len(copies) >= 2
    pool = store.cuda()
    got = fork_pages([pool], *on_gpu(table, lens, parents), page, reserve_seqlens=on_gpu(reserve)[0])
    assert tuple(got[2].tolist()) == want_status
    assert np.array_equal(got[0].cpu().numpy(), want_table) and np.array_equal(got[1].cpu().numpy(), want_lens)
    assert torch.equal(pool.cpu().view(torch.int16),
                       torch.from_numpy(serving.copy_rows(store.view(torch.int16).numpy(), copies, page)))


@pytest.mark.gpu
@pytest.mark.parametrize("case", BIG_STATES, ids=[c[0] for c in BIG_STATES])
def test_compaction_of_large_tables(case):
    from fgw_b200.operators.mha.page_ops import compact_pages
    table, lens, pages, page, store = big_state(case)
    table[2::11] = table[1::11][:len(table[2::11])]
    lens[2::11] = np.minimum(lens[2::11], lens[1::11][:len(lens[2::11])])
    want_table, want_status, copies = serving.compact_pages(table, lens, page, pages)
    pool = store.cuda()
    got, status = compact_pages([pool], *on_gpu(table, lens), page)
    assert tuple(status.tolist()) == want_status and want_status[1] > 50
    assert np.array_equal(got.cpu().numpy(), want_table)
    assert torch.equal(pool.cpu().view(torch.int16),
                       torch.from_numpy(serving.copy_rows(store.view(torch.int16).numpy(), copies, page)))


MANY_REQUESTS = [
    # (name, new, held, heads, kv heads, dim, page, causal): more requests than threads share out one each (288), than the
    # plan sorts (2048), and more items than it sorts
    ("tokens_300", [1] * 300, [(13 * i) % 200 for i in range(300)], 4, 2, 64, 16, True),
    ("tokens_2100", [int(i % 5 > 0) for i in range(2100)], [1 + (29 * i) % 90 for i in range(2100)], 2, 1, 32, 16, True),
    ("mixed_600", [(0, 1, 1, 40, 3, 1, 200)[i % 7] for i in range(600)], [200 + (17 * i) % 150 for i in range(600)], 2, 1,
     64, 16, True),
    ("mixed_2100", [(0, 1, 1, 2, 300)[i % 5] if i % 50 < 5 else 1 for i in range(2100)],
     [300 + (11 * i) % 60 for i in range(2100)], 2, 2, 32, 16, True),
    ("chunks_2100", [33 + i % 3 for i in range(2100)], [40 + (7 * i) % 200 for i in range(2100)], 2, 1, 16, 16, True),
    ("items_of_one_token", [900, 1, 700, 650], [1000, 40, 700, 900], 128, 1, 256, 64, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", MANY_REQUESTS, ids=[c[0] for c in MANY_REQUESTS])
def test_attention_of_many_requests(case):
    from fgw_b200.operators.mha.chunk_attention import paged_chunk_attention
    _, new, held, heads, kv_heads, dim, page, causal = case
    q, k, v, table, lens, cu = attend_case(case, torch.bfloat16, seed=51)
    args = [q.cuda(), k.cuda(), v.cuda()]
    out = torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda")
    got = paged_chunk_attention(*args, *on_gpu(table, lens, cu), page, is_causal=causal, out=out)
    want, spread = torch_attention(*args, table, lens, cu, page, causal)
    bound = 2.0 ** -8 * (2 * want.abs() + spread) + 2.0 ** -16 * spread + 1e-6
    assert bool(((got.double() - want).abs() <= bound).all())
    assert torch.equal(got, paged_chunk_attention(*args, *on_gpu(table, lens, cu), page, is_causal=causal))
