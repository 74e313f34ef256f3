// Attention of a ragged batch of new tokens over a paged KV cache (fgw_chunk_attention in include/fgw_mha.h): argument
// checks, workspace, the plan kernel and the choice of kernels.
//
// out[t, h] = sum_j softmax_j(scale q[t, h] . k[j, h / G]) v[j, h / G] over the first vis(t) cached tokens of t's request:
// vis = len - n + i + 1 for the i-th of its n new tokens when causal, len otherwise; rows with vis <= 0 are zeros.
//
// Two kernels share the work, each request going whole to one of them: requests with few (token, head of a group) rows per
// key head to the decode kernel (fgw_chunk_decode.cu, bound by HBM), the others to the tensor kernel
// (fgw_chunk_sm100.cu, tcgen05). Lengths are device data, so the host does not know which requests are which: when the
// requests' average rows fit an item of the decode kernel it launches that alone, which then takes everything (a longer
// request in several items), else both. The plan (for the tensor kernel), tensor, decode and merge kernels follow one
// another as programmatic dependent launches, so each one's set-up overlaps the one before; the decode kernel needs
// nothing of the others and starts on the SMs that the tensor kernel leaves first.
#include <algorithm>
#include <numeric>

#include "fgw_chunk.cuh"

namespace fgw {

constexpr int kPlanListThreads = 512;  // against 1024: 9.0 -> 8.3 us of plan for a mixed step, 256 no better
constexpr int kPlanSorted = 2048;     // rows of a list sorted in shared memory; longer lists keep the request order
// What the tensor kernel's time is dealt by, in quarters of a KV tile's step of two query tiles. From a fit to the times of
// its CTAs (D = 64: 1.93 us per step of two query tiles, 1.52 us of one, 4.5 us per item; D = 128: 2.95, 2.0 and 4.1 us).
constexpr int kStepCost = 4, kOneTileStepCost = 3;
constexpr int kItemCost = 9;           // an item's start and end
constexpr int kCutCost = 32;           // cutting items: pieces, merge
constexpr int kTensorMinUnits = 2;    // units a program's range has at least when every item is cut
constexpr int kMergeThreads = 256;
constexpr int kMergeRows[2] = {4, 64};  // rows merged by one CTA, by list

// Sum over the CTA of each thread's value before it in thread order, and the total.
template <typename V>
__device__ __forceinline__ V block_scan(V v, V& total, V* shared) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  V sum = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const V up = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += up;
  }
  __syncthreads();
  if (lane == 31) shared[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    V w = lane < (kPlanListThreads / 32) ? shared[lane] : V(0);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const V up = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w += up;
    }
    shared[lane] = w;
  }
  __syncthreads();
  total = shared[kPlanListThreads / 32 - 1];
  return sum - v + (warp > 0 ? shared[warp - 1] : V(0));
}

// The tensor kernel's work list: the items by descending cost, dealt in whole rounds of one item per program: in snake
// order, the last round to the programs with the least load first. Where the longest program would exceed an equal share
// by more than 5 % and what cutting costs, only as many rounds are whole as stay within each program's share, and the rest
// is cut into a contiguous range of units per program that fills its share up. The last round by load, against snake
// order throughout: a batch of prompts 64.6 -> 58.3 us (CTAs of 28 to 53 us -> 28 to 45), single tokens and chunks
// mixed 160.9 -> 158.4 us. The sort compares every row with every other: nothing for the tens of rows of such a step, but
// 193 us for 2000 requests of 70 tokens, whose items then take 262.
struct PlanShared {
  long long scan_l[32];
  int scan_i[32];
  int4 raw[kPlanSorted], rows[kPlanSorted];  // {request, first token, units, cost}
  long long prefix[kPlanSorted + 1];
  int first[kPlanSorted + 1];
  alignas(16) uint32_t loads[kStreamMaxPrograms];
};

__global__ void __launch_bounds__(kPlanListThreads)
    chunk_plan_kernel(const __grid_constant__ ChunkArgs a, const __grid_constant__ ChunkList list) {
  grid_dependents_launch();
  extern __shared__ uint8_t plan_smem[];
  PlanShared& sh = *reinterpret_cast<PlanShared*>(plan_smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // rows of each request, and their place in the list; lists that fit stay in shared memory
  int* first = a.batch <= kPlanSorted ? sh.first : list.first;
  int rows = 0;
  for (int base = 0; base < a.batch; base += kPlanListThreads) {
    const int b = base + tid;
    int all;
    const int mine = b < a.batch ? item_rows(a, new_tokens(a.cu, a.tokens, b).count, false) : 0;
    const int at = block_scan(mine, all, sh.scan_i);
    if (b < a.batch) first[b] = rows + at;
    rows += all;
  }
  rows = min(rows, list.max_rows);
  if (tid == 0) first[a.batch] = rows;
  __syncthreads();
  const bool small = rows <= kPlanSorted;
  int4* raw = small ? sh.raw : list.unsorted;
  for (int b = warp; b < a.batch; b += kPlanListThreads / 32) {
    const int begin = min(first[b], rows), end = min(first[b + 1], rows);
    if (begin >= end) continue;
    const int count = new_tokens(a.cu, a.tokens, b).count;
    const int len = held_tokens(a.lens, b, a.width, a.page);
    for (int r = begin + lane; r < end; r += 32) {
      const int t0 = (r - begin) * a.tokens_per_item;
      const int units = item_units<128>(a, count, len, t0);
      const bool one_tile = a.dim <= 128 && count - t0 <= a.tokens_per_item / 2;
      raw[r] = make_int4(b, t0, units, units * (one_tile ? kOneTileStepCost : kStepCost) + kItemCost);
    }
  }
  __syncthreads();
  // by descending cost (ties: in order), so that whole items are dealt longest first; with fewer items than programs
  // all are cut and the order does not matter
  const int programs = a.programs;
  const int items = rows * a.kv_heads;
  const bool order = small && items > programs;
  int4* sorted = small ? sh.rows : list.rows;
  for (int r = tid; r < rows; r += kPlanListThreads) {
    const int4 row = raw[r];
    int rank = r;
    if (order) {
      rank = 0;
      for (int s = 0; s < rows; ++s) rank += (raw[s].w > row.w || (raw[s].w == row.w && s < r)) ? 1 : 0;
    }
    sorted[rank] = row;
    if (small) list.rows[rank] = row;
  }
  __syncthreads();
  long long* prefix = small ? sh.prefix : list.prefix;
  long long total = 0;
  for (int base = 0; base < rows; base += kPlanListThreads) {
    const int r = base + tid;
    long long all;
    const long long at = block_scan(r < rows ? static_cast<long long>(sorted[r].z) * a.kv_heads : 0ll, all, sh.scan_l);
    if (r < rows) prefix[r] = total + at;
    total += all;
  }
  if (tid == 0) prefix[rows] = total;
  __syncthreads();
  const bool mine = tid < programs;
  auto item_of = [&](int round) {  // this program's item in a round in snake order, {0, 0, 0, 0} when it has none
    const int item = round * programs + ((round & 1) ? programs - 1 - tid : tid);
    return mine && item < items ? sorted[a.by_kv_heads.quotient(item)] : make_int4(0, 0, 0, 0);
  };
  const long long quotient = divide(total, programs);
  const int remainder = static_cast<int>(total - quotient * programs);
  const long long fair = mine ? quotient + (tid < remainder ? 1 : 0) : 0;  // units of an equal share
  const int all_rounds = (items + programs - 1) / programs;
  int rounds = 0, snake = 0, ranges = programs, last = items;
  long long load = 0;
  if (items > programs) {
    for (int r = 0; r + 1 < all_rounds; ++r) load += item_of(r).w;
    const uint32_t have = static_cast<uint32_t>(min(load, 0xfffffffell));
    if (tid < kStreamMaxPrograms) sh.loads[tid] = mine ? have : 0xffffffffu;
    __syncthreads();
    if (mine) {
      int rank = 0;
#pragma unroll 4
      for (int p = 0; p < programs; p += 4) {
        const uint4 four = *reinterpret_cast<const uint4*>(&sh.loads[p]);
        rank += (four.x < have || (four.x == have && p < tid)) + (four.y < have || (four.y == have && p + 1 < tid)) +
                (four.z < have || (four.z == have && p + 2 < tid)) + (four.w < have || (four.w == have && p + 3 < tid));
      }
      last = min((all_rounds - 1) * programs + rank, items);
      if (last < items) load += sorted[a.by_kv_heads.quotient(last)].w;
    }
    long long all_cost;
    block_scan(mine ? load : 0ll, all_cost, sh.scan_l);
    const long long equal = divide(all_cost, programs);
    if (__syncthreads_and(!mine || load <= equal + equal / 20 + kCutCost)) {
      rounds = all_rounds;
      snake = all_rounds - 1;
    } else {
      load = 0;
      while (static_cast<long long>(rounds + 1) * programs <= items) {
        const int units = item_of(rounds).z;
        if (!__syncthreads_and(load + units <= fair)) break;
        load += units;
        ++rounds;
      }
      snake = rounds;
    }
  } else {
    ranges = static_cast<int>(max(1ll, min(static_cast<long long>(programs), total / kTensorMinUnits)));
  }
  const int cut = min(rounds * programs, items);  // first cut item
  const bool none = cut == items;
  long long share = 0;
  if (!none && rounds > 0) {
    share = fair - load;
  } else if (!none && tid < ranges) {
    const long long each = divide(total, ranges);
    share = each + (tid < total - each * ranges ? 1 : 0);
  }
  long long rest;
  const long long before = block_scan(mine ? share : 0ll, rest, sh.scan_l);
  if (mine) {
    long long u = total;
    int item = last, off = 0;  // the last round's item, else the first of the cut range
    if (!none) {
      const int cut_row = a.by_kv_heads.quotient(cut);
      u = prefix[cut_row] + static_cast<long long>(cut - cut_row * a.kv_heads) * sorted[cut_row].z + before;
      int lo = 0, hi = rows - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (prefix[mid] <= u) {
          lo = mid;
        } else {
          hi = mid - 1;
        }
      }
      if (u < total) {
        const int units = sorted[lo].z;
        const long long within = u - prefix[lo];
        const int hk = static_cast<int>(divide(within, units));
        item = lo * a.kv_heads + hk;
        off = static_cast<int>(within - static_cast<long long>(hk) * units);
      }
    }
    list.prog_u[tid] = u;
    list.prog_item[tid] = item;
    list.prog_off[tid] = off;
  }
  if (tid == 0) {
    list.prog_u[programs] = total;
    list.meta->items = items;
    list.meta->rounds = rounds;
    list.meta->snake = snake;
  }
}

// Merges the pieces of the cut items of both kernels, a few rows per CTA, every thread four values of one row: a
// running peak of the pieces' LSEs, their weights 2^(lse - peak) and the weighted sum, in piece order, eight pieces'
// loads at a time. Bound by the latency of two dependent trips to L2 (the cut, then its pieces). Also writes zeros into the
// rows of no request and reduces the CTAs' errors to the header's word.
struct MergeList {
  ChunkSlots slots;
  const long long* prog_u;  // [programs + 1]: programs without units hold no piece (nullptr: all hold one)
  int slot_rows, rows, parts;  // `parts` CTAs per program, `rows` rows each
  bool by_column;           // O laid out [dim / 4][rows][4], else [rows][dim]
};
struct MergeArgs {
  ChunkArgs a;
  WorkspaceHeader* ws;
  MergeList list[2];  // decode, tensor; parts 0: kernel not launched
};

// The first error of the calls on this device since it was last read {fgw_status, wait site}: a caller whose workspace is
// gone when the call returns has no other place to look.
__device__ int g_chunk_error[2];

__device__ void merge_errors(const MergeArgs& m) {
  int code = 0, site = 0;
  for (int k = 0; k < 2; ++k) {
    for (int p = threadIdx.x; m.list[k].parts > 0 && p < m.a.programs; p += 32) {
      const int2 e = m.list[k].slots.errors[p];
      if (e.x != 0 && code == 0) {
        code = e.x;
        site = e.y;
      }
    }
  }
  const uint32_t any = __ballot_sync(0xffffffffu, code != 0);
  const int from = any != 0 ? __ffs(any) - 1 : 0;
  code = __shfl_sync(0xffffffffu, code, from);
  site = __shfl_sync(0xffffffffu, site, from);
  if (threadIdx.x == 0) {
    m.ws->error = code;
    m.ws->error_site = site;
    if (code != 0 && atomicCAS(&g_chunk_error[0], 0, code) == 0) g_chunk_error[1] = site;
  }
}

template <typename T>
__global__ void __launch_bounds__(kMergeThreads) chunk_merge_kernel(const __grid_constant__ MergeArgs m) {
  using Tr = ElemTraits<T>;
  const ChunkArgs& a = m.a;
  const int tid = threadIdx.x;
  const int decode_ctas = m.list[0].parts * a.programs;
  const int kind = static_cast<int>(blockIdx.x) < decode_ctas ? 0 : 1;
  const MergeList& l = m.list[kind];
  const int at = blockIdx.x - (kind ? decode_ctas : 0);
  const int q = at / l.parts, row0 = at % l.parts * l.rows;
  const int groups = a.dim / 4;
  const int tile_tokens = kTensorTileRows / a.group;
  const long long step = static_cast<long long>(l.slot_rows) * groups;  // float4s of a slot
  grid_dependency_wait();
  const ChunkCut cut = l.slots.cuts[q];
  const long long first = min(max(static_cast<long long>(a.cu[0]), 0ll), a.tokens);
  const long long end = min(max(static_cast<long long>(a.cu[a.batch]), first), a.tokens);
  if (cut.last >= q) {
    for (int i = tid; i < l.rows * groups; i += kMergeThreads) {
      // neighbouring threads read neighbouring 16 bytes of the slot
      const int r = l.by_column ? i % l.rows : i / groups, g = l.by_column ? i / l.rows : i % groups;
      const int row = row0 + r;
      // a slot's rows are (tile, row of the tile); a tile holds whole tokens
      const int tile = row / kTensorTileRows, in_tile = row % kTensorTileRows;
      const int in_token = a.by_group.quotient(in_tile), token = tile * tile_tokens + in_token;
      if (row >= l.slot_rows || in_token >= tile_tokens || token >= cut.count) continue;
      const float4* src = reinterpret_cast<const float4*>(l.slots.o) +
                          (l.by_column ? static_cast<long long>(g) * l.slot_rows + row : static_cast<long long>(row) * groups + g);
      const float* lses = l.slots.lse + row;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float peak = kEmptyLse, sum = 0.f;
      for (int p0 = q; p0 <= cut.last; p0 += 8) {
        float4 v[8];
        float w[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int p = p0 + u;
          w[u] = kEmptyLse;
          v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (p <= cut.last && (l.prog_u == nullptr || l.prog_u[p] < l.prog_u[p + 1])) {
            const int slot = 2 * p + (p == q ? 1 : 0);
            w[u] = lses[static_cast<long long>(slot) * l.slot_rows];
            v[u] = src[slot * step];
          }
        }
        float next = peak;
#pragma unroll
        for (int u = 0; u < 8; ++u) next = fmaxf(next, w[u]);
        const float keep = fast_exp2(peak - next);
        sum *= keep;
        acc.x *= keep;
        acc.y *= keep;
        acc.z *= keep;
        acc.w *= keep;
        peak = next;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const float wk = w[u] <= kValidLse ? 0.f : fast_exp2(w[u] - peak);  // a piece's NaN stays one
          sum += wk;
          acc.x = fmaf(wk, v[u].x, acc.x);
          acc.y = fmaf(wk, v[u].y, acc.y);
          acc.z = fmaf(wk, v[u].z, acc.z);
          acc.w = fmaf(wk, v[u].w, acc.w);
        }
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      T* out = static_cast<T*>(a.out) + (cut.token0 + token) * a.out_stride +
               static_cast<long long>(cut.hk * a.group + in_tile - in_token * a.group) * a.dim + g * 4;
      *reinterpret_cast<uint2*>(out) =
          make_uint2(Tr::pack2(acc.x * inv, acc.y * inv), Tr::pack2(acc.z * inv, acc.w * inv));
    }
  }
  // rows of no request
  const int chunks = a.heads * a.dim / 8;
  const long long none = (first + a.tokens - end) * chunks;
  for (long long i = static_cast<long long>(blockIdx.x) * kMergeThreads + tid; i < none;
       i += static_cast<long long>(gridDim.x) * kMergeThreads) {
    const long long k = i / chunks;
    const long long t = k < first ? k : end + k - first;
    reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + t * a.out_stride)[i % chunks] = make_uint4(0, 0, 0, 0);
  }
  if (blockIdx.x == 0 && tid < 32) merge_errors(m);
}

cudaError_t take_chunk_error(int (&words)[2]) {
  const cudaError_t err = cudaMemcpyFromSymbol(words, g_chunk_error, sizeof(words), 0, cudaMemcpyDeviceToHost);
  if (err != cudaSuccess || words[0] == 0) return err;
  const int none[2] = {0, 0};
  return cudaMemcpyToSymbol(g_chunk_error, none, sizeof(none), 0, cudaMemcpyHostToDevice);
}

int chunk_validate(const fgw_chunk_params& p) {
  for (int r : p.reserved) {
    if (r != 0) return FGW_ERR_INVALID_ARGUMENT;
  }
  if (p.tokens < 0 || p.tokens > 0x7fffffffll || p.batch <= 0 || p.heads <= 0 || p.kv_heads <= 0 ||
      p.heads % p.kv_heads != 0 || p.table_width <= 0 || p.page_size <= 0 || p.page_size % 16 != 0 ||
      p.pool_rows <= 0 || p.pool_rows % p.page_size != 0) {
    return FGW_ERR_INVALID_ARGUMENT;
  }
  if (p.head_dim < 16 || p.head_dim > 256 || p.head_dim % 16 != 0) return FGW_ERR_INVALID_ARGUMENT;
  if (static_cast<long long>(p.page_size) * p.table_width > 0x7fffffffll) return FGW_ERR_INVALID_ARGUMENT;
  if (p.pool_rows > 0x7fffffffll) return FGW_ERR_INVALID_ARGUMENT;
  if (p.dtype != FGW_DTYPE_FLOAT16 && p.dtype != FGW_DTYPE_BFLOAT16) return FGW_ERR_INVALID_ARGUMENT;
  if ((p.causal != 0 && p.causal != 1) || p.wait_budget_ms < 0) return FGW_ERR_INVALID_ARGUMENT;
  if (!(p.softmax_scale > 0.f) || p.softmax_scale > 1e30f) return FGW_ERR_INVALID_ARGUMENT;
  const long long row = static_cast<long long>(p.heads) * p.head_dim;
  if (p.q_stride < row || p.q_stride % 8 != 0 || p.out_stride < row || p.out_stride % 8 != 0) {
    return FGW_ERR_INVALID_ARGUMENT;
  }
  if (p.heads / p.kv_heads > kMaxGroup) return FGW_ERR_UNSUPPORTED;
  // items and list rows are counted in 32 bits
  if ((p.tokens + p.batch) * p.kv_heads > 0x7fffffffll) return FGW_ERR_INVALID_ARGUMENT;
  return FGW_OK;
}

int chunk_validate_pointers(const fgw_chunk_params& p) {
  const void* data[4] = {p.q, p.k_cache, p.v_cache, p.out};
  for (const void* d : data) {
    if (d == nullptr || reinterpret_cast<uintptr_t>(d) % 16 != 0) return FGW_ERR_INVALID_ARGUMENT;
  }
  return p.block_table == nullptr || p.cache_seqlens == nullptr || p.cu_seqlens_q == nullptr ? FGW_ERR_INVALID_ARGUMENT
                                                                                             : FGW_OK;
}

int chunk_box_rows(int page, int keys) { return std::gcd(page, keys); }

static CUresult chunk_kv_map(CUtensorMap* map, const fgw_chunk_params& p, const void* base, int box_rows) {
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(p.head_dim), static_cast<cuuint64_t>(p.kv_heads),
                              static_cast<cuuint64_t>(p.pool_rows)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(p.head_dim) * 2,
                                 static_cast<cuuint64_t>(p.head_dim) * p.kv_heads * 2};
  const cuuint32_t box[3] = {64, 1, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t ones[3] = {1, 1, 1};
  const CUtensorMapDataType type =
      p.dtype == FGW_DTYPE_BFLOAT16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return encode_tiled_cached(map, type, 3, const_cast<void*>(base), dims, strides, box, ones,
                             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

CUresult chunk_kv_maps(CUtensorMap* kmap, CUtensorMap* vmap, const fgw_chunk_params& p, const ChunkArgs& a) {
  const CUresult err = chunk_kv_map(kmap, p, p.k_cache, a.box_rows / (a.short_boxes & 1 ? 2 : 1));
  return err != CUDA_SUCCESS ? err : chunk_kv_map(vmap, p, p.v_cache, a.box_rows / (a.short_boxes & 2 ? 2 : 1));
}

// Rows of a decode item (16, 32 or 64): enough for the requests' average rows where that is at all possible, else (chunks
// among them) for single tokens, which are then its work. 33 to 64 rows, against the tensor kernel: D = 256, 13 requests of
// 56 rows over 2000 keys 54.2 -> 34.7 us, 8 of 40 over 8000 with two key heads 80.2 -> 67.8 us, 32 of 64 over 3000 65.1 ->
// 62.2 us; D = 192, 32 of 64 over 3000 49.8 -> 53.1 us, where many requests fill the tensor kernel too.
// Going by the average is its weak spot: where it is at most 64, a long chunk among many single tokens goes through this
// kernel too, in items of so few rows that its cache is read again for each (32 heads on 8 of 128, 199 tokens over caches to
// 8K: 615 us; with a chunk of 64 637, of 512 798, of 2048 2631, of 3500, which the average gives away, 854 us).
static int decode_rows(const fgw_chunk_params& p) {
  constexpr long long most = 64;
  const long long group = p.heads / p.kv_heads;
  const long long average = (p.tokens * group + p.batch - 1) / p.batch;
  const long long want = std::max(average <= most ? average : 0, group);
  return want <= 16 ? 16 : static_cast<int>(std::min<long long>(most, want <= 32 ? 32 : 64));
}
static bool decode_on(const fgw_chunk_params& p) { return p.heads / p.kv_heads <= decode_rows(p); }
static bool tensor_on(const fgw_chunk_params& p) {
  return !decode_on(p) || p.tokens * (p.heads / p.kv_heads) > static_cast<long long>(decode_rows(p)) * p.batch;
}

// The workspace from `at` on (sizes alone when it is null), by class: slots of both kernels, the tensor kernel's list.
struct ChunkLayout {
  ChunkSlots slots[2];
  int tokens_per_item[2], slot_rows[2];
  ChunkList list;
  size_t bytes;
};

static ChunkLayout chunk_layout(const fgw_chunk_params& p, uint8_t* const begin) {
  const int group = p.heads / p.kv_heads, nb = (p.head_dim + 63) / 64;
  ChunkLayout l = {};
  uint8_t* at = begin;
  auto take = [&](size_t n) {
    uint8_t* here = at;
    at += (n + 255) & ~size_t(255);
    return here;
  };
  take(sizeof(WorkspaceHeader));
  const size_t programs = kStreamMaxPrograms;
  const bool on[2] = {decode_on(p), tensor_on(p)};
  l.tokens_per_item[0] = decode_rows(p) / group;
  l.slot_rows[0] = decode_rows(p);
  l.tokens_per_item[1] = kTensorTileRows / group * chunk_tensor_tiles(nb);
  l.slot_rows[1] = kTensorTileRows * chunk_tensor_tiles(nb);
  for (int k = 0; k < 2; ++k) {
    if (!on[k]) continue;
    l.slots[k].cuts = reinterpret_cast<ChunkCut*>(take(programs * sizeof(ChunkCut)));
    l.slots[k].errors = reinterpret_cast<int2*>(take(programs * sizeof(int2)));
    l.slots[k].lse = reinterpret_cast<float*>(take(2 * programs * l.slot_rows[k] * 4));
    l.slots[k].o = reinterpret_cast<float*>(take(2 * programs * l.slot_rows[k] * static_cast<size_t>(p.head_dim) * 4));
  }
  if (on[1]) {
    ChunkList& w = l.list;
    w.max_rows = static_cast<int>(p.tokens / l.tokens_per_item[1] + p.batch);
    const size_t rows = w.max_rows;
    w.meta = reinterpret_cast<ChunkMeta*>(take(sizeof(ChunkMeta)));
    w.rows = reinterpret_cast<int4*>(take(rows * sizeof(int4)));
    w.unsorted = reinterpret_cast<int4*>(take(rows * sizeof(int4)));
    w.prefix = reinterpret_cast<long long*>(take((rows + 1) * 8));
    w.first = reinterpret_cast<int32_t*>(take((static_cast<size_t>(p.batch) + 1) * 4));
    w.prog_item = reinterpret_cast<int32_t*>(take(programs * 4));
    w.prog_off = reinterpret_cast<int32_t*>(take(programs * 4));
    w.prog_u = reinterpret_cast<long long*>(take((programs + 1) * 8));
  }
  l.bytes = static_cast<size_t>(at - begin);
  return l;
}

size_t chunk_workspace_bytes(const fgw_chunk_params& p) { return chunk_layout(p, nullptr).bytes; }

cudaError_t launch_chunk(const fgw_chunk_params& p, int short_boxes, void* workspace, int sm_count, int device,
                         cudaStream_t stream) {
  const ChunkLayout layout = chunk_layout(p, static_cast<uint8_t*>(workspace));
  const bool on[2] = {decode_on(p), tensor_on(p)};
  ChunkArgs a[2] = {};
  a[0].out = p.out;
  a[0].table = p.block_table;
  a[0].lens = p.cache_seqlens;
  a[0].cu = p.cu_seqlens_q;
  a[0].q = p.q;
  a[0].tokens = p.tokens;
  a[0].q_stride = p.q_stride;
  a[0].out_stride = p.out_stride;
  a[0].batch = p.batch;
  a[0].heads = p.heads;
  a[0].kv_heads = p.kv_heads;
  a[0].group = p.heads / p.kv_heads;
  a[0].dim = p.head_dim;
  a[0].width = p.table_width;
  a[0].page = p.page_size;
  a[0].causal = p.causal;
  a[0].programs = std::min(sm_count, kStreamMaxPrograms);
  a[0].by_page = FastDiv(p.page_size);
  a[0].by_group = FastDiv(a[0].group);
  a[0].by_kv_heads = FastDiv(p.kv_heads);
  a[0].small_rows = decode_rows(p);
  a[0].split = on[0] && on[1] ? 1 : 0;
  a[0].scale_log2 = p.softmax_scale * kLog2e;
  a[0].short_boxes = short_boxes;
  a[0].budget_ns = static_cast<uint64_t>(p.wait_budget_ms > 0 ? p.wait_budget_ms : 2000) * 1000000ull;
  a[1] = a[0];
  MergeArgs merge = {};
  merge.ws = static_cast<WorkspaceHeader*>(workspace);
  for (int k = 0; k < 2; ++k) {
    if (!on[k]) continue;  // a decode item holds no token of more than 64 heads per key head
    a[k].tokens_per_item = layout.tokens_per_item[k];
    a[k].by_item_tokens = FastDiv(layout.tokens_per_item[k]);
    a[k].slots = layout.slots[k];
    merge.list[k].slots = layout.slots[k];
    merge.list[k].slot_rows = layout.slot_rows[k];
    merge.list[k].rows = kMergeRows[k];
    merge.list[k].parts = (layout.slot_rows[k] + kMergeRows[k] - 1) / kMergeRows[k];
    merge.list[k].by_column = k == 1;
    merge.list[k].prog_u = k == 1 ? layout.list.prog_u : nullptr;
  }
  merge.a = a[0];
  cudaError_t err = cudaSuccess;
  if (on[1]) {
    err = prepare_kernel(reinterpret_cast<const void*>(chunk_plan_kernel), sizeof(PlanShared), device, nullptr);
    if (err != cudaSuccess) return err;
    chunk_plan_kernel<<<1, kPlanListThreads, sizeof(PlanShared), stream>>>(a[1], layout.list);
    err = cudaGetLastError();
  }
  if (err == cudaSuccess && on[1]) err = launch_chunk_tensor(p, a[1], layout.list, device, stream);
  if (err == cudaSuccess && on[0]) err = launch_chunk_decode(p, a[0], device, stream);
  if (err != cudaSuccess) return err;
  const unsigned grid = static_cast<unsigned>(a[0].programs * (merge.list[0].parts + merge.list[1].parts));
  return p.dtype == FGW_DTYPE_BFLOAT16
             ? launch_after_plan(chunk_merge_kernel<__nv_bfloat16>, grid, kMergeThreads, 0, stream, merge)
             : launch_after_plan(chunk_merge_kernel<__half>, grid, kMergeThreads, 0, stream, merge);
}

}  // namespace fgw
