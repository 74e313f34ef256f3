// Attention of a ragged batch of new tokens over a paged KV cache (fgw_chunk_attention in include/fgw_mha.h): argument
// checks, workspace, the plan kernel and the choice of kernels.
//
// out[t, h] = sum_j softmax_j(scale q[t, h] . k[j, h / G]) v[j, h / G] over the first vis(t) cached tokens of t's request:
// vis = len - n + i + 1 for the i-th of its n new tokens when causal, len otherwise; rows with vis <= 0 are zeros.
//
// Two kernels share the work, each request going whole to one of them: requests with at most 16 (token, head of a group)
// rows per key head to the decode kernel (fgw_chunk_decode.cu, bound by HBM), the others to the tensor kernel
// (fgw_chunk_sm100.cu, tcgen05). Lengths are device data, so the host does not know which requests are which: with at
// most 16 rows per request on average it launches the decode kernel alone, which then takes everything (a longer
// request in several items), else both, in the order plan, decode, tensor.
#include <algorithm>
#include <numeric>

#include "fgw_chunk.cuh"

namespace fgw {

constexpr int kPlanListThreads = 1024;
constexpr int kPlanSorted = 2048;  // rows of a list sorted in shared memory; longer lists keep the request order

enum ChunkClass { kDecodeList = 0, kTensorList = 1 };

struct ChunkPlanArgs {
  ChunkArgs a[2];   // by class; only the lists differ
  bool on[2];
  bool split;       // requests go by their rows; otherwise everything is the decode list's
  int row_bytes;    // of an output row
};

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

__global__ void __launch_bounds__(kPlanListThreads) chunk_plan_kernel(const __grid_constant__ ChunkPlanArgs plan) {
  grid_dependents_launch();
  __shared__ long long scan_l[32];
  __shared__ int scan_i[32];
  __shared__ int units_s[kPlanSorted];
  const int cls = plan.on[kDecodeList] ? static_cast<int>(blockIdx.x) : kTensorList;
  const ChunkArgs& a = plan.a[cls];
  const ChunkList& list = a.list;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (blockIdx.x == 0 && tid == 0) {
    a.ws->error = 0;
    a.ws->error_site = 0;
  }
  for (int p = tid; p < a.programs; p += kPlanListThreads) list.counters[p] = 0;

  // rows of each request, and their place in the list
  auto rows_of = [&](int b) {
    const NewTokens nt = new_tokens(a.cu, a.tokens, b);
    const bool small = nt.count * a.group <= kDecodeRows;
    if (plan.split && small != (cls == kDecodeList)) return 0;
    return (nt.count + list.tokens_per_item - 1) / list.tokens_per_item;
  };
  int rows = 0;
  for (int base = 0; base < a.batch; base += kPlanListThreads) {
    const int b = base + tid;
    int all;
    const int at = block_scan(b < a.batch ? rows_of(b) : 0, all, scan_i);
    if (b < a.batch) list.first[b] = rows + at;
    rows += all;
  }
  rows = min(rows, list.max_rows);
  if (tid == 0) list.first[a.batch] = rows;
  __syncthreads();
  for (int b = warp; b < a.batch; b += kPlanListThreads / 32) {
    const int begin = min(list.first[b], rows), end = min(list.first[b + 1], rows);
    if (begin >= end) continue;
    const NewTokens nt = new_tokens(a.cu, a.tokens, b);
    const int len = held_tokens(a.lens, b, a.width, a.page);
    for (int r = begin + lane; r < end; r += 32) {
      const int t0 = (r - begin) * list.tokens_per_item;
      const int last = min(t0 + list.tokens_per_item, nt.count) - 1;
      const int seen = max(a.causal ? len - nt.count + last + 1 : len, 0);
      const int units = max((seen + list.keys_per_unit - 1) / list.keys_per_unit, 1);  // no keys: zeros to write
      list.unsorted[r] = make_int4(b, t0, units, 0);
      if (r < kPlanSorted) units_s[r] = units;
    }
  }
  __syncthreads();
  // by descending units (ties: in order), so that whole items are dealt longest first
  const int items = rows * a.kv_heads;
  const bool sorted = rows <= kPlanSorted;
  const bool order = sorted && items >= a.programs;
  for (int r = tid; r < rows; r += kPlanListThreads) {
    const int4 row = list.unsorted[r];
    int rank = r;
    if (order) {
      rank = 0;
      for (int s = 0; s < rows; ++s) rank += (units_s[s] > row.z || (units_s[s] == row.z && s < r)) ? 1 : 0;
    }
    list.rows[rank] = row;
  }
  __syncthreads();
  long long total = 0;
  for (int base = 0; base < rows; base += kPlanListThreads) {
    const int r = base + tid;
    const int units = r < rows ? list.rows[r].z : 0;
    if (sorted && r < rows) units_s[r] = units;
    long long all;
    const long long at = block_scan(static_cast<long long>(units) * a.kv_heads, all, scan_l);
    if (r < rows) list.prefix[r] = total + at;
    total += all;
  }
  if (tid == 0) list.prefix[rows] = total;
  __syncthreads();
  // whole rounds in snake order while every program stays within its share
  const int programs = a.programs;
  const bool mine = tid < programs;
  const long long share = mine ? program_start(total, programs, tid + 1) - program_start(total, programs, tid) : 0;
  long long load = 0;
  int rounds = 0;
  while (static_cast<long long>(rounds + 1) * programs <= items) {
    const int item = rounds * programs + ((rounds & 1) ? programs - 1 - tid : tid);
    int units = 0;
    if (mine) units = sorted ? units_s[item / a.kv_heads] : list.rows[item / a.kv_heads].z;
    if (!__syncthreads_and(!mine || load + units <= share)) break;
    load += units;
    ++rounds;
  }
  long long rest;
  const long long before = block_scan(mine ? share - load : 0ll, rest, scan_l);
  const int cut = rounds * programs;  // first cut item
  const int cut_row = cut / a.kv_heads;
  long long cut_u = total;
  if (cut < items) {
    cut_u = list.prefix[cut_row] + static_cast<long long>(cut % a.kv_heads) * list.rows[cut_row].z;
  }
  if (mine) {
    const long long u = cut_u + before;
    list.prog_u[tid] = u;
    if (tid == programs - 1) list.prog_u[programs] = total;
    int lo = 0, hi = max(rows - 1, 0);
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (list.prefix[mid] <= u) {
        lo = mid;
      } else {
        hi = mid - 1;
      }
    }
    int item = 0, off = 0;
    if (rows > 0 && u < total) {
      const int units = list.rows[lo].z;
      const long long within = u - list.prefix[lo];
      item = lo * a.kv_heads + static_cast<int>(within / units);
      off = static_cast<int>(within % units);
    }
    list.prog_item[tid] = item;
    list.prog_off[tid] = off;
  }
  if (tid == 0) {
    list.meta->items = items;
    list.meta->rounds = rounds;
  }
  // rows of no request
  const long long first = min(max(static_cast<long long>(a.cu[0]), 0ll), a.tokens);
  const long long end = min(max(static_cast<long long>(a.cu[a.batch]), first), a.tokens);
  const int chunks = plan.row_bytes / 16;
  const long long none = first + a.tokens - end;
  for (long long i = static_cast<long long>(blockIdx.x) * kPlanListThreads + tid; i < none * chunks;
       i += static_cast<long long>(gridDim.x) * kPlanListThreads) {
    const long long k = i / chunks;
    const long long t = k < first ? k : end + k - first;
    reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + t * a.out_stride)[i % chunks] = make_uint4(0, 0, 0, 0);
  }
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

CUresult chunk_kv_map(CUtensorMap* map, const fgw_chunk_params& p, const void* base, int box_rows) {
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

static bool decode_on(const fgw_chunk_params& p) { return p.heads / p.kv_heads <= kDecodeRows; }
static bool tensor_on(const fgw_chunk_params& p) {
  return !decode_on(p) || p.tokens * (p.heads / p.kv_heads) > static_cast<long long>(kDecodeRows) * p.batch;
}

// The work list of one class at `at` (sizes alone when at is null); returns the bytes it takes.
static size_t carve_list(const fgw_chunk_params& p, int cls, uint8_t* at, ChunkList* out) {
  const int group = p.heads / p.kv_heads, nb = (p.head_dim + 63) / 64;
  ChunkList l;
  int slot_rows;
  if (cls == kDecodeList) {
    l.tokens_per_item = kDecodeRows / group;
    l.keys_per_unit = chunk_decode_keys(nb);
    slot_rows = kDecodeRows;
  } else {
    l.tokens_per_item = kTensorTileRows / group * chunk_tensor_tiles(nb);
    l.keys_per_unit = 128;
    slot_rows = kTensorTileRows * chunk_tensor_tiles(nb);
  }
  l.max_rows = static_cast<int>(p.tokens / l.tokens_per_item + p.batch);
  uint8_t* const begin = at;
  auto take = [&](size_t n) {
    uint8_t* here = at;
    at += (n + 255) & ~size_t(255);
    return here;
  };
  const size_t rows = l.max_rows, programs = kStreamMaxPrograms;
  l.meta = reinterpret_cast<ChunkMeta*>(take(sizeof(ChunkMeta)));
  l.rows = reinterpret_cast<int4*>(take(rows * sizeof(int4)));
  l.unsorted = reinterpret_cast<int4*>(take(rows * sizeof(int4)));
  l.prefix = reinterpret_cast<long long*>(take((rows + 1) * 8));
  l.first = reinterpret_cast<int32_t*>(take((static_cast<size_t>(p.batch) + 1) * 4));
  l.prog_item = reinterpret_cast<int32_t*>(take(programs * 4));
  l.prog_off = reinterpret_cast<int32_t*>(take(programs * 4));
  l.prog_u = reinterpret_cast<long long*>(take((programs + 1) * 8));
  l.counters = reinterpret_cast<int32_t*>(take(programs * 4));
  l.slot_lse = reinterpret_cast<float*>(take(2 * programs * slot_rows * 4));
  l.slot_o = reinterpret_cast<float*>(take(2 * programs * slot_rows * static_cast<size_t>(p.head_dim) * 4));
  if (out != nullptr) *out = l;
  return static_cast<size_t>(at - begin);
}

size_t chunk_workspace_bytes(const fgw_chunk_params& p) {
  size_t bytes = sizeof(WorkspaceHeader);
  if (decode_on(p)) bytes += carve_list(p, kDecodeList, nullptr, nullptr);
  if (tensor_on(p)) bytes += carve_list(p, kTensorList, nullptr, nullptr);
  return bytes;
}

cudaError_t launch_chunk(const fgw_chunk_params& p, void* workspace, int sm_count, int device, cudaStream_t stream) {
  ChunkPlanArgs plan = {};
  plan.on[kDecodeList] = decode_on(p);
  plan.on[kTensorList] = tensor_on(p);
  plan.split = plan.on[kDecodeList] && plan.on[kTensorList];
  plan.row_bytes = p.heads * p.head_dim * 2;
  ChunkArgs a = {};
  a.out = p.out;
  a.table = p.block_table;
  a.lens = p.cache_seqlens;
  a.cu = p.cu_seqlens_q;
  a.q = p.q;
  a.ws = static_cast<WorkspaceHeader*>(workspace);
  a.tokens = p.tokens;
  a.q_stride = p.q_stride;
  a.out_stride = p.out_stride;
  a.batch = p.batch;
  a.heads = p.heads;
  a.kv_heads = p.kv_heads;
  a.group = p.heads / p.kv_heads;
  a.dim = p.head_dim;
  a.width = p.table_width;
  a.page = p.page_size;
  a.causal = p.causal;
  a.programs = std::min(sm_count, kStreamMaxPrograms);
  a.scale_log2 = p.softmax_scale * kLog2e;
  a.budget_ns = static_cast<uint64_t>(p.wait_budget_ms > 0 ? p.wait_budget_ms : 2000) * 1000000ull;
  uint8_t* at = static_cast<uint8_t*>(workspace) + sizeof(WorkspaceHeader);
  for (int cls = 0; cls < 2; ++cls) {
    plan.a[cls] = a;
    if (plan.on[cls]) at += carve_list(p, cls, at, &plan.a[cls].list);
  }
  chunk_plan_kernel<<<plan.split ? 2 : 1, kPlanListThreads, 0, stream>>>(plan);
  cudaError_t err = cudaGetLastError();
  if (err == cudaSuccess && plan.on[kDecodeList]) err = launch_chunk_decode(p, plan.a[kDecodeList], device, stream);
  if (err == cudaSuccess && plan.on[kTensorList]) err = launch_chunk_tensor(p, plan.a[kTensorList], device, stream);
  return err;
}

}  // namespace fgw
