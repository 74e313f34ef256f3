// Page-table operators of a paged KV cache: fork (share, copy on write, reserve, free), compact and copy
// (fgw_page_fork, fgw_page_compact, fgw_page_copy in include/fgw_mha.h).
//
// The table and the lengths alone say which pages are live: row b holds the first ceil(len[b] / page) entries of
// its row, and a page that no row holds is free. So there are no counts or free lists that could disagree with the
// table, and a row is freed by giving it no parent.
//
// One cluster of eight CTAs does the bookkeeping (page_plan_kernel): it marks the held pages in a bitmap, ranks the
// free pages by a prefix sum over the bitmap, hands them out in (row, column) order and leaves a list of the pages to
// copy. All of it is integer work in a fixed order (atomics only where the order cannot show: OR, MIN, ADD of counts),
// so results do not depend on timing. It is bound by latency: a chain of cluster barriers, each around one or two
// round trips to L2. page_copy_kernel then moves the bytes, bound by HBM.
#include <cooperative_groups.h>

#include <algorithm>

#include "fgw_common.cuh"
#include "fgw_kernels.h"

namespace cg = cooperative_groups;

namespace fgw {

constexpr int kPlanCtas = 8;       // one portable cluster
constexpr int kPlanThreads = 512;
constexpr int kBlockWords = 32;    // bitmap words ranked together by one warp (1024 pages)
constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 4;
constexpr int kPoolsPerLaunch = 224;  // pool pointers passed by value in one copy launch

struct PageCopy {
  int32_t src, dst, rows;  // rows: token rows of the page to copy; <= 0 skips the entry
};

// Workspace: copy list | copy count and totals | bitmap | per-block ranks | free list | row arrays.
struct PageWs {
  PageCopy* copies;
  int32_t* totals;   // [0] copies, [1] needed pages, [2] free pages, [3] moved pages
  uint32_t* used;    // bitmap of the held pages
  int32_t* blocks;   // free pages before each block of 1024 pages, exclusive
  int32_t* list;     // fork: free pages in order; compact: holes, then new ids of the moved pages
  int32_t* first;    // [batch] first row with this parent
  int32_t* need;     // [batch + 1] new pages of each row, then their exclusive prefix
};

struct PageArgs {
  const int32_t* table;
  const int32_t* lens;
  const int32_t* parents;
  const int32_t* reserve;
  int32_t* table_out;
  int32_t* lens_out;
  int32_t* status;
  PageWs ws;
  int batch, width, page, pages, words, blocks;
};

static size_t align256(size_t n) { return (n + 255) & ~size_t(255); }

static size_t carve_pages(const fgw_page_params& p, void* base, PageWs* ws) {
  uint8_t* at = static_cast<uint8_t*>(base);
  const size_t words = (static_cast<size_t>(p.num_pages) + 31) / 32;
  const size_t blocks = (words + kBlockWords - 1) / kBlockWords;
  const size_t copies = std::max<size_t>(p.batch, p.num_pages / 2 + 1);
  auto take = [&](size_t n) {
    uint8_t* here = at;
    at += align256(n);
    return here;
  };
  PageWs w;
  w.totals = reinterpret_cast<int32_t*>(take(64));
  w.copies = reinterpret_cast<PageCopy*>(take(copies * sizeof(PageCopy)));
  w.used = reinterpret_cast<uint32_t*>(take(blocks * kBlockWords * 4));
  w.blocks = reinterpret_cast<int32_t*>(take((blocks + 1) * 4));
  w.list = reinterpret_cast<int32_t*>(take(2 * static_cast<size_t>(p.num_pages) * 4));
  w.first = reinterpret_cast<int32_t*>(take(static_cast<size_t>(p.batch) * 4));
  w.need = reinterpret_cast<int32_t*>(take((static_cast<size_t>(p.batch) + 1) * 4));
  if (ws != nullptr) *ws = w;
  return static_cast<size_t>(at - static_cast<uint8_t*>(base));
}

// What row i becomes: its parent (-1: freed), tokens, entries it takes over and entries it shall have.
struct ForkRow {
  int parent, len, full, held, want;
};

__device__ __forceinline__ int clamped_len(const PageArgs& a, int len) {
  const long long cap = static_cast<long long>(a.width) * a.page;
  return static_cast<int>(min(static_cast<long long>(max(len, 0)), cap));
}

__device__ __forceinline__ ForkRow fork_row(const PageArgs& a, int i) {
  ForkRow r;
  r.parent = a.parents[i];
  if (r.parent < 0 || r.parent >= a.batch) {
    r.parent = -1;
    r.len = r.full = r.held = r.want = 0;
    return r;
  }
  r.len = clamped_len(a, a.lens[r.parent]);
  const int room = a.reserve != nullptr ? max(clamped_len(a, a.reserve[i]), r.len) : r.len;
  r.full = r.len / a.page;
  r.held = (r.len + a.page - 1) / a.page;
  r.want = room / a.page + (room % a.page != 0);
  return r;
}

__device__ __forceinline__ void mark_row(const PageArgs& a, int row, int held, int lane, int lanes) {
  const int32_t* entries = a.table + static_cast<long long>(row) * a.width;
  for (int w = lane; w < held; w += lanes) {
    const int id = entries[w];
    if (id >= 0 && id < a.pages) atomicOr(&a.ws.used[id >> 5], 1u << (id & 31));
  }
}

// Exclusive prefix sum of x[0, n) in place by one CTA; returns the total to every thread.
__device__ int cta_exclusive_scan(int32_t* x, int n, int* shared) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int carry = 0;
  for (int base = 0; base < n; base += blockDim.x) {
    const int i = base + threadIdx.x;
    const int v = i < n ? x[i] : 0;
    int sum = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += up;
    }
    if (lane == 31) shared[warp] = sum;
    __syncthreads();
    int before = carry, all = carry;
    for (int w = 0; w < warps; ++w) {
      if (w < warp) before += shared[w];
      all += shared[w];
    }
    if (i < n) x[i] = before + sum - v;
    carry = all;
    __syncthreads();
  }
  return carry;
}

template <bool kFork>
__global__ void __cluster_dims__(kPlanCtas, 1, 1) __launch_bounds__(kPlanThreads) page_plan_kernel(const PageArgs a) {
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ int shared[32];
  const int tid = blockIdx.x * kPlanThreads + threadIdx.x;
  constexpr int kThreads = kPlanCtas * kPlanThreads;
  const int lane = threadIdx.x & 31;
  const int warp = tid >> 5;
  constexpr int kWarps = kThreads / 32;
  const int padded_words = a.blocks * kBlockWords;

  // Nothing held, no first rows. Bits past the last page count as held, so they are never handed out.
  for (int w = tid; w < padded_words; w += kThreads) {
    const long long first_page = 32ll * w;
    uint32_t bits = 0;
    if (first_page + 32 > a.pages) bits = first_page >= a.pages ? 0xffffffffu : 0xffffffffu << (a.pages & 31);
    a.ws.used[w] = bits;
  }
  if (kFork) {
    for (int i = tid; i < a.batch; i += kThreads) a.ws.first[i] = a.batch;
  }
  if (tid < 4) a.ws.totals[tid] = 0;
  cluster.sync();
  if (kFork) {
    for (int i = tid; i < a.batch; i += kThreads) {
      const int parent = a.parents[i];
      if (parent >= 0 && parent < a.batch) atomicMin(&a.ws.first[parent], i);
    }
    cluster.sync();
  }
  // The held pages; of the rows with one parent only the first marks.
  for (int i = warp; i < a.batch; i += kWarps) {
    if (kFork) {
      const ForkRow r = fork_row(a, i);
      const bool is_first = r.parent >= 0 && __ldcg(&a.ws.first[r.parent]) == i;
      if (is_first) mark_row(a, r.parent, r.held, lane, 32);
      const int copy = r.parent >= 0 && !is_first && r.len > r.full * a.page;
      if (lane == 0) a.ws.need[i] = copy + r.want - r.held;
    } else {
      const int len = clamped_len(a, a.lens[i]);
      mark_row(a, i, len / a.page + (len % a.page != 0), lane, 32);
    }
  }
  cluster.sync();
  for (int b = warp; b < a.blocks; b += kWarps) {
    const int free_here = 32 - __popc(__ldcg(&a.ws.used[b * kBlockWords + lane]));
    const int sum = __reduce_add_sync(0xffffffffu, free_here);
    if (lane == 0) a.ws.blocks[b] = sum;
  }
  cluster.sync();
  if (blockIdx.x == 0) {
    const int free_pages = cta_exclusive_scan(a.ws.blocks, a.blocks, shared);
    if (threadIdx.x == 0) a.ws.totals[2] = free_pages;
  } else if (kFork && blockIdx.x == 1) {
    const int needed = cta_exclusive_scan(a.ws.need, a.batch, shared);
    if (threadIdx.x == 0) a.ws.totals[1] = needed;
  }
  cluster.sync();
  const int free_pages = __ldcg(&a.ws.totals[2]);
  const int live = a.pages - free_pages;
  const int needed = kFork ? __ldcg(&a.ws.totals[1]) : 0;
  // Fork: the first `needed` free pages in order. Compact: the free pages below `live` (list[rank]) and the held
  // pages from `live` on, which are the last in the order of held pages (list[pages + live - 1 - rank]).
  for (int b = warp; b < a.blocks; b += kWarps) {
    int rank = __ldcg(&a.ws.blocks[b]);
    if (kFork && rank >= needed) continue;
    const int w = b * kBlockWords + lane;
    const uint32_t used = __ldcg(&a.ws.used[w]);
    const int free_here = 32 - __popc(used);
    int sum = free_here;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += up;
    }
    rank += sum - free_here;
    for (int bit = 0; bit < 32; ++bit) {
      const int id = w * 32 + bit;
      if ((used >> bit & 1) == 0) {
        if (kFork ? rank < needed : id < live) a.ws.list[rank] = id;
        ++rank;
      } else if (!kFork && id >= live && id < a.pages) {
        const int held_rank = id - rank;  // held pages before this one
        a.ws.list[a.pages + live - 1 - held_rank] = id;
        atomicAdd(&a.ws.totals[3], 1);
      }
    }
  }
  cluster.sync();
  if (kFork) {
    const bool fits = needed <= free_pages;
    for (int i = warp; i < a.batch; i += kWarps) {
      const ForkRow r = fork_row(a, i);
      int32_t* out = a.table_out + static_cast<long long>(i) * a.width;
      if (!fits) {  // the state stays as it was
        const int32_t* in = a.table + static_cast<long long>(i) * a.width;
        for (int w = lane; w < a.width; w += 32) out[w] = in[w];
        if (lane == 0) a.lens_out[i] = a.lens[i];
        continue;
      }
      const int32_t* in = a.table + static_cast<long long>(max(r.parent, 0)) * a.width;
      const bool copies = r.parent >= 0 && r.len > r.full * a.page && __ldcg(&a.ws.first[r.parent]) != i;
      const int kept = copies ? r.full : r.held;  // entries taken over as they are
      const int base = __ldcg(&a.ws.need[i]);
      for (int w = lane; w < a.width; w += 32) {
        out[w] = w < kept ? in[w] : (w < r.want ? __ldcg(&a.ws.list[base + w - kept]) : -1);
      }
      if (lane == 0) {
        a.lens_out[i] = r.len;
        if (copies) {
          const int src = in[r.full];
          const int at = atomicAdd(&a.ws.totals[0], 1);
          a.ws.copies[at] = {src, __ldcg(&a.ws.list[base]), src >= 0 && src < a.pages ? r.len - r.full * a.page : 0};
        }
      }
    }
    if (tid == 0) {
      a.status[0] = needed;
      a.status[1] = free_pages;
    }
  } else {
    const int moved = __ldcg(&a.ws.totals[3]);
    const int32_t* movers = a.ws.list + a.pages;  // [k] = the (moved - 1 - k)-th moved page
    for (int k = tid; k < moved; k += kThreads) {
      const int src = __ldcg(&movers[moved - 1 - k]);
      a.ws.copies[k] = {src, __ldcg(&a.ws.list[k]), a.page};
    }
    if (tid == 0) {
      a.ws.totals[0] = moved;
      a.status[0] = live;
      a.status[1] = moved;
    }
    cluster.sync();
    for (int i = warp; i < a.batch; i += kWarps) {
      const int len = clamped_len(a, a.lens[i]);
      const int held = len / a.page + (len % a.page != 0);
      const int32_t* in = a.table + static_cast<long long>(i) * a.width;
      int32_t* out = a.table_out + static_cast<long long>(i) * a.width;
      for (int w = lane; w < a.width; w += 32) {
        int id = w < held ? in[w] : -1;
        if (id >= live && id < a.pages) {
          // the moved pages are in order in copies[].src: the k-th goes to the k-th hole
          int lo = 0, hi = moved - 1;
          while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (__ldcg(&a.ws.copies[mid].src) < id) {
              lo = mid + 1;
            } else {
              hi = mid;
            }
          }
          id = __ldcg(&a.ws.copies[lo].dst);
        }
        out[w] = id;
      }
    }
  }
}

struct PoolList {
  void* at[kPoolsPerLaunch];
};

// Copies the listed pages' rows in every pool, 16 KB of one page at a time. Sources and destinations are distinct
// pages (held and free ones), so the order of the copies does not matter.
__global__ void __launch_bounds__(kCopyThreads)
    page_copy_kernel(const __grid_constant__ PoolList pools, int pool_count, const PageCopy* list,
                     const int32_t* list_count, long long page_units, long long row_units) {
  constexpr int kChunk = kCopyThreads * kCopyUnroll;
  const long long chunks = (page_units + kChunk - 1) / kChunk;
  const long long units = static_cast<long long>(*list_count) * pool_count * chunks;
  for (long long u = blockIdx.x; u < units; u += gridDim.x) {
    const long long chunk = u % chunks;
    const long long rest = u / chunks;
    const int pool = static_cast<int>(rest % pool_count);
    const PageCopy c = list[rest / pool_count];
    const long long end = c.rows * row_units;
    uint4* base = static_cast<uint4*>(pools.at[pool]);
    const uint4* src = base + c.src * page_units;
    uint4* dst = base + c.dst * page_units;
    const long long first = chunk * kChunk + threadIdx.x;
    uint4 v[kCopyUnroll];
#pragma unroll
    for (int k = 0; k < kCopyUnroll; ++k) {
      if (first + k * kCopyThreads < end) v[k] = __ldcs(&src[first + k * kCopyThreads]);
    }
#pragma unroll
    for (int k = 0; k < kCopyUnroll; ++k) {
      if (first + k * kCopyThreads < end) __stcs(&dst[first + k * kCopyThreads], v[k]);
    }
  }
}

// The caller's page lists as a copy list: entries with a page outside the pool are skipped.
__global__ void page_list_kernel(const int32_t* src, const int32_t* dst, int n, int pages, int page, PageCopy* list,
                                 int32_t* count) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i == 0) *count = n;
  if (i >= n) return;
  const int s = src[i], d = dst[i];
  list[i] = {s, d, s >= 0 && s < pages && d >= 0 && d < pages && s != d ? page : 0};
}

static cudaError_t launch_copies(const fgw_page_params& p, const PageCopy* list, const int32_t* count, int sm_count,
                                 cudaStream_t stream) {
  const long long row_units = p.row_bytes / 16;
  for (int at = 0; at < p.pool_count; at += kPoolsPerLaunch) {
    const int n = std::min(kPoolsPerLaunch, p.pool_count - at);
    PoolList pools;
    for (int i = 0; i < kPoolsPerLaunch; ++i) pools.at[i] = i < n ? p.pools[at + i] : nullptr;
    page_copy_kernel<<<8 * sm_count, kCopyThreads, 0, stream>>>(pools, n, list, count, row_units * p.page_size,
                                                                row_units);
    const cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return err;
  }
  return cudaSuccess;
}

int page_validate(const fgw_page_params& p, int op) {
  for (int r : p.reserved) {
    if (r != 0) return FGW_ERR_INVALID_ARGUMENT;
  }
  if (p.pool_count < 0 || p.num_pages <= 0 || p.page_size <= 0) return FGW_ERR_INVALID_ARGUMENT;
  if (static_cast<long long>(p.num_pages) > (1ll << 30)) return FGW_ERR_INVALID_ARGUMENT;
  if (p.pool_count > 0) {
    if (p.pools == nullptr || p.row_bytes <= 0 || p.row_bytes % 16 != 0) return FGW_ERR_INVALID_ARGUMENT;
    for (int i = 0; i < p.pool_count; ++i) {
      if (p.pools[i] == nullptr || reinterpret_cast<uintptr_t>(p.pools[i]) % 16 != 0) return FGW_ERR_INVALID_ARGUMENT;
    }
  }
  if (op == kPageCopy) {
    if (p.copy_count < 0 || (p.copy_count > 0 && (p.src_pages == nullptr || p.dst_pages == nullptr))) {
      return FGW_ERR_INVALID_ARGUMENT;
    }
    return FGW_OK;
  }
  if (p.batch <= 0 || p.table_width <= 0) return FGW_ERR_INVALID_ARGUMENT;
  if (static_cast<long long>(p.page_size) * p.table_width > 0x7fffffffll) return FGW_ERR_INVALID_ARGUMENT;
  if (static_cast<long long>(p.batch) * p.table_width > 0x7fffffffll) return FGW_ERR_INVALID_ARGUMENT;
  if (p.block_table == nullptr || p.cache_seqlens == nullptr || p.table_out == nullptr || p.status == nullptr ||
      p.table_out == p.block_table) {
    return FGW_ERR_INVALID_ARGUMENT;
  }
  if (op == kPageFork &&
      (p.parents == nullptr || p.seqlens_out == nullptr || p.seqlens_out == p.cache_seqlens)) {
    return FGW_ERR_INVALID_ARGUMENT;
  }
  return FGW_OK;
}

size_t page_workspace_bytes(const fgw_page_params& p, int op) {
  if (op == kPageCopy) return 256 + align256(static_cast<size_t>(p.copy_count) * sizeof(PageCopy));
  return carve_pages(p, nullptr, nullptr);
}

cudaError_t launch_page_op(const fgw_page_params& p, int op, void* workspace, int sm_count, cudaStream_t stream) {
  if (op == kPageCopy) {
    if (p.copy_count == 0 || p.pool_count == 0) return cudaSuccess;
    int32_t* count = static_cast<int32_t*>(workspace);
    PageCopy* list = reinterpret_cast<PageCopy*>(static_cast<uint8_t*>(workspace) + 256);
    page_list_kernel<<<(p.copy_count + 255) / 256, 256, 0, stream>>>(p.src_pages, p.dst_pages, p.copy_count,
                                                                     p.num_pages, p.page_size, list, count);
    const cudaError_t err = cudaGetLastError();
    return err != cudaSuccess ? err : launch_copies(p, list, count, sm_count, stream);
  }
  PageArgs a;
  carve_pages(p, workspace, &a.ws);
  a.table = p.block_table;
  a.lens = p.cache_seqlens;
  a.parents = p.parents;
  a.reserve = p.reserve_seqlens;
  a.table_out = p.table_out;
  a.lens_out = p.seqlens_out;
  a.status = p.status;
  a.batch = p.batch;
  a.width = p.table_width;
  a.page = p.page_size;
  a.pages = p.num_pages;
  a.words = (p.num_pages + 31) / 32;
  a.blocks = (a.words + kBlockWords - 1) / kBlockWords;
  if (op == kPageFork) {
    page_plan_kernel<true><<<kPlanCtas, kPlanThreads, 0, stream>>>(a);
  } else {
    page_plan_kernel<false><<<kPlanCtas, kPlanThreads, 0, stream>>>(a);
  }
  const cudaError_t err = cudaGetLastError();
  return err != cudaSuccess ? err : launch_copies(p, a.ws.copies, a.ws.totals, sm_count, stream);
}

}  // namespace fgw
