// Page-table operators of a paged KV cache: fork (share, copy on write, reserve, free), compact and copy
// (fgw_page_fork, fgw_page_compact, fgw_page_copy in include/fgw_mha.h).
//
// The table and the lengths alone say which pages are live: row b holds the first ceil(len[b] / page) entries of
// its row, and a page that no row holds is free. So there are no counts or free lists that could disagree with the
// table, and a row is freed by giving it no parent.
//
// page_plan_kernel does the bookkeeping: it marks the held pages in a bitmap, ranks the free pages by a prefix sum over
// the bitmap, hands them out in (row, column) order and leaves a list of the pages to copy. All of it is integer work in
// a fixed order (atomics only where the order cannot show: OR, MIN, ADD of counts), so results do not depend on timing.
// It is bound by latency: a chain of barriers, each around one or two round trips to L2. Tables of up to 32K entries over
// up to 128K pages are one CTA's work with the bitmap and the row arrays in shared memory; larger ones go to a cluster
// of eight CTAs over global memory (eight rows over one layer: 9.7 against 11.8 us with the copy). page_copy_kernel then
// moves the bytes, bound by HBM; it is launched beside the plan and waits for it. Measured: 700 pages of 128 KB in 8 pools
// (1.47 GB read and written) 257 us, 5.7 TB/s; 55 half-filled pages in 16 pools 28 us, of which the plan takes 10. That
// ends which other rows hold are told from ends that only forks of one row share is a second bitmap: no time that shows.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "fgw_common.cuh"
#include "fgw_kernels.h"
#include "fgw_ragged.cuh"

namespace cg = cooperative_groups;

namespace fgw {

constexpr int kPlanCtas = 8;       // one portable cluster
constexpr int kPlanThreads = 1024;
constexpr int kSmallPages = 1 << 17, kSmallRows = 4096, kSmallEntries = 1 << 15;  // one CTA's share
constexpr int kPlanLoads = 4;
// The plan's loops count entries and rows in 32 bits and step by up to all threads' loads past the last one.
static_assert(FGW_PAGE_MAX_ENTRIES + 1ll * kPlanCtas * kPlanThreads * kPlanLoads <= 0x7fffffffll, "loops over a table");
constexpr int kBlockWords = 32;    // bitmap words ranked together by one warp (1024 pages)
constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 8;  // 32 KB of a page per step: 257 us against 263 with 16 KB (1.47 GB moved)
constexpr int kPoolsPerLaunch = 224;  // pool pointers passed by value in one copy launch

struct PageCopy {
  int32_t src, dst, rows;  // rows: token rows of the page to copy; <= 0 skips the entry
};

// Workspace: copy count and totals | copy list | bitmaps | per-block ranks | free list | row arrays.
struct PageWs {
  PageCopy* copies;
  int32_t* totals;   // [0] copies, [1] needed pages, [2] free pages, [3] moved pages
  uint32_t* used;    // bitmap of the held pages; fork: of those that hold a row's partly filled end
  uint32_t* shut;    // fork: bitmap of the pages that no row may keep as its partly filled end
  int32_t* blocks;   // free pages before each block of 1024 pages, exclusive
  int32_t* list;     // fork: free pages in order; compact: holes, moved pages (last first), then new ids by page
  int32_t* first;    // [batch] first row with this parent
  int32_t* need;     // [batch + 1] new pages of each row, then their exclusive prefix
  int4* rows;        // [batch] what each row becomes: {parent, entries kept, entries wanted, entries held}; until the
                     // copies are known, fork's entries kept are the full ones
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
  FastDiv by_width;
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
  w.shut = reinterpret_cast<uint32_t*>(take(blocks * kBlockWords * 4));
  w.blocks = reinterpret_cast<int32_t*>(take((blocks + 1) * 4));
  w.list = reinterpret_cast<int32_t*>(take(3 * static_cast<size_t>(p.num_pages) * 4));
  w.first = reinterpret_cast<int32_t*>(take(static_cast<size_t>(p.batch) * 4));
  w.need = reinterpret_cast<int32_t*>(take((static_cast<size_t>(p.batch) + 1) * 4));
  w.rows = reinterpret_cast<int4*>(take(static_cast<size_t>(p.batch) * 16));
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

// Exclusive prefix sum of x[0, n) in place by one CTA; returns the total to every thread.
template <typename Load>
__device__ int cta_exclusive_scan(int32_t* x, int n, int* shared, Load load) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int carry = 0;
  for (int base = 0; base < n; base += blockDim.x) {
    const int i = base + threadIdx.x;
    const int v = i < n ? load(&x[i]) : 0;
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

// Scratch of the one-CTA form in shared memory.
struct SmallWs {
  int32_t totals[4];
  uint32_t used[kSmallPages / 32];
  uint32_t shut[kSmallPages / 32];
  int32_t blocks[kSmallPages / (32 * kBlockWords) + 1];
  int32_t first[kSmallRows];
  int32_t need[kSmallRows + 1];
  alignas(16) int4 rows[kSmallRows];
};

template <bool kFork, int kCtas>
__device__ __forceinline__ void page_plan(PageArgs a, int* shared) {
  extern __shared__ uint8_t plan_smem[];
  if constexpr (kCtas == 1) {
    SmallWs& small = *reinterpret_cast<SmallWs*>(plan_smem);
    a.ws.used = small.used;
    a.ws.shut = small.shut;
    a.ws.blocks = small.blocks;
    a.ws.first = small.first;
    a.ws.need = small.need;
    a.ws.rows = small.rows;
  }
  int32_t* totals = kCtas == 1 ? reinterpret_cast<SmallWs*>(plan_smem)->totals : a.ws.totals;
  auto sync = [&]() {
    if constexpr (kCtas == 1) {
      __syncthreads();
    } else {
      cg::this_cluster().sync();
    }
  };
  // what other threads have written since the last barrier, past this SM's L1
  auto fresh = [&](const auto* x) {
    if constexpr (kCtas == 1) {
      return *const_cast<const volatile std::remove_reference_t<decltype(*x)>*>(x);
    } else {
      return __ldcg(x);
    }
  };
  const int tid = blockIdx.x * kPlanThreads + threadIdx.x;
  constexpr int kThreads = kCtas * kPlanThreads;
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
    if (kFork) a.ws.shut[w] = 0;
  }
  if (tid < 4) totals[tid] = 0;
  for (int i = tid; i < a.batch; i += kThreads) {
    if (kFork) {
      a.ws.first[i] = a.batch;
      const ForkRow r = fork_row(a, i);
      a.ws.rows[i] = make_int4(r.parent, r.full, r.want, r.held);
    } else {
      const int len = clamped_len(a, a.lens[i]);
      a.ws.rows[i] = make_int4(i, 0, 0, len / a.page + (len % a.page != 0));
    }
  }
  sync();
  if (kFork) {
    for (int i = tid; i < a.batch; i += kThreads) {
      const int parent = fresh(&a.ws.rows[i].x);
      if (parent >= 0) atomicMin(&a.ws.first[parent], i);
    }
    sync();
  }
  // The held pages; of the rows with one parent only the first marks. Table entries are taken flat, four loads of a
  // thread at a time. A partly filled end may stay with its row only if no other parent's row, and no other entry of its
  // own, holds that page: full pages shut it, and so does the second end on one page, whichever of them comes second.
  const int entries = a.batch * a.width;
  for (int base = tid; base < entries; base += kThreads * kPlanLoads) {
    int ids[kPlanLoads];
    bool full[kPlanLoads];  // fork: a full page's entry
#pragma unroll
    for (int u = 0; u < kPlanLoads; ++u) {
      ids[u] = -1;
      const long long at = base + static_cast<long long>(u) * kThreads;
      if (at >= entries) continue;
      const int i = a.by_width.quotient(static_cast<int>(at)), w = static_cast<int>(at) - i * a.width;
      const int parent = fresh(&a.ws.rows[i].x), held = fresh(&a.ws.rows[i].w);
      if (w >= held || (kFork && fresh(&a.ws.first[parent]) != i)) continue;  // held is 0 without a parent
      ids[u] = a.table[static_cast<long long>(parent) * a.width + w];
      full[u] = kFork && w < fresh(&a.ws.rows[i].y);
    }
#pragma unroll
    for (int u = 0; u < kPlanLoads; ++u) {
      if (ids[u] < 0 || ids[u] >= a.pages) continue;
      const int word = ids[u] >> 5;
      const uint32_t bit = 1u << (ids[u] & 31);
      if (!kFork) {
        atomicOr(&a.ws.used[word], bit);
      } else if (full[u] || (atomicOr(&a.ws.used[word], bit) & bit) != 0) {
        atomicOr(&a.ws.shut[word], bit);
      }
    }
  }
  sync();
  auto held_pages = [&](int word) {
    uint32_t bits = fresh(&a.ws.used[word]);
    if (kFork) bits |= fresh(&a.ws.shut[word]);
    return bits;
  };
  if (kFork) {
    for (int i = tid; i < a.batch; i += kThreads) {
      const int parent = fresh(&a.ws.rows[i].x), full = fresh(&a.ws.rows[i].y), held = fresh(&a.ws.rows[i].w);
      bool copies = false;
      if (held > full) {
        const int end = a.table[static_cast<long long>(parent) * a.width + full];
        copies = fresh(&a.ws.first[parent]) != i ||
                 (end >= 0 && end < a.pages && (fresh(&a.ws.shut[end >> 5]) >> (end & 31) & 1) != 0);
      }
      a.ws.need[i] = (copies ? 1 : 0) + fresh(&a.ws.rows[i].z) - held;
      if (!copies) a.ws.rows[i].y = held;
    }
  }
  for (int b = warp; b < a.blocks; b += kWarps) {
    const int free_here = 32 - __popc(held_pages(b * kBlockWords + lane));
    const int sum = __reduce_add_sync(0xffffffffu, free_here);
    if (lane == 0) a.ws.blocks[b] = sum;
  }
  sync();
  if (blockIdx.x == 0) {
    const int free_pages = cta_exclusive_scan(a.ws.blocks, a.blocks, shared, fresh);
    if (threadIdx.x == 0) totals[2] = free_pages;
  }
  if (kFork && blockIdx.x == (kCtas > 1 ? 1 : 0)) {
    const int needed = cta_exclusive_scan(a.ws.need, a.batch, shared, fresh);
    if (threadIdx.x == 0) totals[1] = needed;
  }
  sync();
  const int free_pages = fresh(&totals[2]);
  const int live = a.pages - free_pages;
  const int needed = kFork ? fresh(&totals[1]) : 0;
  // Fork: the first `needed` free pages in order. Compact: the free pages below `live` (list[rank]) and the held
  // pages from `live` on, which are the last in the order of held pages (list[pages + live - 1 - rank]).
  for (int b = warp; b < a.blocks; b += kWarps) {
    int rank = fresh(&a.ws.blocks[b]);
    if (kFork && rank >= needed) continue;
    const int w = b * kBlockWords + lane;
    const uint32_t used = held_pages(w);
    const int free_here = 32 - __popc(used);
    int sum = free_here;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += up;
    }
    rank += sum - free_here;
    int moves = 0;
    for (int bit = 0; bit < 32; ++bit) {
      const int id = w * 32 + bit;
      if ((used >> bit & 1) == 0) {
        if (kFork ? rank < needed : id < live) a.ws.list[rank] = id;
        ++rank;
      } else if (!kFork && id >= live && id < a.pages) {
        const int held_rank = id - rank;  // held pages before this one
        a.ws.list[a.pages + live - 1 - held_rank] = id;
        ++moves;
      }
    }
    if (!kFork) {
      moves = __reduce_add_sync(0xffffffffu, moves);
      if (lane == 0 && moves > 0) atomicAdd(&totals[3], moves);
    }
  }
  sync();
  const bool fits = needed <= free_pages;  // else the state stays as it was
  const int moved = kFork ? 0 : fresh(&totals[3]);
  int32_t* new_id = a.ws.list + 2ll * a.pages;
  if (kFork) {
    for (int i = tid; i < a.batch; i += kThreads) {
      const ForkRow r = fork_row(a, i);
      a.lens_out[i] = fits ? r.len : a.lens[i];
      if (!fits || r.held == r.full || fresh(&a.ws.rows[i].y) == r.held) continue;  // nothing to copy
      const int src = a.table[static_cast<long long>(r.parent) * a.width + r.full];
      const int dst = __ldcg(&a.ws.list[fresh(&a.ws.need[i])]);
      const int at = atomicAdd(&totals[0], 1);
      a.ws.copies[at] = {src, dst, src >= 0 && src < a.pages ? r.len - r.full * a.page : 0};
    }
    if (tid == 0) {
      a.status[0] = needed;
      a.status[1] = free_pages;
    }
  } else {
    const int32_t* movers = a.ws.list + a.pages;  // [k] = the (moved - 1 - k)-th moved page
    for (int k = tid; k < moved; k += kThreads) {
      const int src = __ldcg(&movers[moved - 1 - k]), dst = __ldcg(&a.ws.list[k]);
      a.ws.copies[k] = {src, dst, a.page};
      new_id[src] = dst;
    }
    if (tid == 0) {
      a.ws.totals[0] = moved;
      a.status[0] = live;
      a.status[1] = moved;
    }
    sync();
  }
  for (int base = tid; base < entries; base += kThreads * kPlanLoads) {
    int ids[kPlanLoads];
#pragma unroll
    for (int u = 0; u < kPlanLoads; ++u) {
      ids[u] = -1;
      const long long at = base + static_cast<long long>(u) * kThreads;
      if (at >= entries) continue;
      const int i = a.by_width.quotient(static_cast<int>(at)), w = static_cast<int>(at) - i * a.width;
      if (kFork && !fits) {
        ids[u] = a.table[at];
        continue;
      }
      const int parent = fresh(&a.ws.rows[i].x);
      const int kept = kFork ? fresh(&a.ws.rows[i].y) : fresh(&a.ws.rows[i].w);  // taken over as they are
      if (w < kept) {
        ids[u] = a.table[static_cast<long long>(parent) * a.width + w];
      } else if (kFork && w < fresh(&a.ws.rows[i].z)) {
        ids[u] = __ldcg(&a.ws.list[fresh(&a.ws.need[i]) + w - kept]);
      }
    }
#pragma unroll
    for (int u = 0; u < kPlanLoads; ++u) {
      const long long at = base + static_cast<long long>(u) * kThreads;
      if (at >= entries) continue;
      if (!kFork && ids[u] >= live && ids[u] < a.pages) ids[u] = __ldcg(&new_id[ids[u]]);
      a.table_out[at] = ids[u];
    }
  }
  if (kFork && kCtas == 1) {
    sync();
    if (tid == 0) a.ws.totals[0] = totals[0];
  }
}

template <bool kFork>
__global__ void __cluster_dims__(kPlanCtas, 1, 1) __launch_bounds__(kPlanThreads) page_plan_kernel(const PageArgs a) {
  __shared__ int shared[32];
  grid_dependents_launch();
  page_plan<kFork, kPlanCtas>(a, shared);
}
template <bool kFork>
__global__ void __launch_bounds__(kPlanThreads) page_plan_small_kernel(const PageArgs a) {
  __shared__ int shared[32];
  grid_dependents_launch();
  page_plan<kFork, 1>(a, shared);
}

struct PoolList {
  void* at[kPoolsPerLaunch];
};

// Copies the listed pages' rows in every pool, 32 KB of one page at a time. Sources and destinations are distinct
// pages (held and free ones), so the order of the copies does not matter.
__global__ void __launch_bounds__(kCopyThreads)
    page_copy_kernel(const __grid_constant__ PoolList pools, int pool_count, const PageCopy* list,
                     const int32_t* list_count, long long page_units, long long row_units) {
  constexpr int kChunk = kCopyThreads * kCopyUnroll;
  grid_dependency_wait();  // the plan's list
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
__global__ void __launch_bounds__(256) page_list_kernel(const int32_t* src, const int32_t* dst, int n, int pages, int page, PageCopy* list,
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
    // the first waits for the plan only where it runs; the others follow it in stream order
    cudaError_t err;
    if (at == 0) {
      err = launch_after_plan(page_copy_kernel, 8 * sm_count, kCopyThreads, 0, stream, pools, n, list, count,
                              row_units * p.page_size, row_units);
    } else {
      page_copy_kernel<<<8 * sm_count, kCopyThreads, 0, stream>>>(pools, n, list, count, row_units * p.page_size,
                                                                  row_units);
      err = cudaGetLastError();
    }
    if (err != cudaSuccess) return err;
  }
  return cudaSuccess;
}

template <bool kFork>
static cudaError_t launch_plan_op(const PageArgs& a, int device, cudaStream_t stream) {
  const bool small = a.pages <= kSmallPages && a.batch <= kSmallRows &&
                     static_cast<long long>(a.batch) * a.width <= kSmallEntries;
  if (!small) {
    page_plan_kernel<kFork><<<kPlanCtas, kPlanThreads, 0, stream>>>(a);
    return cudaGetLastError();
  }
  auto kernel = page_plan_small_kernel<kFork>;
  const cudaError_t err = prepare_kernel(reinterpret_cast<const void*>(kernel), sizeof(SmallWs), device, nullptr);
  if (err != cudaSuccess) return err;
  kernel<<<1, kPlanThreads, sizeof(SmallWs), stream>>>(a);
  return cudaGetLastError();
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
  if (static_cast<long long>(p.batch) * p.table_width > FGW_PAGE_MAX_ENTRIES) return FGW_ERR_INVALID_ARGUMENT;
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

cudaError_t launch_page_op(const fgw_page_params& p, int op, void* workspace, int sm_count, int device,
                           cudaStream_t stream) {
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
  a.by_width = FastDiv(p.table_width);
  a.words = (p.num_pages + 31) / 32;
  a.blocks = (a.words + kBlockWords - 1) / kBlockWords;
  const cudaError_t err = op == kPageFork ? launch_plan_op<true>(a, device, stream) : launch_plan_op<false>(a, device, stream);
  return err != cudaSuccess ? err : launch_copies(p, a.ws.copies, a.ws.totals, sm_count, stream);
}

}  // namespace fgw
