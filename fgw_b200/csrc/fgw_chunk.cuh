// Shared parts of the chunk-attention kernels: work items, the workspace and the cursors with which every role of a CTA
// walks its share of the work.
//
// A work item is a run of a request's new tokens for one key head: its rows are (token, query head of the group) pairs,
// so the heads that share keys share every K/V tile. Items cost their KV tiles ("units"). Both kernels lay the units of
// their items end to end and give every program (persistent CTA) a contiguous range, so no CTA waits for a longer one;
// the tensor kernel first deals whole items where that balances as well (chunk_plan_kernel). A piece of an item cut
// between programs leaves a normalised partial result and its LSE in one of its program's two slots, and
// chunk_merge_kernel, which follows, merges the pieces in their order: results do not depend on timing.
#pragma once

#include "fgw_common.cuh"
#include "fgw_kernels.h"
#include "fgw_ragged.cuh"

namespace fgw {

constexpr int kTensorTileRows = 128;
// The limit of the waits with which a CTA leaves no copy in flight. They follow loads that are already issued, so they
// end at once unless a load is lost.
constexpr uint64_t kDrainBudgetNs = 100000000ull;

// The item whose first piece a program holds when that item goes on in later programs; last < 0: none.
struct ChunkCut {
  int token0, count, hk, last;
};

// What one kernel leaves for the merge, in the workspace.
struct ChunkSlots {
  ChunkCut* cuts;    // [programs]
  int2* errors;      // [programs] {fgw_status, wait site} of each CTA
  float* lse;        // [2 * programs, slot rows] base-2
  float* o;          // [2 * programs, slot rows, dim], the tensor kernel's [2 * programs, dim / 4, slot rows, 4]
};

// The tensor kernel's work list, written by the plan kernel.
struct ChunkMeta {
  int items;      // rows of the list x key heads
  int rounds;     // rounds of whole items: snake order, then, when all items are whole, a round dealt by load
  int snake;      // rounds of them in snake order
  int pad;
};
struct ChunkList {
  ChunkMeta* meta;
  int4* rows;              // sorted: {request, first token in the request, units, cost}
  int4* unsorted;          // plan scratch, as are prefix and first
  long long* prefix;       // [rows + 1] first unit of each row's first item
  int32_t* first;          // [batch + 1] first row of each request
  int32_t* prog_item;      // [programs] the round dealt by load, or the first item of the program's cut range
  int32_t* prog_off;       // [programs] units of that item before the range
  long long* prog_u;       // [programs + 1] first unit of the range
  int max_rows;
};

struct ChunkArgs {
  void* out;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* cu;
  const void* q;
  long long tokens, q_stride, out_stride;
  int batch, heads, kv_heads, group, dim, width, page, causal, box_rows, programs;
  int tokens_per_item;
  FastDiv by_page, by_group, by_item_tokens, by_kv_heads;
  int small_rows;  // rows of a decode item; requests of at most so many go to the decode kernel
  int split;       // requests go by their rows; otherwise everything is the launched kernel's
  int short_boxes; // self-test, host only: K's (1) and V's (2) boxes have half the rows that the kernels wait for
  float scale_log2;
  uint64_t budget_ns;
  ChunkSlots slots;
};

__device__ __forceinline__ void chunk_error(const ChunkArgs& a, int site) {
  int* slot = reinterpret_cast<int*>(&a.slots.errors[blockIdx.x]);
  if (atomicCAS(slot, 0, FGW_ERR_DEVICE_TIMEOUT) == 0) slot[1] = site;
}

// The new tokens [first, first + count) of request b among all tokens; offsets out of order or range give none.
struct NewTokens {
  int first, count;
};
__device__ __forceinline__ NewTokens new_tokens(const int32_t* cu, long long tokens, int b) {
  const int top = static_cast<int>(tokens);
  const int first = min(max(cu[b], 0), top);
  return {first, min(max(cu[b + 1], first), top) - first};
}

__device__ __forceinline__ int held_tokens(const int32_t* lens, int b, int width, int page) {
  return min(max(lens[b], 0), width * page);
}

// n / d rounded up, for 0 <= n < 2^31: the sum with d - 1 would pass 31 bits.
template <int d>
__device__ __forceinline__ int ceil_div(int n) {
  return n / d + (n % d != 0);
}

// Rows of the request's list, 0 when it belongs to the other kernel.
__device__ __forceinline__ int item_rows(const ChunkArgs& a, int count, bool decode) {
  if (a.split && (count * a.group <= a.small_rows) != decode) return 0;
  return count > 0 ? a.by_item_tokens.quotient(count - 1) + 1 : 0;
}

// KV tiles of the item that starts at the request's token t0; one without keys still costs one (zeros to write).
template <int kKeys>
__device__ __forceinline__ int item_units(const ChunkArgs& a, int count, int len, int t0) {
  const int last = t0 + min(a.tokens_per_item, count - t0) - 1;
  const int seen = max(a.causal ? len - count + last + 1 : len, 0);
  return max(ceil_div<kKeys>(seen), 1);
}

// One run of KV tiles of one item processed by this CTA: a whole item, or a piece of one cut between programs.
struct ChunkSegment {
  int b, hk;
  int token0;      // first token of the item among all tokens
  int count;       // tokens of the item
  int seen0;       // keys its first token sees, before clamping at 0 (each later token: one more when causal)
  int limit;       // keys its last token sees: nothing from here on is loaded
  int n_begin, n;  // KV tiles of this segment
  int slot;        // a piece's slot, -1 for a whole item
  bool starts;     // the piece that starts a cut item
  long long end_u; // last unit + 1 of the item (cut ranges)
};

// Fills in the segment of `count` units from `first` on of an item.
template <int kKeys>
__device__ __forceinline__ void make_segment(const ChunkArgs& a, ChunkSegment& s, int b, int hk, const NewTokens& nt,
                                             int len, int t0, int units, int first, int count) {
  s.b = b;
  s.hk = hk;
  s.token0 = nt.first + t0;
  s.count = min(a.tokens_per_item, nt.count - t0);
  s.seen0 = a.causal ? len - nt.count + t0 + 1 : len;
  s.limit = max(a.causal ? s.seen0 + s.count - 1 : len, 0);
  const int tiles = ceil_div<kKeys>(s.limit);
  s.n_begin = first;
  s.n = max(0, min(first + count, tiles) - first);
  // a piece that starts inside its item is its program's first, one that starts the item its program's last
  s.starts = first == 0 && count < units;
  s.slot = count == units ? -1 : 2 * static_cast<int>(blockIdx.x) + (first == 0 ? 1 : 0);
}

// Keys that the item's i-th token sees.
__device__ __forceinline__ int seen_keys(const ChunkArgs& a, const ChunkSegment& s, int i) {
  return max(a.causal ? s.seen0 + i : s.seen0, 0);
}

cudaError_t launch_chunk_decode(const fgw_chunk_params& p, ChunkArgs a, int device, cudaStream_t stream);
cudaError_t launch_chunk_tensor(const fgw_chunk_params& p, ChunkArgs a, const ChunkList& list, int device,
                                cudaStream_t stream);

// K and V tensor maps {D, kv heads, pool rows} with boxes of 64 values x a.box_rows tokens, 128-byte swizzle.
CUresult chunk_kv_maps(CUtensorMap* kmap, CUtensorMap* vmap, const fgw_chunk_params& p, const ChunkArgs& a);
// Rows per box: boxes never cross a page or a tile of `keys` tokens.
int chunk_box_rows(int page, int keys);

// Per-width shapes of the two kernels (D up to 64, 128, 192, 256: NB = 1..4 blocks of 64 values).
__host__ __device__ constexpr int chunk_decode_keys(int nb, int row_tiles) { return nb <= 2 && row_tiles <= 2 ? 128 : 64; }
__host__ __device__ constexpr int chunk_tensor_tiles(int nb) { return nb <= 2 ? 2 : 1; }

}  // namespace fgw
