// Shared parts of the chunk-attention kernels: the work list that the plan kernel leaves in the workspace and the cursor
// with which every role of a CTA walks its share of it.
//
// A work item is a run of a request's new tokens for one key head: its rows are (token, query head of the group) pairs,
// so the heads that share keys share every K/V tile. Items cost their KV tiles ("units"). The plan sorts the items by
// cost, deals whole rounds of one item per CTA in snake order while no CTA gets more than its share of all units, and
// cuts the rest into one contiguous range of units per CTA, each CTA's range sized to fill up its share. With fewer
// items than CTAs (single tokens, short batches) that is split-KV with equal splits; with many it is whole items with
// a levelled tail. An item cut between CTAs is merged by the piece that arrives last, in piece order, so results do
// not depend on timing.
#pragma once

#include "fgw_common.cuh"
#include "fgw_kernels.h"
#include "fgw_ragged.cuh"

namespace fgw {

constexpr int kDecodeRows = 16;      // rows of a decode item: one m16 MMA tile
constexpr int kTensorTileRows = 128;

// Totals of one kernel's work list.
struct ChunkMeta {
  int items;      // rows of the list x key heads
  int rounds;     // whole rounds dealt in snake order; items from rounds * programs on are cut
  int pad[2];
};

// One kernel's work list (device memory in the workspace).
struct ChunkList {
  ChunkMeta* meta;
  int4* rows;              // sorted: {request, first token in the request, units, 0}
  int4* unsorted;
  long long* prefix;       // [rows + 1] first unit of each row's first item
  int32_t* first;          // [batch + 1] plan scratch: first row of each request
  int32_t* prog_item;      // [programs] first item of the program's cut range
  int32_t* prog_off;       // [programs] units of that item before the range
  long long* prog_u;       // [programs + 1] first unit of the range
  int32_t* counters;       // [programs] pieces arrived of the item cut at the end of this program's range
  float* slot_lse;         // [2 * programs, slot rows]
  float* slot_o;           // [2 * programs, slot rows, dim]
  int max_rows;
  int tokens_per_item;
  int keys_per_unit;
};

struct ChunkArgs {
  void* out;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* cu;
  const void* q;
  WorkspaceHeader* ws;
  long long tokens, q_stride, out_stride;
  int batch, heads, kv_heads, group, dim, width, page, causal, box_rows, programs;
  float scale_log2;
  uint64_t budget_ns;
  ChunkList list;
};

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

// One run of KV tiles of one item processed by this CTA: a whole item, or a piece of one cut between CTAs.
struct ChunkSegment {
  int b, hk;
  int token0;      // first token of the item among all tokens
  int count;       // tokens of the item
  int seen0;       // keys its first token sees, before clamping at 0 (each later token: one more when causal)
  int limit;       // keys its last token sees: nothing from here on is loaded
  int n_begin, n;  // KV tiles of this segment
  int units;       // of the item
  bool piece;      // the item's other tiles belong to other programs
  long long u0;    // first unit of the item
};

struct ChunkCursor {
  int round, rounds, items;
  int item, off;
  long long u, u_end;
};

__device__ __forceinline__ void cursor_init(const ChunkArgs& a, ChunkCursor& k) {
  k.round = 0;
  k.rounds = a.list.meta->rounds;
  k.items = a.list.meta->items;
  k.item = a.list.prog_item[blockIdx.x];
  k.off = a.list.prog_off[blockIdx.x];
  k.u = a.list.prog_u[blockIdx.x];
  k.u_end = a.list.prog_u[blockIdx.x + 1];
}

__device__ __forceinline__ bool next_segment(const ChunkArgs& a, ChunkCursor& k, ChunkSegment& s) {
  int item, first, count;
  const bool whole = k.round < k.rounds;
  if (whole) {
    item = static_cast<int>(snake_item(k.round));
    ++k.round;
  } else {
    if (k.u >= k.u_end) return false;
    item = k.item;
  }
  const int4 row = a.list.rows[item / a.kv_heads];
  s.units = row.z;
  if (whole) {
    first = 0;
    count = s.units;
    s.u0 = 0;
  } else {
    first = k.off;
    count = static_cast<int>(min(static_cast<long long>(s.units - first), k.u_end - k.u));
    s.u0 = k.u - first;
    k.u += count;
    k.off += count;
    if (k.off >= s.units) {
      ++k.item;
      k.off = 0;
    }
  }
  s.b = row.x;
  s.hk = item % a.kv_heads;
  const NewTokens nt = new_tokens(a.cu, a.tokens, s.b);
  const int len = held_tokens(a.lens, s.b, a.width, a.page);
  s.token0 = nt.first + row.y;
  s.count = min(a.list.tokens_per_item, nt.count - row.y);
  s.seen0 = a.causal ? len - nt.count + row.y + 1 : len;
  s.limit = max(a.causal ? s.seen0 + s.count - 1 : len, 0);
  const int tiles = (s.limit + a.list.keys_per_unit - 1) / a.list.keys_per_unit;
  s.piece = count < s.units;
  s.n_begin = first;
  s.n = max(0, min(first + count, tiles) - first);
  return true;
}

// Keys that the item's i-th token sees.
__device__ __forceinline__ int seen_keys(const ChunkArgs& a, const ChunkSegment& s, int i) {
  return max(a.causal ? s.seen0 + i : s.seen0, 0);
}

// The programs that hold pieces of the cut item of segment `s`: those of [q_first, q_last] that have units at all. The
// piece that starts the item is its program's last and uses slot 2 q + 1; a piece that starts inside the item is its
// program's first and uses slot 2 q. So every program has two slots, and one item whose first piece it holds.
struct ChunkPieces {
  int q_first, q_last, pieces;
  const long long* prog_u;
  __device__ __forceinline__ bool holds(int q) const { return prog_u[q] < prog_u[q + 1]; }
  __device__ __forceinline__ int slot(int q) const { return 2 * q + (q == q_first ? 1 : 0); }
};

__device__ __forceinline__ ChunkPieces chunk_pieces(const ChunkArgs& a, const ChunkSegment& s) {
  ChunkPieces c;
  c.prog_u = a.list.prog_u;
  c.q_first = c.q_last = blockIdx.x;
  while (c.prog_u[c.q_first] > s.u0) --c.q_first;
  while (c.prog_u[c.q_last + 1] < s.u0 + s.units) ++c.q_last;
  c.pieces = 0;
  for (int q = c.q_first; q <= c.q_last; ++q) c.pieces += c.holds(q) ? 1 : 0;
  return c;
}

cudaError_t launch_chunk_decode(const fgw_chunk_params& p, ChunkArgs a, int device, cudaStream_t stream);
cudaError_t launch_chunk_tensor(const fgw_chunk_params& p, ChunkArgs a, int device, cudaStream_t stream);

// K/V tensor map {D, kv heads, pool rows} with boxes of 64 values x box_rows tokens, 128-byte swizzle.
CUresult chunk_kv_map(CUtensorMap* map, const fgw_chunk_params& p, const void* base, int box_rows);
// Rows per box: boxes never cross a page or a tile of `keys` tokens.
int chunk_box_rows(int page, int keys);

// Per-width shapes of the two kernels (D up to 64, 128, 192, 256: NB = 1..4 blocks of 64 values).
__host__ __device__ constexpr int chunk_decode_keys(int nb) { return nb <= 2 ? 128 : 64; }
__host__ __device__ constexpr int chunk_tensor_tiles(int nb) { return nb <= 2 ? 2 : 1; }

}  // namespace fgw
