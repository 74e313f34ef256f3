// Chunk attention, tensor kernel (tcgen05): the requests with more rows than a decode item.
//
// Rows of a 128-row tile are (token, query head of the group) pairs of one key head, token by token: 128 / G tokens of G
// heads. One TMA box {64 values, G heads, 128 / G tokens} loads such a tile from the queries as they lie in memory, and
// each K/V tile serves all heads of the group.
//
// Up to D = 128 a work item is two tiles (A, B) that share every K/V tile; above, O takes 256 columns of TMEM and an item
// is one tile. Each tile has an MMA warp, so one tile's waits do not hold up the other's MMAs. S and O live in TMEM, and so
// does P, the A operand of PV. In (64, 128] S and O of two tiles fill TMEM and P overwrites the S it came from: per KV tile
// PV(j) follows P's first and second half, then QK(j + 1). Elsewhere P has columns of its own, QK(j + 1) is issued as soon
// as the softmax has read S(j), and two softmax warpgroups share a tile.
//
// Bound by the softmax's chain of waits, TMEM loads, maximum, 2^x and TMEM stores, far more than by any unit: a tile pair
// costs 2048 cycles of 2^x whatever D is and 1024 (D = 64) or 2048 (D = 128) of MMA, and a step takes 3600 to 4000. At
// D = 64 a step without its MMAs takes as long, without its 2^x 0.8 of the time. Measured: 4096 tokens over 28K cached, 32
// heads on 8 key heads of 128, 1790 to 1914 us by the card's clock = 1.08 to 1.15 PFLOP/s; 16 requests of chunks and single tokens, 24 heads on 8 of 64, 154 us;
// 8 prompts of up to 1024, 16 heads of 128, 53.5 us. At D = 64, steps kept and what they replaced: P apart, two warpgroups
// per tile, an MMA warp per tile, turns together 165 -> 159 us. Tried and slower or without effect: two warpgroups per
// tile at D = 128 (1902 to 2478 us, by the spills), a third score buffer (178 to 192 us), QK of the next item issued beside
// the last PV of the one before, a warp that hands out the segments, part of the 2^x on the FMA pipe (184 to 193 us).
#include <algorithm>
#include <climits>

#include "fgw_chunk.cuh"

namespace fgw {

// A CTA's whole items, then its range of units of the cut ones.
struct TensorCursor {
  int round, rounds, snake, items;
  int item, off;
  long long u, u_end;
};

// A softmax warp's place in shared memory where its registers are short.
struct SoftmaxWalk {
  TensorCursor cur;
  ChunkSegment sg;
  int more, pad;
};

template <int NB>
struct TensorShape {
  static constexpr int kTiles = chunk_tensor_tiles(NB);
  static constexpr int kBN = 128;
  static constexpr int kTileBytes = 128 * 128;         // one 64-value block of a 128-row operand
  static constexpr int kQBytes = NB * kTileBytes;      // one query tile
  static constexpr int kKVBytes = NB * kBN * 128;      // one K (or V) stage
  static constexpr int kStages = NB == 1 ? 4 : (NB == 2 ? 2 : 1);
  // The 2^x of tile A's and B's steps in turns, for so many steps of an item: both tiles' scores come together at an
  // item's start, and without turns they then share the SFUs and idle them together. At D = 64 the tiles fall back into
  // step by themselves (mixed step 154 us with turns throughout, 162 to 167 with one to six, 176 without). At D = 128 two
  // steps set them apart (prompts 57.6 -> 53.4 us, 8 x 1000 tokens over 3000 cached 528 -> 473 us, over 10000 1387 ->
  // 1328 us), more cost again (1338 us; 4096 tokens over 28K 1808 against 1790 us, 1757 without).
  static constexpr int kTurnSteps = NB == 1 ? INT_MAX : (NB == 2 ? 2 : 0);
  static constexpr bool kTurns = kTurnSteps > 0;
  // Where P is apart the softmax alone paces a tile, and two warpgroups share it: each thread half a row.
  static constexpr int kHalves = NB == 2 ? 1 : 2;
  static constexpr int kSoftmaxWarps = 4 * kHalves;  // of one query tile
  static constexpr int kThreads = 128 + 128 * kTiles * kHalves;
  // Registers per thread after the warpgroup split: 4 x 32 x 88 + 8 x 32 x 208 = 384 x 168 with two softmax warpgroups
  // (NB = 2), 4 x 32 x 64 + 16 x 32 x 104 = 640 x 96 with four (NB = 1); one tile needs no split.
  static constexpr int kRegsControl = NB == 1 ? 64 : 88;
  static constexpr int kRegsSoftmax = NB == 1 ? 104 : 208;
  // TMEM columns. Where there is room, P has columns of its own: then QK of a tile's next scores waits only until the
  // softmax has read the last ones. At D in (64, 128] S and O of two tiles fill TMEM, and P overwrites S.
  static constexpr bool kApart = NB != 2;
  __device__ __forceinline__ static uint32_t s_col(int t) { return static_cast<uint32_t>(t) * 128u; }
  __device__ __forceinline__ static uint32_t o_col(int t) { return 256u + static_cast<uint32_t>(t) * (NB == 1 ? 64u : 128u); }
  __device__ __forceinline__ static uint32_t p_col(int t) {
    return NB == 1 ? 384u + static_cast<uint32_t>(t) * 64u : (NB == 2 ? s_col(t) : 128u);
  }
  static constexpr int kTmemCols = 512;
  static constexpr int kK = kTiles * kQBytes;
  static constexpr int kV = kK + kStages * kKVBytes;
  static constexpr int kBar = kV + kStages * kKVBytes;
  // q_full, q_empty, {k,v}_{full,empty}[S], s_full, p_half, p_full, pv_done, o_empty, s_read [2], mma_done, v_raw
  static constexpr int kNumBars = 2 + 4 * kStages + 12 + 2;
  static constexpr int kTmemSlot = kBar + kNumBars * 8;
  static constexpr int kWalks = kTmemSlot + 16;  // segment and cursor of each softmax warp (kHalves == 2)
  static constexpr int kMax = kWalks + (kHalves - 1) * kSoftmaxWarps * kTiles * static_cast<int>(sizeof(SoftmaxWalk));
  static constexpr int kBytes = kMax + (kHalves - 1) * kTiles * 2048 + 1024;  // [2 turns][tiles][2][128] floats
  static_assert(kBytes <= 232448, "shared memory of one CTA");
};

__device__ __forceinline__ void cursor_init(const ChunkList& list, TensorCursor& k) {
  k.round = 0;
  k.rounds = list.meta->rounds;
  k.snake = list.meta->snake;
  k.items = list.meta->items;
  k.item = list.prog_item[blockIdx.x];
  k.off = list.prog_off[blockIdx.x];
  k.u = list.prog_u[blockIdx.x];
  k.u_end = list.prog_u[blockIdx.x + 1];
}

__device__ __forceinline__ bool next_segment(const ChunkArgs& a, const ChunkList& list, TensorCursor& k,
                                             ChunkSegment& s) {
  int item = k.items;
  if (k.round < k.rounds) {
    item = k.round < k.snake ? static_cast<int>(snake_item(k.round)) : k.item;
    ++k.round;
  }
  const bool whole = item < k.items;  // the last round may be short
  if (!whole) {
    if (k.u >= k.u_end) return false;
    item = k.item;
  }
  const int list_row = a.by_kv_heads.quotient(item);
  const int4 row = list.rows[list_row];
  const int units = row.z, first = whole ? 0 : k.off;
  const int count = whole ? units : static_cast<int>(min(static_cast<long long>(units - first), k.u_end - k.u));
  make_segment<128>(a, s, row.x, item - list_row * a.kv_heads, new_tokens(a.cu, a.tokens, row.x),
                    held_tokens(a.lens, row.x, a.width, a.page), row.y, units, first, count);
  if (!whole) {
    s.end_u = k.u - first + units;
    k.u += count;
    k.off += count;
    if (k.off >= units) {
      ++k.item;
      k.off = 0;
    }
  }
  return true;
}

// max(a, b, c) in one instruction (sm_100 three-input max; NaN-free inputs here)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^(s * scale - m) for 2 N scores, packed to 16-bit pairs; the row sum adds the rounded values PV multiplies (with the
// lazily rescaled maximum a row's largest P may exceed 1 and round, and that rounding must cancel).
template <typename Tr, int N, int kSums>
__device__ __forceinline__ void exp2_pack(const uint32_t* sr, float2 scale2, float2 negm2, float2 (&acc)[kSums],
                                          uint32_t (&packed)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float2 x = __ffma2_rn(make_float2(__uint_as_float(sr[2 * i]), __uint_as_float(sr[2 * i + 1])), scale2, negm2);
    packed[i] = Tr::pack2(fast_exp2(x.x), fast_exp2(x.y));
    acc[i % kSums] = Tr::add2(acc[i % kSums], packed[i]);
  }
}

__device__ __forceinline__ void st_shared(uint32_t at, float x) {
  asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(x) : "memory");
}
__device__ __forceinline__ float ld_shared(uint32_t at) {
  float x;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(at) : "memory");
  return x;
}

// Tiles of the segment that query tile t works on, and its first token within the item.
__device__ __forceinline__ int tile_steps(const ChunkArgs& a, const ChunkSegment& s, int t, int tokens) {
  const int left = s.count - t * tokens;
  if (left <= 0) return 0;
  const int seen = seen_keys(a, s, t * tokens + min(left, tokens) - 1);
  return max(0, min(s.n_begin + s.n, ceil_div<128>(seen)) - s.n_begin);
}

template <typename T, int NB>
__global__ void __launch_bounds__(TensorShape<NB>::kThreads, 1)
    chunk_tensor_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                        const __grid_constant__ CUtensorMap vmap, const __grid_constant__ ChunkArgs a,
                        const __grid_constant__ ChunkList list) {
  using S = TensorShape<NB>;
  using Tr = ElemTraits<T>;
  constexpr int BN = S::kBN, NS = S::kStages, kTiles = S::kTiles;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_smem = smem;
  uint8_t* k_smem = smem + S::kK;
  uint8_t* v_smem = smem + S::kV;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBar);
  uint64_t* q_full = bars + 0;
  uint64_t* q_empty = bars + 1;
  uint64_t* k_full = bars + 2;
  uint64_t* k_empty = k_full + NS;
  uint64_t* v_full = k_empty + NS;
  uint64_t* v_empty = v_full + NS;
  uint64_t* s_full = v_empty + NS;  // [2]
  uint64_t* p_half = s_full + 2;    // [2]: the first 64 keys of P_t are in TMEM
  uint64_t* p_full = p_half + 2;    // [2]
  uint64_t* pv_done = p_full + 2;   // [2]
  uint64_t* o_empty = pv_done + 2;  // [2]
  uint64_t* s_read = o_empty + 2;   // [2]: S_t is in the softmax's registers (kApart)
  uint64_t* mma_done = s_read + 2;
  uint64_t* v_raw = mma_done + 1;   // a ragged V tile has landed
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + S::kTmemSlot);

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, kTiles);  // one arrival per MMA warp
    for (int i = 0; i < NS; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], kTiles);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], kTiles);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_half[t], S::kSoftmaxWarps);  // one arrival per softmax warp
      mbar_init(&p_full[t], S::kSoftmaxWarps);
      mbar_init(&pv_done[t], 1);
      mbar_init(&o_empty[t], S::kSoftmaxWarps);
      mbar_init(&s_read[t], S::kSoftmaxWarps);
    }
    mbar_init(mma_done, kTiles);
    mbar_init(v_raw, 1);
    fence_barrier_init();
    a.slots.errors[blockIdx.x] = make_int2(0, 0);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, S::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  const int D = a.dim;
  const int tile_tokens = kTensorTileRows / a.group;
  grid_dependency_wait();  // the plan's lists from here on
  grid_dependents_launch();

  if (kTiles == 2 && warp < 4) setmaxnreg_dec<S::kRegsControl>();
  if (warp == 0 || warp == 3) {
    // ------------------------------------------------------------------------- TMA producers
    // Warp 0 loads Q and K, warp 3 V. Lane l issues the l-th box of a tile: boxes x blocks of 64 values, at most 32.
    const bool loads_k = warp == 0, loads_v = !loads_k;
    if (lane == 0) {
      if (loads_k) tma_prefetch_desc(&qmap);
      if (loads_k) tma_prefetch_desc(&kmap);
      if (loads_v) tma_prefetch_desc(&vmap);
    }
    bool ok = true;
    uint32_t kc = 0, qc = 0, raw = 0;
    uint32_t given_up = 0, given_up_q = 0;  // kc and qc when a wait gave up: nothing is loaded from there on
    const int boxes = BN / a.box_rows;
    const int box = lane % boxes, blk = lane / boxes;
    const uint32_t box_bytes = a.box_rows * 128;
    const uint32_t q_bytes = static_cast<uint32_t>(tile_tokens) * a.group * 128;
    auto wait_or_fail = [&](uint64_t* bar, uint32_t parity, int site) {
      if (ok && !__all_sync(0xffffffffu, mbar_wait(bar, parity, a.budget_ns))) {
        ok = false;
        given_up = kc;
        given_up_q = qc;
        if (lane == 0) chunk_error(a, site);
      }
      return ok;
    };
    TensorCursor cur;
    cursor_init(list, cur);
    ChunkSegment sg;
    while (__shfl_sync(0xffffffffu, static_cast<int>(next_segment(a, list, cur, sg)), 0)) {
      const int n = __shfl_sync(0xffffffffu, sg.n, 0);
      if (n <= 0) continue;
      if (loads_k && wait_or_fail(q_empty, (qc & 1) ^ 1, 80) && lane == 0) {
        const int tiles_q = kTiles == 2 && sg.count > tile_tokens ? 2 : 1;
        mbar_arrive_expect_tx(q_full, tiles_q * NB * q_bytes);
        for (int t = 0; t < tiles_q; ++t) {
          for (int b = 0; b < NB; ++b) {
            tma_load_4d(q_smem + t * S::kQBytes + b * S::kTileBytes, &qmap, q_full, b * 64, 0, sg.hk,
                        sg.token0 + t * tile_tokens);
          }
        }
      }
      ++qc;
      const int32_t* table = a.table + static_cast<long long>(sg.b) * a.width;
      for (int j = 0; j < n; ++j) {
        const int tok = (sg.n_begin + j) * BN + box * a.box_rows;
        const bool load = blk < NB && tok < sg.limit;
        const int page = a.by_page.quotient(tok);
        const int row = load ? table[page] * a.page + tok - page * a.page : 0;
        const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, load)) * box_bytes;
        const int st = kc % NS;
        const uint32_t parity = ((kc / NS) & 1) ^ 1;
        uint8_t* dst = k_smem + st * S::kKVBytes + blk * BN * 128 + box * box_bytes;
        if (loads_k && wait_or_fail(&k_empty[st], parity, 81)) {
          if (lane == 0) mbar_arrive_expect_tx(&k_full[st], bytes);
          __syncwarp();
          if (load) tma_load_3d(dst, &kmap, &k_full[st], blk * 64, sg.hk, row);
        }
        if (loads_v && wait_or_fail(&v_empty[st], parity, 82)) {
          // Rows past the last visible key, whatever the stage or the page holds there, must reach PV as zeros: the tile
          // that holds the end lands on a barrier of its own and becomes visible when they are zeroed.
          const int past = BN - (sg.limit - (sg.n_begin + j) * BN);
          uint64_t* landed = past > 0 ? v_raw : &v_full[st];
          if (lane == 0) mbar_arrive_expect_tx(landed, bytes);
          __syncwarp();
          if (load) tma_load_3d(dst + (S::kV - S::kK), &vmap, landed, blk * 64, sg.hk, row);
          if (past > 0 && wait_or_fail(v_raw, raw++ & 1, 92)) {
            uint8_t* end = v_smem + st * S::kKVBytes + (BN - past) * 128;  // whole 128-byte rows: swizzled within
            for (int i = lane; i < past * 8; i += 32) {
#pragma unroll
              for (int b = 0; b < NB; ++b) *reinterpret_cast<uint4*>(end + b * BN * 128 + i * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&v_full[st]);
          }
        }
        ++kc;
      }
    }
    // Leave no copy in flight, whichever role gave up: the last load of every stage lands before the CTA may end.
    const uint32_t loaded = ok ? kc : given_up, loaded_q = ok ? qc : given_up_q;
    uint64_t* full = loads_k ? k_full : v_full;
    for (uint32_t i = loaded > NS ? loaded - NS : 0; i < loaded; ++i) {
      mbar_wait(&full[i % NS], (i / NS) & 1, kDrainBudgetNs);
    }
    if (loads_k && loaded_q > 0) mbar_wait(q_full, (loaded_q - 1) & 1, kDrainBudgetNs);
    // a ragged V tile lands on a barrier of its own, also the one whose wait gave up
    if (loads_v && raw > 0) mbar_wait(v_raw, (raw - 1) & 1, kDrainBudgetNs);
  } else if (warp <= kTiles) {
    // ------------------------------------------------------------------------- MMA issuer
    // One warp per query tile, so that one tile's waits do not hold up the other's MMAs; a K or V stage, and Q, are free
    // when both have gone through them. The whole warp runs this role converged, its loop state warp-uniform; every tcgen05 issue is predicated on one
    // elected lane.
    const uint32_t leader = elect_one_sync();
    const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem, 0);
    bool ok = true;
    const int t = warp - 1;
    uint32_t kc = 0, vc = 0, qc = 0;  // K tiles, V tiles and items so far
    uint32_t pc = 0, oc = 0;          // steps and items of this query tile
    const uint32_t idesc_qk = umma_idesc_f16(Tr::kUmmaFormat, 128, BN, 0, 0);
    const uint32_t idesc_pv = umma_idesc_f16(Tr::kUmmaFormat, 128, D, 0, 1);
    uint32_t q_lo = umma_desc_lo(smem_u32(q_smem), 16);
    uint32_t k_lo = umma_desc_lo(smem_u32(k_smem), 16);
    uint32_t v_lo = umma_desc_lo(smem_u32(v_smem), BN * 128);
    constexpr uint32_t kHi = umma_desc_hi(1024, 2);
    const int ksteps = D / 16;
    auto wait_or_fail = [&](uint64_t* bar, uint32_t parity, int site) {
      if (ok && !__all_sync(0xffffffffu, mbar_wait(bar, parity, a.budget_ns))) {
        ok = false;
        if (lane == 0) chunk_error(a, site);
      }
      return ok;
    };
    // S_t = Q_t K^T, K from stage st (already waited for)
    auto qk = [&](int st) {
      const uint32_t a_lo = q_lo + static_cast<uint32_t>((t * S::kQBytes) >> 4);
      const uint32_t b_lo = k_lo + static_cast<uint32_t>((st * S::kKVBytes) >> 4);
#pragma unroll
      for (int kk = 0; kk < 4 * NB; ++kk) {
        if (kk < ksteps) {
          umma_f16_ss_e(leader, tmem_u + S::s_col(t), a_lo + (((kk >> 2) * S::kTileBytes + (kk & 3) * 32) >> 4), kHi,
                        b_lo + (((kk >> 2) * BN * 128 + (kk & 3) * 32) >> 4), kHi, idesc_qk, kk > 0 ? 1u : 0u);
        }
      }
      umma_commit_e(leader, &s_full[t]);
    };
    // O_t += P_t V over 64 keys from step k0 (16 keys each), V from stage st; operands advance through opaque registers
    // so that the issuer fits its register budget
    auto pv = [&](int st, bool first, int k0) {
      uint32_t b_lo = v_lo + static_cast<uint32_t>((st * S::kKVBytes) >> 4) + k0 * ((16 * 128) >> 4);
      uint32_t p_col = tmem_u + S::p_col(t) + k0 * 8;
      const uint32_t o_tmem = tmem_u + S::o_col(t);
#pragma unroll
      for (int kk = k0; kk < k0 + BN / 32; ++kk) {
        umma_f16_ts_e(leader, o_tmem, p_col, b_lo, kHi, idesc_pv, (!first || kk > 0) ? 1u : 0u);
        p_col += 8;
        b_lo += (16 * 128) >> 4;
        asm volatile("" : "+r"(p_col), "+r"(b_lo));
      }
    };
    TensorCursor cur;
    cursor_init(list, cur);
    ChunkSegment sg;
    while (__shfl_sync(0xffffffffu, static_cast<int>(next_segment(a, list, cur, sg)), 0)) {
      const int n = __shfl_sync(0xffffffffu, sg.n, 0);
      const int nt = __shfl_sync(0xffffffffu, tile_steps(a, sg, t, tile_tokens), 0);
      if (n <= 0) continue;
      auto seen_k = [&]() { return wait_or_fail(&k_full[kc % NS], (kc / NS) & 1, 86); };
      auto free_k = [&]() {
        if (ok) umma_commit_e(leader, &k_empty[kc % NS]);
        ++kc;
      };
      wait_or_fail(q_full, qc & 1, 83);
      ++qc;
      if (seen_k() && nt > 0) {
        tc_fence_after_sync();
        qk(kc % NS);
      }
      free_k();
      if (n == 1 && ok) umma_commit_e(leader, q_empty);
      for (int j = 0; j < n; ++j) {
        // opaque, so the descriptor sums are formed where they are used
        asm volatile("" : "+r"(q_lo), "+r"(k_lo), "+r"(v_lo));
        const bool more = j + 1 < n, qk_next = j + 1 < nt;
        const int vst = vc % NS;
        if (S::kApart && more) {  // the next scores as soon as the softmax has read the last ones
          seen_k();
          if (qk_next && wait_or_fail(&s_read[t], pc & 1, 88)) {
            tc_fence_after_sync();
            qk(kc % NS);
          }
          free_k();
          if (j + 2 == n && ok) umma_commit_e(leader, q_empty);  // every QK of this item is now issued
        }
        // the buffers first, P, which usually comes last, last
        wait_or_fail(&v_full[vst], (vc / NS) & 1, 85);
        if (!S::kApart && more) seen_k();
        if (j < nt) {
          if (j == 0) wait_or_fail(&o_empty[t], (oc & 1) ^ 1, 87);
          if (!S::kApart && wait_or_fail(&p_half[t], pc & 1, 84)) {
            tc_fence_after_sync();
            pv(vst, j == 0, 0);
          }
          if (wait_or_fail(&p_full[t], pc & 1, 89)) {
            tc_fence_after_sync();
            if (S::kApart) pv(vst, j == 0, 0);
            pv(vst, false, BN / 32);
            if (S::kApart || j + 1 == nt) umma_commit_e(leader, &pv_done[t]);
            if (!S::kApart && qk_next) qk(kc % NS);
          }
          ++pc;
        }
        if (ok) umma_commit_e(leader, &v_empty[vst]);
        ++vc;
        if (!S::kApart && more) {
          free_k();
          if (j + 2 == n && ok) umma_commit_e(leader, q_empty);
        }
      }
      if (nt > 0) ++oc;
    }
    // Every MMA has ended before TMEM is released, also those issued before a wait gave up.
    umma_commit_e(leader, mma_done);
    __all_sync(0xffffffffu, mbar_wait(mma_done, 0, kDrainBudgetNs));
  } else if (warp >= 4) {
    // ------------------------------------------------------------------------- softmax / epilogue
    // One or two warpgroups per query tile; a warp reaches the TMEM lanes of its quarter (warp % 4). With two, each has
    // half of every row: kCols keys of a KV tile and, for the rescale and the epilogue, half of O's columns. The two
    // threads of a row sit in two warps that exchange the row's maximum through shared memory and a barrier of 64.
    if (kTiles == 2) setmaxnreg_inc<S::kRegsSoftmax>();
    constexpr int kHalves = S::kHalves, kCols = BN / kHalves;
    const int t = (warp - 4) / S::kSoftmaxWarps, h = kHalves == 2 ? (warp / 4 - 1) % 2 : 0;
    const int row = (warp % 4) * 32 + lane;
    const uint32_t lane_base = static_cast<uint32_t>((warp % 4) * 32) << 16;
    const uint32_t s_addr = tmem + lane_base + S::s_col(t) + h * kCols;
    const uint32_t p_addr = tmem + lane_base + S::p_col(t) + h * (kCols / 2);
    const uint32_t o_addr = tmem + lane_base + S::o_col(t);
    // maxima by turn: a fast warp may be a step ahead of the one it exchanges with
    const uint32_t my_max = smem_u32(smem + S::kMax) + ((t * 2 + h) * 128 + row) * 4;
    const uint32_t other_max = h == 0 ? my_max + 512 : my_max - 512;
    const uint32_t pair_barrier = 1 + t * 4 + warp % 4;
    constexpr uint32_t kTurnBarrier = 9, kTurnThreads = 256 * kHalves;
    auto o_half = [&](int half) {  // this half's 16-column blocks of O
      return half == 0 ? 0 : (half < kHalves ? (D / 16 + 1) / 2 : D / 16);
    };
    bool ok = true;
    uint32_t sc = 0, pd = 0;
    if (warp == 4 && lane == 0) a.slots.cuts[blockIdx.x] = {0, 0, 0, -1};
    auto wait_warp = [&](uint64_t* bar, uint32_t parity, int site) {
      if (ok) {
        ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, a.budget_ns));
        if (!ok && lane == 0) chunk_error(a, site);
      }
      return ok;
    };
    SoftmaxWalk own;
    SoftmaxWalk& walk = kHalves == 2 ? reinterpret_cast<SoftmaxWalk*>(smem + S::kWalks)[warp - 4] : own;
    const ChunkSegment& sg = walk.sg;
    auto advance = [&]() {
      if constexpr (kHalves == 1) {
        return next_segment(a, list, walk.cur, walk.sg);
      } else {
        __syncwarp();  // every lane is done with the segment before
        if (lane == 0) walk.more = next_segment(a, list, walk.cur, walk.sg) ? 1 : 0;
        __syncwarp();
        return *const_cast<volatile int*>(&walk.more) != 0;
      }
    };
    if (S::kTurns && t == 1) named_barrier_arrive(kTurnBarrier, kTurnThreads);  // tile A begins
    if (kHalves == 1 || lane == 0) cursor_init(list, walk.cur);
    while (advance()) {
      int vis;  // keys that this thread's row sees
      {
        const int i_tok = t * tile_tokens + a.by_group.quotient(row);
        // rows of no token compute on whatever Q's tile holds (rows do not mix) and are never stored
        vis = i_tok < (t + 1) * tile_tokens && i_tok < sg.count ? seen_keys(a, sg, i_tok) : sg.limit;
      }
      const int n_t = tile_steps(a, sg, t, tile_tokens);
      const int n_other = kTiles == 2 ? tile_steps(a, sg, 1 - t, tile_tokens) : 0;
      const int n_both = min(n_t, n_other);
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < n_t; ++j) {
        const int tok0 = (sg.n_begin + j) * BN;
        wait_warp(&s_full[t], sc & 1, 90 + t);
        ++sc;
        const int valid_cols = vis - tok0 - h * kCols;
        uint32_t sr[kCols];
        if (ok) {
          tc_fence_after_sync();
#pragma unroll
          for (int cb = 0; cb < kCols / 64; ++cb) {
            tmem_ld64(s_addr + cb * 64, *reinterpret_cast<uint32_t(*)[64]>(&sr[cb * 64]));
          }
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < kCols; ++i) sr[i] = 0xff800000u;
        }
        if (S::kApart) {
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_read[t]);
        }
        if (valid_cols < kCols) {  // ragged or diagonal tile
#pragma unroll
          for (int col = 0; col < kCols; ++col) {
            if (col >= valid_cols) sr[col] = 0xff800000u;  // -inf
          }
        }
        auto sval = [&](int col) -> float { return __uint_as_float(sr[col]); };
        float mq0 = -INFINITY, mq1 = -INFINITY, mq2 = -INFINITY, mq3 = -INFINITY;
#pragma unroll
        for (int col = 0; col < kCols; col += 8) {
          mq0 = max3(mq0, sval(col), sval(col + 1));
          mq1 = max3(mq1, sval(col + 2), sval(col + 3));
          mq2 = max3(mq2, sval(col + 4), sval(col + 5));
          mq3 = max3(mq3, sval(col + 6), sval(col + 7));
        }
        float mx = max3(mq0, mq1, fmaxf(mq2, mq3));
        if constexpr (kHalves == 2) {
          const uint32_t turn = (sc & 1) * kTiles * 1024;
          st_shared(my_max + turn, mx);
          named_barrier_sync(pair_barrier, 64);
          mx = fmaxf(mx, ld_shared(other_max + turn));
        }
        mx *= a.scale_log2;  // scale > 0; -inf stays -inf
        // with P apart, PV of the step before has to have read it, and O is stable then too
        if (S::kApart && j > 0) {
          wait_warp(&pv_done[t], pd & 1, 93);
          ++pd;
          if (ok) tc_fence_after_sync();
        }
        // The maximum moves only when it grows by more than 2^8 (P then stays below 2^8, far inside both types' range),
        // so O is rarely rescaled. Each row decides for itself: what other rows of the warp hold leaves its bits alone.
        const bool grow = j > 0 && mx > m + 8.0f;
        const float m_new = j == 0 || grow ? mx : m;
        float alpha = 1.f;
        if (__any_sync(0xffffffffu, grow)) {
          if (grow) alpha = m == -INFINITY ? 0.f : fast_exp2(m - m_new);
          if (ok) {
            // O_t is stable: the commit that published S_t(j) also covers PV_t(j - 1), or its own was waited for
            for (int cb = o_half(h); cb < o_half(h + 1); ++cb) {
              uint32_t r[16];
              tmem_ld16(o_addr + cb * 16, r);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
              tmem_st16(o_addr + cb * 16, r);
            }
          }
        }
        const bool in_turn = S::kTurns && j < min(n_both, S::kTurnSteps);
        if (in_turn) named_barrier_sync(kTurnBarrier + t, kTurnThreads);
        const float neg_m = (m_new == -INFINITY) ? 0.f : -m_new;
        float rowsum = 0.f;
        if (ok) {
          const float2 scale2 = make_float2(a.scale_log2, a.scale_log2);
          const float2 negm2 = make_float2(neg_m, neg_m);
          float2 acc[4 / kHalves] = {};
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            uint32_t packed[kCols / 4];
            exp2_pack<Tr>(&sr[part * (kCols / 2)], scale2, negm2, acc, packed);
            if constexpr (kHalves == 2) {
              tmem_st16(p_addr + part * 16, packed);
            } else {
              tmem_st32(p_addr + part * 32, packed);
            }
            if (!S::kApart && part == 0) {
              tmem_wait_st();
              tc_fence_before_sync();
              __syncwarp();
              if (lane == 0) mbar_arrive(&p_half[t]);
            }
            if (in_turn && part == 0) named_barrier_arrive(kTurnBarrier + 1 - t, kTurnThreads);
          }
          tmem_wait_st();
#pragma unroll
          for (const float2& sum : acc) rowsum += sum.x + sum.y;
        } else if (in_turn) {
          named_barrier_arrive(kTurnBarrier + 1 - t, kTurnThreads);
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          if (!S::kApart && !ok) mbar_arrive(&p_half[t]);
          mbar_arrive(&p_full[t]);
        }
        l = l * alpha + rowsum;
        m = m_new;
      }
      // epilogue
      float inv = 0.f;
      if (n_t > 0) {
        wait_warp(&pv_done[t], pd & 1, 93);
        ++pd;
        if constexpr (kHalves == 2) {  // the row's sum over both halves
          const uint32_t turn = (sc & 1) * kTiles * 1024;
          const uint32_t next = kTiles * 1024 - turn;
          st_shared(my_max + next, l);
          named_barrier_sync(pair_barrier, 64);
          l = h == 0 ? l + ld_shared(other_max + next) : ld_shared(other_max + next) + l;
          named_barrier_sync(pair_barrier, 64);  // read by both before the next exchange
        }
        inv = 1.f / l;
        if (ok) tc_fence_after_sync();
      }
      const int row_token = a.by_group.quotient(row), row_head = row - row_token * a.group;
      const int i_tok = t * tile_tokens + row_token;  // token within the item
      const bool row_valid = row_token < tile_tokens && i_tok < sg.count;
      T* out_row = static_cast<T*>(a.out) + (row_valid ? (sg.token0 + i_tok) * a.out_stride : 0) +
                   static_cast<long long>(sg.hk * a.group + row_head) * D;
      auto load_o = [&](int cb, float (&o)[16]) {
        if (n_t > 0 && ok) {
          uint32_t r[16];
          tmem_ld16(o_addr + cb * 16, r);
          tmem_wait_ld();
          // no key seen: exact zeros; a NaN among the scores stays one
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = l == 0.f ? 0.f : __uint_as_float(r[i]) * inv;
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = 0.f;
        }
      };
      if (sg.slot < 0) {
        for (int cb = o_half(h); cb < o_half(h + 1); ++cb) {
          float o[16];
          load_o(cb, o);  // warp-collective: every lane, valid row or not
          if (row_valid) {
            uint4* dst = reinterpret_cast<uint4*>(out_row + cb * 16);
            dst[0] = make_uint4(Tr::pack2(o[0], o[1]), Tr::pack2(o[2], o[3]), Tr::pack2(o[4], o[5]), Tr::pack2(o[6], o[7]));
            dst[1] = make_uint4(Tr::pack2(o[8], o[9]), Tr::pack2(o[10], o[11]), Tr::pack2(o[12], o[13]),
                                Tr::pack2(o[14], o[15]));
          }
        }
        if (n_t > 0) {
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&o_empty[t]);
        }
        continue;
      }
      // A piece of an item cut between CTAs: FP32 O and base-2 LSE go to its slot, O in groups of four columns ([D / 4]
      // [rows][4]), so a warp's rows write 512 contiguous bytes per group.
      constexpr int kSlotRows = kTensorTileRows * kTiles;
      const int r = kTensorTileRows * t + row;
      float4* slot_o = reinterpret_cast<float4*>(a.slots.o) + static_cast<long long>(sg.slot) * (D / 4) * kSlotRows + r;
      for (int cb = o_half(h); cb < o_half(h + 1); ++cb) {
        float o[16];
        load_o(cb, o);
        if (row_valid) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            slot_o[(cb * 4 + i) * kSlotRows] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          }
        }
      }
      if (row_valid && h == 0) {
        a.slots.lse[static_cast<long long>(sg.slot) * kSlotRows + r] = n_t == 0 || l == 0.f ? kEmptyLse : m + fast_log2(l);
      }
      if (n_t > 0) {
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_empty[t]);
      }
      if (sg.starts && warp == 4 && lane == 0) {
        int last = blockIdx.x;
        while (list.prog_u[last + 1] < sg.end_u) ++last;
        a.slots.cuts[blockIdx.x] = {sg.token0, sg.count, sg.hk, last};
      }
    }
    if (S::kTurns && t == 0) named_barrier_sync(kTurnBarrier, kTurnThreads);  // no arrival is left over
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, S::kTmemCols);
  }
}

template <typename T, int NB>
static cudaError_t launch_tensor_t(const fgw_chunk_params& p, ChunkArgs a, const ChunkList& list, int device,
                                   cudaStream_t stream) {
  using S = TensorShape<NB>;
  auto kernel = chunk_tensor_kernel<T, NB>;
  int regs = 0;
  cudaError_t err = prepare_kernel(reinterpret_cast<const void*>(kernel), S::kBytes, device, &regs);
  if (err != cudaSuccess) return err;
  // setmaxnreg.inc draws on the registers the block was launched with: refuse a build that would not cover the split
  const int allocated = ((regs + 7) / 8) * 8 * S::kThreads;
  if (S::kTiles == 2 && allocated < 4 * 32 * S::kRegsControl + 8 * S::kHalves * 32 * S::kRegsSoftmax) return cudaErrorNotSupported;
  a.box_rows = chunk_box_rows(p.page_size, S::kBN);
  CUtensorMap qmap, kmap, vmap;
  // a tile's rows: all heads of the group, token by token
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(p.head_dim), static_cast<cuuint64_t>(a.group),
                              static_cast<cuuint64_t>(p.kv_heads), static_cast<cuuint64_t>(p.tokens)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(p.head_dim) * 2,
                                 static_cast<cuuint64_t>(p.head_dim) * a.group * 2,
                                 static_cast<cuuint64_t>(p.q_stride) * 2};
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(a.group), 1,
                             static_cast<cuuint32_t>(kTensorTileRows / a.group)};
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  const CUtensorMapDataType type =
      p.dtype == FGW_DTYPE_BFLOAT16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  if (encode_tiled_cached(&qmap, type, 4, const_cast<void*>(p.q), dims, strides, box, ones,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
    return cudaErrorInvalidValue;
  }
  if (chunk_kv_maps(&kmap, &vmap, p, a) != CUDA_SUCCESS) return cudaErrorInvalidValue;
  return launch_after_plan(kernel, static_cast<unsigned>(a.programs), S::kThreads, S::kBytes, stream, qmap, kmap, vmap,
                           a, list);
}

template <typename T>
static cudaError_t launch_tensor_nb(const fgw_chunk_params& p, const ChunkArgs& a, const ChunkList& list, int device,
                                    cudaStream_t stream) {
  switch ((p.head_dim + 63) / 64) {
    case 1:
      return launch_tensor_t<T, 1>(p, a, list, device, stream);
    case 2:
      return launch_tensor_t<T, 2>(p, a, list, device, stream);
    case 3:
      return launch_tensor_t<T, 3>(p, a, list, device, stream);
    default:
      return launch_tensor_t<T, 4>(p, a, list, device, stream);
  }
}

cudaError_t launch_chunk_tensor(const fgw_chunk_params& p, ChunkArgs a, const ChunkList& list, int device,
                                   cudaStream_t stream) {
  return p.dtype == FGW_DTYPE_BFLOAT16 ? launch_tensor_nb<__nv_bfloat16>(p, a, list, device, stream)
                                       : launch_tensor_nb<__half>(p, a, list, device, stream);
}

}  // namespace fgw
