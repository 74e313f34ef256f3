// Chunk attention, decode kernel: items of at most 16, 32 or 64 (token, query head) rows of one request and key
// head.
//
// Bound by HBM: each item reads its K and V once and computes little per byte, so the kernel is a stream of K/V tiles
// with a short chain of arithmetic behind it. One persistent CTA per SM: a producer warp keeps a ring of K/V tiles full
// (TMA through the page table, about 190 KB in flight or in use), eight consumer warps share each tile: scores by keys
// (a warp takes 16 or 8 of them), one exchange of row maxima through shared memory, P to shared memory, then P V by
// values (a warp takes an eighth of the head). So a warp holds an eighth of O, nothing is left to add up across warps
// at the end of an item, and up to 64 rows fit; two barriers of the eight warps per tile are the price. (Each warp
// carrying its own keys to the end, with the whole O of 16 rows in registers, needed no barrier per tile but took 5200
// cycles to merge the warps' states: 25.0 us against 18.3 us for eight single tokens.) m16n8k16 MMAs: tcgen05's
// 128-row form would leave most rows of its tile empty and carry the scores through TMEM twice.
//
// The work is split without a plan kernel: every CTA sums the units of all requests and finds the start of its own
// range. That costs two or three trips to L2 before the first load; a plan kernel ahead of it took 6 us by itself. Divisions by
// variables, chains of which stood between those trips, are multiplications (FastDiv): 18.3 to 14.2 us.
//
// Measured: 64 tokens over caches of up to 8K (1.28 GB, pages of 16) 216 us, 5.91 TB/s, 0.90 of the copy rate; the rest is
// the start (cursor, first loads) and the merge, some 14 us in all. Eight tokens over 1K (21 MB): 14 us, of which
// the start takes 3, the stream 4 and the merge kernel 4.
#include <algorithm>
#include <type_traits>

#include "fgw_chunk.cuh"

namespace fgw {

constexpr int kDecodeMinUnits = 2;  // units a program takes at least: a piece costs a merge

// NB blocks of 64 values per head, MT tiles of 16 rows per item.
template <int NB, int MT>
struct DecodeShape {
  static constexpr int kBN = chunk_decode_keys(NB, MT);
  static constexpr int kWarps = 8;                     // consumer warps
  static constexpr int kThreads = 32 * (kWarps + 1);
  static constexpr int kRows = 16 * MT;
  static constexpr int kDim = NB * 64;
  static constexpr int kKeys = kBN / kWarps;           // keys of a warp: 16 or 8
  static constexpr int kBlockBytes = kBN * 128;        // 64 values of every key
  static constexpr int kTileBytes = NB * kBlockBytes;  // K or V tile
  static constexpr int kQBytes = kRows * kDim * 2;
  static constexpr int kPBytes = kRows * kBN * 2;
  static constexpr int kMaxBytes = kRows * kWarps * 4;
  static constexpr int kRoom = 232448 - 2048 - kQBytes - kPBytes - kMaxBytes;
  static constexpr int kStages = kRoom / (2 * kTileBytes) < 8 ? kRoom / (2 * kTileBytes) : 8;
  static constexpr int kQ = kStages * 2 * kTileBytes;
  static constexpr int kP = kQ + kQBytes;
  static constexpr int kMax = kP + kPBytes;            // [kRows][kWarps] maxima, then sums
  static constexpr int kBar = kMax + kMaxBytes;
  static constexpr int kFlag = kBar + 2 * kStages * 8;
  static constexpr int kBytes = kFlag + 16 + 1024;
  static_assert(kBytes + 512 <= 232448 && kStages >= 2, "shared memory of one CTA");
};

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}

template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A CTA's range of units of all items, laid out by request, row and key head.
struct DecodeCursor {
  int b, row, hk, off;   // next item and the units of it before the range
  long long u, u_end;    // units left
  long long quotient;    // every program's units, the first `remainder` have one more
  int remainder;
};

// The program that holds unit u.
__device__ __forceinline__ int range_of(const DecodeCursor& k, long long u) {
  const long long longer = k.remainder * (k.quotient + 1);
  if (u < longer) return static_cast<int>(divide(u, static_cast<int>(k.quotient) + 1));
  return k.remainder + static_cast<int>(divide(u - longer, static_cast<int>(k.quotient)));
}

// Units of request b's items for one key head.
template <int kKeys>
__device__ __forceinline__ long long request_units(const ChunkArgs& a, int b) {
  const NewTokens nt = new_tokens(a.cu, a.tokens, b);
  const int len = held_tokens(a.lens, b, a.width, a.page);
  const int rows = item_rows(a, nt.count, true);
  long long units = 0;
  for (int r = 0; r < rows; ++r) units += item_units<kKeys>(a, nt.count, len, r * a.tokens_per_item);
  return units;
}

// Thread t takes the t-th of kThreads equal runs of requests, so one sum over the CTA gives the total and one over the
// threads before it the run that holds the range's start, which its thread then walks.
template <int kThreads, int kKeys>
__device__ __forceinline__ DecodeCursor decode_cursor(const ChunkArgs& a, long long* shared, DecodeCursor* found) {
  const int run = a.batch <= kThreads ? 1 : (a.batch + kThreads - 1) / kThreads;
  const int begin = min(static_cast<int>(threadIdx.x) * run, a.batch), end = min(begin + run, a.batch);
  long long first_units = 0, mine = 0;
  for (int b = begin; b < end; ++b) {
    const long long units = request_units<kKeys>(a, b);
    if (b == begin) first_units = units;
    mine += units;
  }
  mine *= a.kv_heads;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long before = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, before, d);
    if (lane >= d) before += up;
  }
  if (lane == 31) shared[warp] = before;
  if (threadIdx.x == 0) found->u = found->u_end = 0;
  __syncthreads();
  long long total = 0, base = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w == warp) base = total;
    total += shared[w];
  }
  before += base - mine;  // units of the runs before this one
  const int programs = static_cast<int>(max(1ll, min(static_cast<long long>(a.programs), total / kDecodeMinUnits)));
  const int p = blockIdx.x;
  const long long quotient = divide(total, programs);
  const int remainder = static_cast<int>(total - quotient * programs);
  const long long u = range_start(quotient, remainder, p), u_end = range_start(quotient, remainder, p + 1);
  if (p < programs && u < u_end && before <= u && u < before + mine) {
    long long left = u - before, units = first_units;
    int b = begin;
    while (left >= units * a.kv_heads) {
      left -= units * a.kv_heads;
      units = request_units<kKeys>(a, ++b);
    }
    const NewTokens nt = new_tokens(a.cu, a.tokens, b);
    const int len = held_tokens(a.lens, b, a.width, a.page);
    int row = 0;
    int w = item_units<kKeys>(a, nt.count, len, 0);
    while (left >= static_cast<long long>(w) * a.kv_heads) {
      left -= static_cast<long long>(w) * a.kv_heads;
      ++row;
      w = item_units<kKeys>(a, nt.count, len, row * a.tokens_per_item);
    }
    const int hk = static_cast<int>(divide(left, w));
    *found = {b, row, hk, static_cast<int>(left - static_cast<long long>(hk) * w), u, u_end, quotient, remainder};
  }
  __syncthreads();
  return *found;
}

template <int kKeys>
__device__ __forceinline__ bool next_segment(const ChunkArgs& a, DecodeCursor& k, ChunkSegment& s) {
  if (k.u >= k.u_end) return false;
  NewTokens nt = new_tokens(a.cu, a.tokens, k.b);
  while (k.row >= item_rows(a, nt.count, true)) {  // on to the next request with rows
    ++k.b;
    k.row = 0;
    nt = new_tokens(a.cu, a.tokens, k.b);
  }
  const int t0 = k.row * a.tokens_per_item;
  const int len = held_tokens(a.lens, k.b, a.width, a.page);
  const int units = item_units<kKeys>(a, nt.count, len, t0);
  const int count = static_cast<int>(min(static_cast<long long>(units - k.off), k.u_end - k.u));
  make_segment<kKeys>(a, s, k.b, k.hk, nt, len, t0, units, k.off, count);
  s.end_u = k.u - k.off + units;
  k.u += count;
  k.off += count;
  if (k.off >= units) {
    k.off = 0;
    if (++k.hk == a.kv_heads) {
      k.hk = 0;
      ++k.row;
    }
  }
  return true;
}

// Mask of a register of two 16-bit V values, of keys `key` and `key + 1`, that keeps those below the limit.
__device__ __forceinline__ uint32_t kept_keys(int key, int limit) {
  return key + 1 < limit ? 0xffffffffu : (key < limit ? 0x0000ffffu : 0u);
}

// Byte offset of 16-byte chunk `chunk` of row `row` in a tile of 128-byte rows, blocks of 64 values `block` bytes apart,
// in TMA's 128-byte swizzle.
__device__ __forceinline__ uint32_t swizzled(int row, int chunk, int block) {
  return (chunk >> 3) * block + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
}

template <typename T, int NB, int MT>
__global__ void __launch_bounds__(DecodeShape<NB, MT>::kThreads, 1)
    chunk_decode_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                        const __grid_constant__ ChunkArgs a) {
  using S = DecodeShape<NB, MT>;
  using Tr = ElemTraits<T>;
  constexpr int NS = S::kStages, NW = S::kWarps, BN = S::kBN, kRows = S::kRows;
  constexpr int kConsumers = NW * 32;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBar);
  uint64_t* empty = full + NS;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + S::kFlag);  // a consumer's wait gave up
  __shared__ long long scan[S::kThreads / 32];
  __shared__ DecodeCursor found;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == NW * 32) {
    tma_prefetch_desc(&kmap);
    tma_prefetch_desc(&vmap);
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], NW);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (threadIdx.x == 0) {
    a.slots.errors[blockIdx.x] = make_int2(0, 0);
    a.slots.cuts[blockIdx.x] = {0, 0, 0, -1};
  }
  grid_dependents_launch();
  DecodeCursor cur = decode_cursor<S::kThreads, BN>(a, scan, &found);  // with barriers of the whole CTA
  ChunkSegment sg;

  if (warp == NW) {
    // ---------------------------------------------------------------------------------- producer
    // Lane l issues the l-th box of a tile: boxes x blocks of 64 values x {K, V}, at most 32 of them.
    const int boxes = BN / a.box_rows;
    const int which = lane / (boxes * NB);  // 0: K, 1: V, more: idle
    const int box = lane % boxes, blk = (lane / boxes) % NB;
    const uint32_t box_bytes = a.box_rows * 128;
    const uint64_t policy = l2_policy_evict_first();
    bool ok = true;
    uint32_t st = 0, phase = 0, issued = 0;  // issued: stages given to loads
    while (ok && next_segment<BN>(a, cur, sg)) {
      const int32_t* table = a.table + static_cast<long long>(sg.b) * a.width;
      for (int j = 0; j < sg.n && ok; ++j) {
        const int tok = (sg.n_begin + j) * BN + box * a.box_rows;
        const bool load = which < 2 && tok < sg.limit;
        const int page = a.by_page.quotient(tok);
        const int row = load ? table[page] * a.page + tok - page * a.page : 0;
        const int loads = __popc(__ballot_sync(0xffffffffu, load));
        ok = __all_sync(0xffffffffu, mbar_wait(&empty[st], phase ^ 1, a.budget_ns));
        if (!ok) {
          if (lane == 0) chunk_error(a, 70);
          break;
        }
        if (lane == 0) mbar_arrive_expect_tx(&full[st], loads * box_bytes);
        ++issued;
        __syncwarp();
        if (load) {
          uint8_t* dst = smem + (2 * st + which) * S::kTileBytes + blk * S::kBlockBytes + box * box_bytes;
          tma_load_3d_hint(dst, which ? &vmap : &kmap, &full[st], blk * 64, sg.hk, row, policy);
        }
        if (++st == NS) {
          st = 0;
          phase ^= 1;
        }
      }
    }
    // Leave no copy in flight, whichever role gave up: the last load of every stage lands before the CTA may end.
    for (uint32_t i = issued > NS ? issued - NS : 0; i < issued; ++i) {
      mbar_wait(&full[i % NS], (i / NS) & 1, kDrainBudgetNs);
    }
    return;
  }

  // ------------------------------------------------------------------------------------ consumers
  float* row_max = reinterpret_cast<float*>(smem + S::kMax);  // [row][warp]
  const int g = lane / 4, c2 = (lane % 4) * 2;  // accumulator rows g and g + 8, columns c2 and c2 + 1
  const uint32_t base = smem_u32(smem);
  const uint32_t q_at = base + S::kQ, p_at = base + S::kP;
  uint32_t st = 0, phase = 0;
  bool aborted = false;  // uniform over the consumers
  while (next_segment<BN>(a, cur, sg)) {
    int seen[MT][2];
    long long out_at[MT][2];  // element offset of the row's output, -1: no row
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int r = mt * 16 + g + 8 * u, i = a.by_group.quotient(r);
        const bool valid = i < sg.count;
        seen[mt][u] = valid ? seen_keys(a, sg, i) : 0;
        out_at[mt][u] = valid ? (sg.token0 + i) * a.out_stride + static_cast<long long>(sg.hk * a.group + r - i * a.group) * a.dim
                              : -1;
      }
    }
    if (sg.n == 0) {  // no keys: zeros
      for (int i = threadIdx.x; i < sg.count * a.group * a.dim / 8; i += kConsumers) {
        const int r = i / (a.dim / 8);
        T* out = static_cast<T*>(a.out) + (sg.token0 + r / a.group) * a.out_stride +
                 static_cast<long long>(sg.hk * a.group + r % a.group) * a.dim;
        reinterpret_cast<uint4*>(out)[i % (a.dim / 8)] = make_uint4(0, 0, 0, 0);
      }
      continue;
    }
    // Q of the item's rows to shared memory
    for (int i = threadIdx.x; i < kRows * S::kDim / 8; i += kConsumers) {
      const int r = i / (S::kDim / 8), chunk = i % (S::kDim / 8);
      uint4 x = make_uint4(0, 0, 0, 0);
      if (r < sg.count * a.group && chunk * 8 < a.dim) {
        const int t = a.by_group.quotient(r);
        x = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + (sg.token0 + t) * a.q_stride +
                                                 static_cast<long long>(sg.hk * a.group + r - t * a.group) * a.dim) + chunk);
      }
      *reinterpret_cast<uint4*>(smem + S::kQ + swizzled(r, chunk, kRows * 128)) = x;
    }
    named_barrier_sync(1, kConsumers);
    float o[MT][NB][4], m[MT][2], l[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int i = 0; i < NB; ++i) o[mt][i][0] = o[mt][i][1] = o[mt][i][2] = o[mt][i][3] = 0.f;
      m[mt][0] = m[mt][1] = -INFINITY;
      l[mt][0] = l[mt][1] = 0.f;
    }
    for (int j = 0; j < sg.n; ++j) {
      const bool got = __all_sync(0xffffffffu, mbar_wait(&full[st], phase, a.budget_ns));
      if (!got && lane == 0) {
        chunk_error(a, 71);
        *abort_flag = 1;
      }
      const int key0 = (sg.n_begin + j) * BN + warp * S::kKeys;  // this warp's first key
      const uint32_t ktile = base + 2 * st * S::kTileBytes, vtile = ktile + S::kTileBytes;
      constexpr int NT = S::kKeys / 8;
      float s[MT][NT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int i = 0; i < NT; ++i) s[mt][i][0] = s[mt][i][1] = s[mt][i][2] = s[mt][i][3] = 0.f;
      }
      // S = Q K^T, 16 values per step; with 8 keys one ldmatrix serves two steps
#pragma unroll
      for (int ks = 0; ks < NB * 4; ks += 3 - NT) {
        uint32_t b[4];
        if constexpr (NT == 2) {
          ldmatrix_x4(b, ktile + swizzled(warp * 16 + (lane / 16) * 8 + lane % 8, ks * 2 + (lane / 8) % 2, S::kBlockBytes));
        } else {
          ldmatrix_x4(b, ktile + swizzled(warp * 8 + lane % 8, ks * 2 + lane / 8, S::kBlockBytes));
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int k = 0; k < 3 - NT; ++k) {
            uint32_t q[4];
            ldmatrix_x4(q, q_at + swizzled(mt * 16 + lane % 16, (ks + k) * 2 + lane / 16, kRows * 128));
            if constexpr (NT == 2) {
              mma_16816<T>(s[mt][0], q, b[0], b[1]);
              mma_16816<T>(s[mt][NT - 1], q, b[2], b[3]);
            } else {
              mma_16816<T>(s[mt][0], q, b[2 * k], b[2 * k + 1]);
            }
          }
        }
      }
      // keys a row does not see, then the warp's part of the row maxima
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float top = -INFINITY;
#pragma unroll
          for (int i = 0; i < NT; ++i) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float& x = s[mt][i][2 * u + e];
              if (key0 + i * 8 + c2 + e >= seen[mt][u]) x = -INFINITY;
              top = fmaxf(top, x);
            }
          }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          if (lane % 4 == 0) row_max[(mt * 16 + g + 8 * u) * NW + warp] = top;
        }
      }
      named_barrier_sync(1, kConsumers);
      if (*abort_flag != 0) {  // all warps read it here, between the same two barriers
        aborted = true;
        break;
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int r = mt * 16 + g + 8 * u;
          const float4 t0 = *reinterpret_cast<const float4*>(&row_max[r * NW]);
          const float4 t1 = *reinterpret_cast<const float4*>(&row_max[r * NW + 4]);
          const float top = fmaxf(fmaxf(fmaxf(t0.x, t0.y), fmaxf(t0.z, t0.w)), fmaxf(fmaxf(t1.x, t1.y), fmaxf(t1.z, t1.w)));
          const float next = fmaxf(m[mt][u], top * a.scale_log2);  // scale > 0; -inf stays -inf
          const float ref = next == -INFINITY ? 0.f : next;
          const float keep = fast_exp2(m[mt][u] - ref);
          l[mt][u] *= keep;
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            o[mt][i][2 * u] *= keep;
            o[mt][i][2 * u + 1] *= keep;
          }
          m[mt][u] = next;
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            const uint32_t p = Tr::pack2(fast_exp2(fmaf(s[mt][i][2 * u], a.scale_log2, -ref)),
                                         fast_exp2(fmaf(s[mt][i][2 * u + 1], a.scale_log2, -ref)));
            // the sum is over the rounded weights that multiply V
            const float2 w = Tr::unpack2(p);
            l[mt][u] += w.x + w.y;
            const int key = warp * S::kKeys + i * 8;
            *reinterpret_cast<uint32_t*>(smem + S::kP + swizzled(r, key / 8, kRows * 128) + c2 * 2) = p;
          }
        }
      }
      named_barrier_sync(1, kConsumers);
      // O += P V for this warp's eighth of the values, 32 keys per step. V rows past the last visible key hold whatever
      // the ring or the page holds, and a zero weight times NaN is NaN: an item's last tile zeroes them as operands.
      const int tile0 = (sg.n_begin + j) * BN;
      auto weigh = [&](auto tail) {
#pragma unroll
        for (int kk = 0; kk < BN / 32; ++kk) {
          uint32_t p[MT][2][4];
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            ldmatrix_x4(p[mt][0], p_at + swizzled(mt * 16 + lane % 16, kk * 4 + lane / 16, kRows * 128));
            ldmatrix_x4(p[mt][1], p_at + swizzled(mt * 16 + lane % 16, kk * 4 + 2 + lane / 16, kRows * 128));
          }
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            uint32_t b[4];
            ldmatrix_x4_trans(b, vtile + swizzled(kk * 32 + lane, warp * NB + i, S::kBlockBytes));
            if constexpr (decltype(tail)::value) {
#pragma unroll
              for (int k = 0; k < 4; ++k) b[k] &= kept_keys(tile0 + kk * 32 + k * 8 + c2, sg.limit);
            }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              mma_16816<T>(o[mt][i], p[mt][0], b[0], b[1]);
              mma_16816<T>(o[mt][i], p[mt][1], b[2], b[3]);
            }
          }
        }
      };
      if (sg.limit - tile0 < BN) {
        weigh(std::true_type{});
      } else {
        weigh(std::false_type{});
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
      if (++st == NS) {
        st = 0;
        phase ^= 1;
      }
    }
    if (aborted) break;
    // the rows' sums over all warps (row_max's readers have passed the last barrier)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        l[mt][u] += __shfl_xor_sync(0xffffffffu, l[mt][u], 1);
        l[mt][u] += __shfl_xor_sync(0xffffffffu, l[mt][u], 2);
        if (lane % 4 == 0) row_max[(mt * 16 + g + 8 * u) * NW + warp] = l[mt][u];
      }
    }
    named_barrier_sync(1, kConsumers);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int r = mt * 16 + g + 8 * u;
        const float4 t0 = *reinterpret_cast<const float4*>(&row_max[r * NW]);
        const float4 t1 = *reinterpret_cast<const float4*>(&row_max[r * NW + 4]);
        const float total = ((t0.x + t0.y) + (t0.z + t0.w)) + ((t1.x + t1.y) + (t1.z + t1.w));
        const bool none = total == 0.f;  // no key seen: zeros; a NaN among the scores stays one
        const float inv = 1.f / total;
        if (sg.slot < 0) {
          if (out_at[mt][u] < 0) continue;
          T* out = static_cast<T*>(a.out) + out_at[mt][u];
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            const int at = (warp * NB + i) * 8;
            if (at >= a.dim) continue;
            const float x = none ? 0.f : o[mt][i][2 * u] * inv, y = none ? 0.f : o[mt][i][2 * u + 1] * inv;
            *reinterpret_cast<uint32_t*>(out + at + c2) = Tr::pack2(x, y);
          }
        } else {
          // a piece: normalised O and base-2 LSE to its slot
          const long long at_row = static_cast<long long>(sg.slot) * kRows + r;
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            const int at = (warp * NB + i) * 8;
            if (at >= a.dim) continue;
            const float x = none ? 0.f : o[mt][i][2 * u] * inv, y = none ? 0.f : o[mt][i][2 * u + 1] * inv;
            *reinterpret_cast<float2*>(a.slots.o + at_row * a.dim + at + c2) = make_float2(x, y);
          }
          if (warp == 0 && lane % 4 == 0) a.slots.lse[at_row] = none ? kEmptyLse : m[mt][u] + fast_log2(total);
        }
      }
    }
    if (sg.starts && threadIdx.x == 0) {
      a.slots.cuts[blockIdx.x] = {sg.token0, sg.count, sg.hk, range_of(cur, sg.end_u - 1)};
    }
  }
  // So that what follows this kernel follows the tensor kernel ahead of it too; CTAs that gave up come here as well.
  grid_dependency_wait();
}

template <typename T, int NB, int MT>
static cudaError_t launch_decode_t(const fgw_chunk_params& p, ChunkArgs a, int device, cudaStream_t stream) {
  using S = DecodeShape<NB, MT>;
  auto kernel = chunk_decode_kernel<T, NB, MT>;
  cudaError_t err = prepare_kernel(reinterpret_cast<const void*>(kernel), S::kBytes, device, nullptr);
  if (err != cudaSuccess) return err;
  a.box_rows = chunk_box_rows(p.page_size, S::kBN);
  CUtensorMap kmap, vmap;
  if (chunk_kv_maps(&kmap, &vmap, p, a) != CUDA_SUCCESS) return cudaErrorInvalidValue;
  if (a.split) {  // after the tensor kernel, which it does not wait for until its end
    return launch_after_plan(kernel, static_cast<unsigned>(a.programs), S::kThreads, S::kBytes, stream, kmap, vmap, a);
  }
  kernel<<<a.programs, S::kThreads, S::kBytes, stream>>>(kmap, vmap, a);
  return cudaGetLastError();
}

template <typename T, int NB>
static cudaError_t launch_decode_nb(const fgw_chunk_params& p, const ChunkArgs& a, int device, cudaStream_t stream) {
  switch (a.small_rows) {
    case 16:
      return launch_decode_t<T, NB, 1>(p, a, device, stream);
    case 32:
      return launch_decode_t<T, NB, 2>(p, a, device, stream);
    default:
      return launch_decode_t<T, NB, 4>(p, a, device, stream);
  }
}

template <typename T>
static cudaError_t launch_decode_type(const fgw_chunk_params& p, const ChunkArgs& a, int device, cudaStream_t stream) {
  switch ((p.head_dim + 63) / 64) {
    case 1:
      return launch_decode_nb<T, 1>(p, a, device, stream);
    case 2:
      return launch_decode_nb<T, 2>(p, a, device, stream);
    case 3:
      return launch_decode_nb<T, 3>(p, a, device, stream);
    default:
      return launch_decode_nb<T, 4>(p, a, device, stream);
  }
}

cudaError_t launch_chunk_decode(const fgw_chunk_params& p, ChunkArgs a, int device, cudaStream_t stream) {
  return p.dtype == FGW_DTYPE_BFLOAT16 ? launch_decode_type<__nv_bfloat16>(p, a, device, stream)
                                       : launch_decode_type<__half>(p, a, device, stream);
}

}  // namespace fgw
