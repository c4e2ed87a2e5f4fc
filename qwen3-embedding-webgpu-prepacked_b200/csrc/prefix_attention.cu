// Attention of a batch of requests behind one cached prefix (tcgen05 + TMA).
//
//   o_r = sum_j p_rj v_j / sum_j p_rj,  p_rj = exp(q_r . k_j / sqrt(128) - m_r)
//
// over the keys j that row r keeps: the prefix's, then its request's own up to
// itself (prefix_plan.h has the rule and the lists of work).
//
// A block of work is `tile_tokens` x 2 packed query tokens x the `group` query
// heads of one kv head: two 128-row tiles A and B, row = token * group + head.
// Rows of different requests share a tile, so the prefix is read and
// multiplied once for the whole block; own keys of other requests are masked.
//
// Warp roles:
//   warp 0      TMA producer: Q, then K_j / V_j into a ring of 4 slots (16-bit
//               prefix) or 3 (8-bit; raw prefix tiles into a ring of 3 stages). Q is
//               loaded again once the last S of an item is done
//   warp 1      TMEM owner; lane 0 issues every tcgen05.mma and commit
//   warps 4-7   softmax of tile A, one thread a row
//   warps 8-11  softmax of tile B
//   warps 2-3 (16-bit prefix) or 12-15 (8-bit) prepare tiles: raw 8-bit tiles are
//               converted into their slot; V tiles with masked keys are cleared of
//               values that are not finite (guard, below)
// TMEM: S_A, S_B (P over them, as 16-bit pairs), O_A, O_B; 512 columns.
// MMA order per key tile: S_A(j), PV_B(j-1), S_B(j), PV_A(j), so the softmax of
// one tile runs under the MMAs of the other.
// In the dual form (few blocks: each has one row tile) the key tiles of a block
// alternate between A and B, both over the same Q, and the two O are merged in
// tensor memory at the end. It has kernels of its own: with both forms in one, the
// softmax warps spilled registers (4 x 5000 tokens 3% slower). For the same reason a launch
// has blocks of one form only: cutting the last round's blocks into one row tile each
// made 16 x 500 tokens 202 us instead of 195.
//
// Guard. A masked key has p = 0, but the MMA still multiplies: 0 * inf = NaN
// would reach rows of other requests. So V tiles in which some row drops a key
// are searched, values that are not finite replaced by 0, and the rows that
// keep such a key get it back in the epilogue (found again by a slow search).
//
// Split. With few blocks the tiles of a block are dealt to a cluster of 2 to 8
// CTAs, each with its own running maximum and sum; at the end every CTA
// leaves its O, m and l in shared memory and merges a share of the rows from
// all of them. No workspace, one launch, and an order that does not vary.
//
// Bits. Scores, m, l and O are f32. P is rounded once to the 16-bit type of V, as both operands
// of a tcgen05 f16 MMA have one type: at most half a step of p (2^-11, bf16 2^-8) for
// each key, against l of the unrounded values. The relative error against 64 bits (rms) grows
// from the output's own rounding, 0.00021 in f16 and 0.0017 in bf16, to 0.00029 and 0.0023; a P of 32
// bits would take the tf32 form, at half the rate, with V as 32 bits too.
//
// What bounds it (16/8 heads). Long requests: a key tile of two row tiles takes about
// 4070 cycles, 1.4 times what its MMAs need (about 2900): S waits for PV, as P lies over
// it, and the exponentials of one row tile take longer than the MMAs of the other. 4 x 5000
// bf16 tokens behind 5000: 1215 to 1380 us with the clock, 890 to 1010 TFLOP/s (0.55 to
// 0.62 of measured). 16 x 500 f16 behind 2000 in E4M3: 193 to 196 us, 755 TFLOP/s; 504 blocks
// for 148 SMs, so the fourth round is less than half full. Small calls: latency. 16 x 1 behind
// 1000 in E4M3: 12.3 to 12.9 us, 16 x 15..150 behind 176: 16.1 to 16.8 us; loads, S, softmax,
// PV, merge and the launch follow one another, on instructions that are not cached yet.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "attn_common.cuh"
#include "convert.cuh"
#include "internal.h"
#include "prefix_attention.h"
#include "ptx.cuh"

namespace qwa {
namespace {
using namespace attn;

// Threads, registers and shared memory of a format. A 16-bit prefix needs no
// conversion: warps 2-3 prepare, the softmax warps get 200 registers and the
// ring four slots. For 8 bits a fourth warpgroup of four preparing warps joins
// and takes its registers from the others, and raw tiles wait in a ring of
// their own. (Two warps with the codes prefetched into registers took 6900 cycles for
// a tile of 128 keys, three times its MMAs.)
template <int kFormat>
struct Layout {
  static constexpr bool kConverts = kFormat != kKvPlain;
  static constexpr int kThreads = kConverts ? 512 : 384;
  static constexpr int kPrepWarp0 = kConverts ? 12 : 2;
  static constexpr int kPrepWarps = kConverts ? 4 : 2;
  static constexpr int kSlotEmptyArrivals = slot_empty_arrivals(kPrepWarps);
  static constexpr int kRegsLaunch = kConverts ? 128 : 168;
  static constexpr int kRegsSupport = kConverts ? 72 : 104;  // producer and issuer
  static constexpr int kRegsPrep = 72;                       // of the fourth warpgroup
  static constexpr int kRegsSoftmax = kConverts ? 184 : 200;
  static_assert(128 * kRegsSupport + 256 * kRegsSoftmax + (kConverts ? 128 * kRegsPrep : 0) <=
                    kThreads * kRegsLaunch,
                "register split");
  static constexpr int kSlots = kConverts ? 3 : 4;   // K_j and V_j tiles in use
  static constexpr int kStages = kConverts ? 3 : 0;  // raw 8-bit tiles on their way
  static constexpr uint32_t kSlotOff = 2 * kTileBytes;  // after Q_A, Q_B
  static constexpr uint32_t kStageOff = kSlotOff + kSlots * kTileBytes;
  static constexpr uint32_t kEpiOff = kStageOff + kStages * (kTileBytes / 2);
  static constexpr uint32_t kStatOff = kEpiOff + 8 * 2048;  // 2 KB for each softmax warp
  static constexpr uint32_t kBarOff = kStatOff + 2048;      // dual: (m, l) of 256 threads
  enum Bar : int {
    kQFull = 0,
    kQEmpty,
    kSlotEmpty,
    kLanded = kSlotEmpty + kSlots,  // a tile has been copied into the slot
    kReady = kLanded + kSlots,      // the preparing warps are done with it
    kOwnGo = kReady + kSlots,       // 8 bits: an own tile may be copied into the slot
    kStageFull = kOwnGo + kSlots,
    kStageEmpty = kStageFull + kStages,
    kSFull = kStageEmpty + kStages,
    kPLo = kSFull + 2,
    kPHi = kPLo + 2,
    kOFinal = kPHi + 2,
    kStat = kOFinal + 2,   // dual: (m, l) of the warpgroup are in shared memory
    kTaken = kStat + 2,    // dual: the warpgroup has read both O
    kDrain = kTaken + 2,
    kNumBars
  };
  static constexpr uint32_t kHolderOff = kBarOff + 8 * kNumBars;
  static constexpr uint32_t kAbortOff = kHolderOff + 4;
  static constexpr uint32_t kLimitOff = kHolderOff + 8;
  // li + 1 of the last item with values put aside. The preparing warps may be
  // ahead of an epilogue: it takes a later item's number for its own, and its search
  // then finds what there is. They may be ahead of one another too, so the number
  // only rises: a late warp must not take back what another has noted.
  static constexpr uint32_t kBadOff = kLimitOff + 8;
  static constexpr uint32_t kSmemUsed = kBadOff + 4;
  static constexpr uint32_t kSmemBytes = kSmemUsed;
  static_assert(kLimitOff % 8 == 0 && kSmemBytes <= 232448, "shared memory budget");
  // split: O of row tile A over Q (64 KB), of B over the first two slots, and
  // (m, l) of the rows where the other form stages its output
  static constexpr uint32_t kPartOffB = kSlotOff;
};
constexpr int kSoftmaxWarp0 = 4;
constexpr int kMaxSplit = 8;  // CTAs of a cluster (the portable size)

template <bool kBf16>
__host__ __device__ constexpr uint32_t idesc_16(uint32_t m, uint32_t n, bool b_mn_major) {
  // A and B format: 0 = f16, 1 = bf16
  return idesc_f16_f32(m, n, b_mn_major) | (kBf16 ? (1u << 7) | (1u << 10) : 0u);
}

// One half of PV (keys 0..63 or 64..127): at most `nk` steps of 16 in all.
template <bool kBf16>
__device__ __forceinline__ void issue_pv_part(uint32_t d_tmem, uint32_t p_tmem, uint64_t v_desc,
                                              bool accumulate, int nk, int half) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int kk = 4 * half + i;
    if (kk < nk)
      mma_ts(d_tmem, p_tmem + kk * 8, v_desc + ((kk * 2048) >> 4), idesc_16<kBf16>(128, 128, true),
             (accumulate || kk > 0) ? 1u : 0u);
  }
}

// exp2(a * scale - m) of 32 scores, packed to 16-bit pairs in a[0..15]; returns
// their sum (of the unrounded values, in f32).
template <bool kBf16>
__device__ __forceinline__ float exp_pack(uint32_t (&a)[32], float scale, float m) {
  const uint64_t s2 = f2_pack(scale, scale), nm2 = f2_pack(-m, -m);
  uint64_t sum2 = f2_pack(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float y0, y1;
    f2_unpack(fma2(f2_pack(__uint_as_float(a[2 * i]), __uint_as_float(a[2 * i + 1])), s2, nm2),
              y0, y1);
    const float e0 = ex2(y0), e1 = ex2(y1);
    sum2 = add2(sum2, f2_pack(e0, e1));
    a[i] = pack2<kBf16>(e0, e1);
  }
  float sum0, sum1;
  f2_unpack(sum2, sum0, sum1);
  return sum0 + sum1;
}

// The keys that a row keeps, in the numbering of one key tensor: [lo, hi], of
// those (sparse) only < cut or >= wlo.
struct Kept {
  int lo, hi, cut, wlo;
};
__device__ __forceinline__ Kept kept_keys(const PrefixArgs& a, bool own, PrefixRow r) {
  if (own) {
    const int own_prefix = max(0, a.sparse_prefix - a.prefix_len);
    return {r.lo, r.hi, r.lo + own_prefix, max(0, r.hi - a.window + 1)};
  }
  return {0, a.prefix_len - 1, a.sparse_prefix,
          max(0, a.prefix_len + r.hi - r.lo - a.window + 1)};
}
__device__ __forceinline__ uint32_t kept_bits(const Kept& k, int k0, int sparse) {
  uint32_t m = low_bits(k.hi - k0 + 1) & ~low_bits(k.lo - k0);
  if (sparse) m &= low_bits(k.cut - k0) | ~low_bits(k.wlo - k0);
  return m;
}
__device__ __forceinline__ void mask_keys(uint32_t (&a)[32], const Kept& k, int k0, int sparse) {
  const uint32_t m = kept_bits(k, k0, sparse);
  if (__all_sync(0xffffffffu, m == 0xffffffffu)) return;
#pragma unroll
  for (int c = 0; c < 32; ++c)
    if (!((m >> c) & 1u)) a[c] = __float_as_uint(-INFINITY);
}

// ------------------------------------------------------------- 8-bit tiles
// Clears the halves of w whose exponent is all ones (inf, NaN).
template <bool kBf16>
__device__ __forceinline__ uint32_t finite_only(uint32_t w, bool& bad) {
  constexpr uint32_t kExp = kBf16 ? 0x7f807f80u : 0x7c007c00u;
  const uint32_t hit = __vcmpeq2(w & kExp, kExp);
  bad |= hit != 0;
  return w & ~hit;
}

__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t x, uint32_t y, uint32_t z,
                                             uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x), "r"(y), "r"(z),
               "r"(w)
               : "memory");
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// Converts a landed raw tile (128 rows of 128 codes) into the slot's swizzled
// layout. Lane (w, l) takes the 16 codes of unit l % 8 in the rows 16 i + 4 w +
// l / 8, i < 8; `scale` is the byte of row 16 (l / 4) + 4 w + l % 4. kGuard: values
// that are not finite become 0; returns whether there were any.
template <bool kBf16, int kFormat, bool kGuard>
__device__ __forceinline__ bool convert_tile(uint32_t stage, uint32_t slot, uint32_t scale, int w,
                                             int lane) {
  bool bad = false;
  const int u = lane & 7;    // dims 16 u .. 16 u + 15
  const int odd = u >> 2;    // lanes of the second half write their odd unit first (banks)
  const int r0 = 4 * w + (lane >> 3);
  const uint32_t from = stage + r0 * 128 + u * 16;
  // r % 8 is the same for all of a lane's rows, 16 apart
  const uint32_t base = slot + odd * kHalfBytes + r0 * 128;
  const uint32_t at_a = base + (static_cast<uint32_t>((u & 3) * 2 + odd) ^ (r0 & 7)) * 16;
  const uint32_t at_b = base + (static_cast<uint32_t>((u & 3) * 2 + 1 - odd) ^ (r0 & 7)) * 16;
  const uint32_t mine = pair_pow2<kBf16>(static_cast<int>(scale) - 127);
  // all loads first: they and the stores are kept in order, and a load behind
  // a store would wait for the conversion before it
  uint4 raw[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) raw[i] = ld_shared_v4(from + i * 2048);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t sc = __shfl_sync(0xffffffffu, mine, i * 4 + (lane >> 3));
    const uint32_t c[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
    uint32_t v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      v[j] = code_pair<kBf16, kFormat == kKvE4M3>((c[j >> 1] >> (16 * (j & 1))) & 0xffffu, sc);
    if constexpr (kGuard) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = finite_only<kBf16>(v[j], bad);
    }
    st_shared_v4(at_a + i * 2048, odd ? v[4] : v[0], odd ? v[5] : v[1], odd ? v[6] : v[2],
                 odd ? v[7] : v[3]);
    st_shared_v4(at_b + i * 2048, odd ? v[0] : v[4], odd ? v[1] : v[5], odd ? v[2] : v[6],
                 odd ? v[3] : v[7]);
  }
  return bad;
}
// Clears a landed V tile (rows [0, width)) of values that are not finite.
template <bool kBf16, int kWarps>
__device__ __forceinline__ bool guard_tile(uint32_t slot, int width, int w, int lane) {
  bool bad = false;
  for (int r = 4 * w + (lane >> 3); r < width; r += 4 * kWarps) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t at = slot + h * kHalfBytes + r * 128 + (lane & 7) * 16;
      uint4 v = ld_shared_v4(at);
      bool hit = false;
      v.x = finite_only<kBf16>(v.x, hit);
      v.y = finite_only<kBf16>(v.y, hit);
      v.z = finite_only<kBf16>(v.z, hit);
      v.w = finite_only<kBf16>(v.w, hit);
      if (hit) st_shared_v4(at, v.x, v.y, v.z, v.w);
      bad |= hit;
    }
  }
  return bad;
}

// What a row gets back for the values that the guard put aside: per dim of a
// 32-dim chunk whether it keeps a key with +inf, -inf or NaN there.
struct Aside {
  uint32_t pos, neg, nan;
};
template <bool kBf16, int kFormat>
__device__ __forceinline__ Aside find_aside(const PrefixArgs& a, int tile_beg, int tile_end,
                                         PrefixRow row, int head, int chunk) {
  Aside s{0u, 0u, 0u};
  for (int j = tile_beg; j < tile_end; ++j) {
    const PrefixTile tile = a.tiles[j];
    if (!(tile.info & kTileGuard)) continue;
    const bool own = tile.info & kTileOwn;
    const Kept k = kept_keys(a, own, row);
    const int width = tile.info & kTileWidthMask;
    for (int c = 0; c < width; c += 32) {
      uint32_t bits = kept_bits(k, tile.key + c, a.sparse);
      if (width - c < 32) bits &= low_bits(width - c);
      for (; bits; bits &= bits - 1) {
        const int64_t key = tile.key + c + __ffs(bits) - 1;
        for (int d = 0; d < 32; ++d) {
          const int dim = chunk * 32 + d;
          uint32_t v;
          if (own) {
            v = a.v_own[key * a.v_stride + head * kHeadDim + dim];
          } else if (kFormat == kKvPlain) {
            v = static_cast<const uint16_t*>(
                a.v_prefix)[(key * a.kv_heads + head) * kHeadDim + dim];
          } else {
            const int64_t at = key * a.kv_heads + head;
            const int e = static_cast<int>(a.v_scale[at]) - 127;
            const uint32_t code = static_cast<const uint8_t*>(a.v_prefix)[at * kHeadDim + dim];
            v = code_pair<kBf16, kFormat == kKvE4M3>(code, pair_pow2<kBf16>(e)) & 0xffffu;
          }
          constexpr uint32_t kExp = kBf16 ? 0x7f80u : 0x7c00u;
          if ((v & kExp) != kExp) continue;
          if ((v & 0x7fffu) != kExp) s.nan |= 1u << d;
          else if (v & 0x8000u) s.neg |= 1u << d;
          else s.pos |= 1u << d;
        }
      }
    }
  }
  return s;
}
__device__ __forceinline__ float with_aside(float o, const Aside& s, int d) {
  if ((s.nan >> d) & 1u) o += NAN;
  if ((s.pos >> d) & 1u) o += INFINITY;
  if ((s.neg >> d) & 1u) o -= INFINITY;
  return o;
}

// Puts them back into O in tensor memory (chunks [c_beg, c_end) at t_o) for the
// lanes with `mine`. Out of line: it is rare, and its registers are not the
// epilogue's.
template <bool kBf16, int kFormat>
__device__ __noinline__ void put_back(const PrefixArgs& a, int tile_beg, int tile_end,
                                      PrefixRow row, int head, int c_beg, int c_end, uint32_t t_o,
                                      bool mine) {
#pragma unroll 1
  for (int c = c_beg; c < c_end; ++c) {
    uint32_t o[32];
    tmem_ld32(t_o + 32 * c, o);
    tmem_wait_ld();
    reg_fence32(o);
    if (mine) {
      const Aside s = find_aside<kBf16, kFormat>(a, tile_beg, tile_end, row, head, c);
#pragma unroll
      for (int i = 0; i < 32; ++i)
        o[i] = __float_as_uint(with_aside(__uint_as_float(o[i]), s, i));
    }
    __syncwarp();
    tmem_st32(t_o + 32 * c, o);
    tmem_wait_st();
  }
}

__device__ __forceinline__ float4 ld_cluster_v4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster_v2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

// The work of one CTA: items [beg, end) of the list with all their tiles, or
// (split) the share `rank` of `ranks` of one item's tiles.
struct Share {
  int beg, end, rank, ranks;
};
template <bool kSplit>
__device__ __forceinline__ Share my_share(const PrefixArgs& a) {
  if constexpr (kSplit) {
    const int item = blockIdx.x / a.splits;
    return {item, item + 1, static_cast<int>(cluster_ctarank()), a.splits};
  } else {
    return {a.cta_offsets[blockIdx.x], a.cta_offsets[blockIdx.x + 1], 0, 1};
  }
}
template <bool kSplit>
__device__ __forceinline__ void share_tiles(const Share& s, const PrefixItem& item, int& beg,
                                            int& end) {
  beg = item.tile_beg;
  end = item.tile_end;
  if constexpr (kSplit) {
    const int n = end - beg;
    end = beg + n * (s.rank + 1) / s.ranks;
    beg = beg + n * s.rank / s.ranks;
  }
}

// The preparing warps (the file's head): w counts them from 0. They follow every
// use of the ring, because a parity says nothing to a role that is more than a
// phase away: each waits for its slot to be empty, then converts, or (8 bits) lets
// the producer, which runs ahead on raw tiles, load an own tile. A slot is empty again
// only with an arrival of each of them, so none falls more than a phase behind
// (slot_empty_arrivals).
template <bool kBf16, int kFormat, bool kSplit>
__device__ __forceinline__ void prepare_tiles(const PrefixArgs& args, const Share& share,
                                              uint32_t sbase, int w, int lane,
                                              volatile int* abort_flag,
                                              const volatile unsigned long long* wait_limit,
                                              int* bad_item) {
  using L = Layout<kFormat>;
  auto bar = [&](int i) -> uint32_t { return sbase + L::kBarOff + 8u * i; };
  // a warp-wide wait: every lane leaves it with the same answer
  auto wait = [&](uint32_t b, uint32_t parity, int code) -> bool {
    const bool got = mbar_wait(b, parity, abort_flag, args.status, code, wait_limit);
    return __all_sync(0xffffffffu, got);
  };
  auto publish = [&](int s, bool bad, int li) {
    if (__any_sync(0xffffffffu, bad) && lane == 0) atomicMax(bad_item, li + 1);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(L::kReady + s));
  };
  int s = 0;               // slot of the current use
  uint32_t parity = 1;     // of the phase that says the slot is empty
  int g = 0;               // raw stage of the next 8-bit tile, and its parity
  uint32_t g_parity = 0;
  uint32_t landed = 0;     // bit slot: parity of the slot's next copy
  for (int it = share.beg, li = 0; it < share.end; ++it, ++li) {
    const PrefixItem item = args.items[it];
    int tb, te;
    share_tiles<kSplit>(share, item, tb, te);
    // this lane's scale byte of a tile, fetched one tile ahead
    auto scale_of = [&](const PrefixTile& tile, int kv) -> uint32_t {
      const int r = tile.key + 16 * (lane >> 2) + 4 * w + (lane & 3);
      if ((tile.info & kTileOwn) || r >= args.prefix_len) return 127;
      return __ldg((kv ? args.v_scale : args.k_scale) +
                   static_cast<int64_t>(r) * args.kv_heads + item.head);
    };
    PrefixTile next = args.tiles[tb];
    uint32_t scale = 0;
    if (L::kConverts) scale = scale_of(next, 0);
    for (int j = tb; j < te; ++j) {
      const PrefixTile tile = next;
      next = args.tiles[j + 1 < te ? j + 1 : j];
      const bool own = tile.info & kTileOwn;
      const bool guard = tile.info & kTileGuard;
      for (int kv = 0; kv < 2; ++kv) {
        const uint32_t slot = sbase + L::kSlotOff + s * kTileBytes;
        if (!wait(bar(L::kSlotEmpty + s), parity, kDevTimeoutSlotEmpty)) return;
        if (L::kConverts && !own) {
          const uint32_t now = scale;
          scale = kv == 0 ? scale_of(tile, 1) : scale_of(next, 0);
          if (!wait(bar(L::kStageFull + g), g_parity, kDevTimeoutSlotFull)) return;
          const uint32_t stage = sbase + L::kStageOff + g * (kTileBytes / 2);
          bool bad = false;
          if (kv == 1 && guard)
            bad = convert_tile<kBf16, kFormat, true>(stage, slot, now, w, lane);
          else
            convert_tile<kBf16, kFormat, false>(stage, slot, now, w, lane);
          publish(s, bad, li);  // all lanes have read the raw tile
          if (lane == 0) mbar_arrive(bar(L::kStageEmpty + g));
          if (++g == L::kStages) {
            g = 0;
            g_parity ^= 1;
          }
        } else {
          if (L::kConverts && w == 0 && lane == 0) mbar_arrive(bar(L::kOwnGo + s));
          const uint32_t copy = (landed >> s) & 1u;
          landed ^= 1u << s;
          if (kv == 1 && guard) {
            if (!wait(bar(L::kLanded + s), copy, kDevTimeoutSlotFull)) return;
            publish(s, guard_tile<kBf16, L::kPrepWarps>(slot, tile.info & kTileWidthMask, w, lane),
                    li);
          }
        }
        // every lane is here: `wait` and `publish` gather the warp
        if (lane == 0) mbar_arrive(bar(L::kSlotEmpty + s));
        if (++s == L::kSlots) {
          s = 0;
          parity ^= 1;
        }
      }
    }
  }
}

// kDual: every block has one row tile (block_tokens == tile_tokens).
template <bool kBf16, int kFormat, bool kSplit, bool kDual>
__global__ void __launch_bounds__(Layout<kFormat>::kThreads, 1)
    prefix_attention_kernel(const __grid_constant__ CUtensorMap tm_q,
                            const __grid_constant__ CUtensorMap tm_k,
                            const __grid_constant__ CUtensorMap tm_v,
                            const __grid_constant__ CUtensorMap tm_pk,
                            const __grid_constant__ CUtensorMap tm_pv,
                            const __grid_constant__ PrefixArgs args) {
  using L = Layout<kFormat>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw;
  const uint32_t sbase = smem_addr(smem);
  if (sbase & 1023u) {  // the swizzled tiles need it; the same in every CTA
    if (threadIdx.x == 0) atomicCAS(args.status, 0, kDevSharedLayout);
    return;
  }
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + L::kHolderOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kAbortOff);
  volatile unsigned long long* wait_limit =
      reinterpret_cast<volatile unsigned long long*>(smem + L::kLimitOff);
  int* bad_item = reinterpret_cast<int*>(smem + L::kBadOff);
  auto bar = [&](int i) -> uint32_t { return sbase + L::kBarOff + 8u * i; };

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const Share share = my_share<kSplit>(args);

  if (threadIdx.x == 0) {
    mbar_init(bar(L::kQFull), 1);
    mbar_init(bar(L::kQEmpty), 1);
    *bad_item = 0;
    for (int i = 0; i < L::kSlots; ++i) {
      mbar_init(bar(L::kSlotEmpty + i), L::kSlotEmptyArrivals);
      mbar_init(bar(L::kLanded + i), 1);
      mbar_init(bar(L::kReady + i), L::kPrepWarps);
      mbar_init(bar(L::kOwnGo + i), 1);
    }
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(bar(L::kStageFull + i), 1);
      mbar_init(bar(L::kStageEmpty + i), L::kPrepWarps);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(bar(L::kSFull + x), 1);
      mbar_init(bar(L::kPLo + x), 128);
      mbar_init(bar(L::kPHi + x), 128);
      mbar_init(bar(L::kOFinal + x), 1);
      mbar_init(bar(L::kStat + x), 128);
      mbar_init(bar(L::kTaken + x), 128);
    }
    mbar_init(bar(L::kDrain), 1);
    *abort_flag = 0;
    *wait_limit = args.wait_ns;
    fence_mbar_init();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    tma_prefetch_desc(&tm_pk);
    tma_prefetch_desc(&tm_pv);
  }
  if (warp == 1) {
    tmem_alloc(smem_addr(tmem_holder), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  // rows of a 128-row tile that a Q load fills
  const int tile_rows = args.group * args.tile_tokens;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::kRegsSupport));
    if (warp == 0) {
      // ---------------------------------------------------------- producer
      if (lane == 0) {
        bool ok = true;
        int s = 0;
        uint32_t parity = 1;  // of the phase that says slot s is empty (16 bits)
        int g = 0;
        uint32_t g_parity = 1;   // raw stage g is empty
        uint32_t go_parity = 0;  // bit slot: parity of the slot's next own tile (8 bits)
        uint32_t landed = 0;     // bit slot: parity of the slot's next copy
        // The last phase issued on each barrier that counts copies (Q, slots,
        // stages), waited for before exit so that no copy lands after it. Only
        // copies complete these phases, one in flight on each.
        uint32_t fly_on = 0, fly_parity = 0;
        auto fly = [&](int i, uint32_t p) {
          fly_on |= 1u << i;
          fly_parity = (fly_parity & ~(1u << i)) | (p << i);
        };
        for (int it = share.beg, li = 0; ok && it < share.end; ++it, ++li) {
          const PrefixItem item = args.items[it];
          int tb, te;
          share_tiles<kSplit>(share, item, tb, te);
          const int nx = item.tokens > args.tile_tokens ? 2 : 1;
          if (!(ok = mbar_wait(bar(L::kQEmpty), (li & 1) ^ 1, abort_flag, args.status,
                               kDevTimeoutQ, wait_limit)))
            break;
          mbar_arrive_expect_tx(bar(L::kQFull), nx * tile_rows * 256);
          fly(0, li & 1);
          for (int x = 0; x < nx; ++x) {
            const uint32_t dst = sbase + x * kTileBytes;
            const int t0 = item.row0 + x * args.tile_tokens;
            tma_load_3d(dst, &tm_q, bar(L::kQFull), 0, item.head * args.group, t0);
            tma_load_3d(dst + kHalfBytes, &tm_q, bar(L::kQFull), 64, item.head * args.group, t0);
          }
          PrefixTile next = args.tiles[tb];
          for (int j = tb; ok && j < te; ++j) {
            const PrefixTile tile = next;  // the next one is loaded a tile ahead
            next = args.tiles[j + 1 < te ? j + 1 : j];
            const bool own = tile.info & kTileOwn;
            for (int kv = 0; kv < 2; ++kv) {
              if (L::kConverts && !own) {  // a raw tile, converted by the preparing warps
                if (!(ok = mbar_wait(bar(L::kStageEmpty + g), g_parity, abort_flag, args.status,
                                     kDevTimeoutSlotEmpty, wait_limit)))
                  break;
                mbar_arrive_expect_tx(bar(L::kStageFull + g), kTileBytes / 2);
                fly(1 + L::kSlots + g, g_parity ^ 1);
                tma_load_3d(sbase + L::kStageOff + g * (kTileBytes / 2), kv ? &tm_pv : &tm_pk,
                            bar(L::kStageFull + g), 0, item.head, tile.key);
                if (++g == L::kStages) {
                  g = 0;
                  g_parity ^= 1;
                }
              } else {
                if (L::kConverts) {
                  if (!(ok = mbar_wait(bar(L::kOwnGo + s), (go_parity >> s) & 1u, abort_flag,
                                       args.status, kDevTimeoutSlotEmpty, wait_limit)))
                    break;
                  go_parity ^= 1u << s;
                } else if (!(ok = mbar_wait(bar(L::kSlotEmpty + s), parity, abort_flag,
                                            args.status, kDevTimeoutSlotEmpty, wait_limit))) {
                  break;
                }
                const uint32_t dst = sbase + L::kSlotOff + s * kTileBytes;
                const CUtensorMap* tm = own ? (kv ? &tm_v : &tm_k) : (kv ? &tm_pv : &tm_pk);
                const uint32_t full = bar(L::kLanded + s);
                fly(1 + s, (landed >> s) & 1u);
                landed ^= 1u << s;
                mbar_arrive_expect_tx(full, kTileBytes);
                tma_load_3d(dst, tm, full, 0, item.head, tile.key);
                tma_load_3d(dst + kHalfBytes, tm, full, 64, item.head, tile.key);
              }
              if (++s == L::kSlots) {
                s = 0;
                parity ^= 1;
              }
            }
          }
        }
        bool drained = true;
        for (int i = 0; i < 1 + L::kSlots + L::kStages; ++i)
          if ((fly_on >> i) & 1u) {
            const int b = i == 0 ? L::kQFull
                                 : (i <= L::kSlots ? L::kLanded + i - 1
                                                   : L::kStageFull + i - 1 - L::kSlots);
            drained &= mbar_drain(bar(b), (fly_parity >> i) & 1u, *wait_limit);
          }
        if (!drained) atomicCAS(args.status, 0, kDevTimeoutDrain);
      }
    } else if (warp == 1) {
      // -------------------------------------------------------- MMA issuer
      if (lane == 0) {
        const uint64_t qa = smem_desc_sw128(sbase, 16, 1024);
        const uint64_t k_desc0 = smem_desc_sw128(sbase + L::kSlotOff, 16, 1024);
        const uint64_t v_desc0 = smem_desc_sw128(sbase + L::kSlotOff, kHalfBytes, 1024);
        bool ok = true;
        int s = 0;               // slot of the next use
        uint32_t landed = 0;     // bit slot: parity of its next copy
        uint32_t ready = 0;      // bit slot: parity of its next prepared tile
        uint32_t t_par = 0;      // bit x: parity of row tile x's next key tile
        bool have_prev = false;  // a PV still to issue, of row tile prev_x
        int prev_x = 1, prev_v = 0, prev_nk = 8;
        bool prev_acc = false, prev_last = false;
        // waits for the tile in slot s, whoever completes it
        auto wait_tile = [&](bool copied, bool prepared) -> bool {
          const uint32_t l = (landed >> s) & 1u, r = (ready >> s) & 1u;
          if (copied) landed ^= 1u << s;
          if (prepared) ready ^= 1u << s;
          return mbar_wait(prepared ? bar(L::kReady + s) : bar(L::kLanded + s), prepared ? r : l,
                           abort_flag, args.status, kDevTimeoutSlotFull, wait_limit);
        };
        // PV of row tile x with the V tile in slot v, as P arrives in halves
        auto run_pv = [&](int x, int v, bool acc, int nk) -> bool {
          const uint64_t vd = v_desc0 + ((v * kTileBytes) >> 4);
          const uint32_t o = tmem + 256 + x * 128, p = tmem + x * 128;
          const uint32_t par = (t_par >> x) & 1u;
          t_par ^= 1u << x;
          if (!mbar_wait(bar(L::kPLo + x), par, abort_flag, args.status, kDevTimeoutPFull,
                         wait_limit))
            return false;
          tc_fence_after();
          issue_pv_part<kBf16>(o, p, vd, acc, nk, 0);
          if (!mbar_wait(bar(L::kPHi + x), par, abort_flag, args.status, kDevTimeoutPFull,
                         wait_limit))
            return false;
          tc_fence_after();
          issue_pv_part<kBf16>(o, p, vd, acc, nk, 1);
          return true;
        };
        auto issue_prev = [&]() -> bool {
          if (!run_pv(kDual ? prev_x : 1, prev_v, prev_acc, prev_nk)) return false;
          tc_commit(bar(L::kSlotEmpty + prev_v));
          if (prev_last) tc_commit(bar(L::kOFinal + (kDual ? prev_x : 1)));
          have_prev = false;
          return true;
        };
        for (int it = share.beg, li = 0; ok && it < share.end; ++it, ++li) {
          const PrefixItem item = args.items[it];
          int tb, te;
          share_tiles<kSplit>(share, item, tb, te);
          const int nx = item.tokens > args.tile_tokens ? 2 : 1;
          int next_info = args.tiles[tb].info;
          // Q is loaded once the last S MMAs of the item before are done; if it
          // is still on its way, the pending PV_B goes first
          if (have_prev && !mbar_try_wait(bar(L::kQFull), li & 1) && !(ok = issue_prev())) break;
          if (!(ok = mbar_wait(bar(L::kQFull), li & 1, abort_flag, args.status, kDevTimeoutQ,
                               wait_limit)))
            break;
          for (int j = tb; j < te; ++j) {
            const int info = next_info;
            next_info = args.tiles[j + 1 < te ? j + 1 : j].info;
            const int width = info & kTileWidthMask;
            const bool converted = L::kConverts && !(info & kTileOwn);
            const bool last = j == te - 1;
            const int x = kDual ? (j - tb) & 1 : 0;
            const int sk = s;
            if (!(ok = wait_tile(!converted, converted))) break;
            s = s + 1 == L::kSlots ? 0 : s + 1;
            tc_fence_after();
            const uint64_t k_desc = k_desc0 + ((sk * kTileBytes) >> 4);
            const uint32_t idesc = idesc_16<kBf16>(128, width, false);
            // (the empty asm keeps the compiler from holding sixteen descriptors
            // of Q in registers through the loop)
            uint64_t q_now = qa;
            asm volatile("" : "+l"(q_now));
            // S of a row tile goes over its P
            if (kDual && have_prev && prev_x == x && !(ok = issue_prev())) break;
            issue_qk(tmem + x * 128, q_now, k_desc, idesc);
            tc_commit(bar(L::kSFull + x));
            if (have_prev && !(ok = issue_prev())) break;
            if (!kDual && nx == 2) {
              q_now = qa + (kTileBytes >> 4);
              asm volatile("" : "+l"(q_now));
              issue_qk(tmem + 128, q_now, k_desc, idesc);
              tc_commit(bar(L::kSFull + 1));
            }
            tc_commit(bar(L::kSlotEmpty + sk));
            if (last) tc_commit(bar(L::kQEmpty));
            const int sv = s;
            if (!(ok = wait_tile(!converted, converted || (info & kTileGuard)))) break;
            s = s + 1 == L::kSlots ? 0 : s + 1;
            if (kDual) {
              prev_x = x;
              prev_acc = j - tb >= 2;
              prev_last = j + 2 >= te;
            } else {
              if (!(ok = run_pv(0, sv, j > tb, width / 16))) break;
              if (last) tc_commit(bar(L::kOFinal + 0));
              if (nx == 1) {
                tc_commit(bar(L::kSlotEmpty + sv));
                continue;
              }
              prev_acc = j > tb;
              prev_last = last;
            }
            have_prev = true;
            prev_v = sv;
            prev_nk = width / 16;
          }
        }
        if (ok && have_prev) ok = issue_prev();
        tc_commit(bar(L::kDrain));
        if (!mbar_drain(bar(L::kDrain), 0, *wait_limit))
          atomicCAS(args.status, 0, kDevTimeoutDrain);
      }
    } else if (!L::kConverts) {
      prepare_tiles<kBf16, kFormat, kSplit>(args, share, sbase, warp - L::kPrepWarp0, lane,
                                            abort_flag, wait_limit, bad_item);
    }
  } else if (L::kConverts && warp >= L::kPrepWarp0) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::kRegsPrep));
    prepare_tiles<kBf16, kFormat, kSplit>(args, share, sbase, warp - L::kPrepWarp0, lane,
                                          abort_flag, wait_limit, bad_item);
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::kRegsSoftmax));
    // ----------------------------------------------------------- softmax
    const int x = (warp - kSoftmaxWarp0) >> 2;
    const int sub = warp & 3;
    const int row = sub * 32 + lane;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(sub * 32) << 16);
    const uint32_t t_s = t_lane + x * 128;
    const uint32_t t_o = t_lane + 256 + x * 128;
    const float scale = args.scale_log2;
    const int token = row / args.group;  // of this row in its tile
    bool ok = true;
    // a warp leaves a wait as one: what follows are instructions of whole warps
    auto wait = [&](uint32_t b, uint32_t parity, int code) -> bool {
      const bool got = mbar_wait(b, parity, abort_flag, args.status, code, wait_limit);
      return __all_sync(0xffffffffu, got);
    };
    // parities of this warpgroup's next key tile (bit 0), item with any (1) and
    // dual item (2)
    uint32_t ph = 0;
    for (int it = share.beg, li = 0; ok && it < share.end; ++it, ++li) {
      // (what only the epilogue needs is read again there: registers)
      int tb, te, first_token, tokens;
      PrefixRow mine = {0, -1};
      {
        const PrefixItem item = args.items[it];
        share_tiles<kSplit>(share, item, tb, te);
        tokens = item.tokens;
        if (!kDual && x == 1 && tokens <= args.tile_tokens) continue;  // no row tile B
        first_token = kDual ? 0 : x * args.tile_tokens;
        if (row < tile_rows && first_token + token < tokens)
          mine = args.rows[item.row0 + first_token + token];
      }
      // dual: A takes the even key tiles, B the odd ones
      const int j0 = kDual ? tb + x : tb;
      constexpr int step = kDual ? 2 : 1;
      float m_run = -INFINITY, l_run = 0.f;
      PrefixTile next = args.tiles[j0 < te ? j0 : tb];
      for (int j = j0; j < te; j += step, ph ^= 1u) {
        const PrefixTile tile = next;
        next = args.tiles[j + step < te ? j + step : j];
        if (!(ok = wait(bar(L::kSFull + x), ph & 1u, kDevTimeoutSFull)))
          break;
        tc_fence_after();
        const bool narrow = (tile.info & kTileWidthMask) <= 64;
        uint32_t a0[32], a1[32], a2[32], a3[32];
        tmem_ld32(t_s + 0, a0);
        tmem_ld32(t_s + 32, a1);
        if (!narrow) {
          tmem_ld32(t_s + 64, a2);
          tmem_ld32(t_s + 96, a3);
        }
        tmem_wait_ld();
        reg_fence32(a0);
        reg_fence32(a1);
        if (!narrow) {
          reg_fence32(a2);
          reg_fence32(a3);
        }
        if (tile.info & kTileMask) {
          const Kept kept = kept_keys(args, tile.info & kTileOwn, mine);
          mask_keys(a0, kept, tile.key, args.sparse);
          mask_keys(a1, kept, tile.key + 32, args.sparse);
          if (!narrow) {
            mask_keys(a2, kept, tile.key + 64, args.sparse);
            mask_keys(a3, kept, tile.key + 96, args.sparse);
          }
        }
        float tmax = fmaxf(chunk_max(a0), chunk_max(a1));
        if (!narrow) tmax = fmaxf(tmax, fmaxf(chunk_max(a2), chunk_max(a3)));
        tmax *= scale;
        const float m_new = fmaxf(m_run, tmax);
        bool need = false;
        float f = 1.f;
        if (j == j0) {
          m_run = m_new;
        } else if (m_new > m_run + 8.f) {
          // lazy rescale: P stays <= 2^8 against a maximum that is out of date
          need = true;
          f = ex2(m_run - m_new);
          l_run *= f;
          m_run = m_new;
        }
        const float m_use = (m_run == -INFINITY) ? 0.f : m_run;
        float sum = exp_pack<kBf16>(a0, scale, m_use) + exp_pack<kBf16>(a1, scale, m_use);
        tmem_st16(t_s + 0, a0);
        tmem_st16(t_s + 16, a1);
        if (__any_sync(0xffffffffu, need)) {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t o[32];
            tmem_ld32(t_o + 32 * c, o);
            tmem_wait_ld();
            reg_fence32(o);
            const uint64_t f2 = f2_pack(f, f);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float r0, r1;
              f2_unpack(mul2(f2_pack(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1])), f2),
                        r0, r1);
              o[2 * i] = __float_as_uint(r0);
              o[2 * i + 1] = __float_as_uint(r1);
            }
            tmem_st32(t_o + 32 * c, o);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(bar(L::kPLo + x));
        if (!narrow) {
          sum += exp_pack<kBf16>(a2, scale, m_use) + exp_pack<kBf16>(a3, scale, m_use);
          tmem_st16(t_s + 32, a2);
          tmem_st16(t_s + 48, a3);
          tmem_wait_st();
          tc_fence_before();
        }
        l_run += sum;
        mbar_arrive(bar(L::kPHi + x));
      }
      // Epilogue. (m, l) of a warpgroup without tiles stay (-inf, 0).
      if (!ok) break;
      const PrefixItem item = args.items[it];
      // (the empty asm keeps what follows from group and lane out of registers
      // that the tile loop needs)
      int group = args.group, ln = lane;
      asm volatile("" : "+r"(group), "+r"(ln));
      if (j0 < te) {
        if (!(ok = wait(bar(L::kOFinal + x), (ph >> 1) & 1u, kDevTimeoutOFinal)))
          break;
        ph ^= 2u;
        tc_fence_after();
      }
      // o = w * (own O) + w2 * (the other's); dual: both warpgroups have the same
      // lanes of tensor memory, so each merges half of the dims
      float w = 1.f, w2 = 0.f;
      bool both = false;
      if constexpr (kDual) {
        float2* stat = reinterpret_cast<float2*>(smem + L::kStatOff);
        stat[x * 128 + row] = make_float2(m_run, l_run);
        tc_fence_before();
        mbar_arrive(bar(L::kStat + x));
        if (!(ok = wait(bar(L::kStat + (x ^ 1)), (ph >> 2) & 1u, kDevTimeoutOFinal)))
          break;
        tc_fence_after();
        const float2 ml = stat[(x ^ 1) * 128 + row];
        const float m = fmaxf(m_run, ml.x);
        w = m_run == -INFINITY ? 0.f : ex2(m_run - m);
        w2 = ml.x == -INFINITY ? 0.f : ex2(ml.x - m);
        l_run = w * l_run + w2 * ml.y;
        m_run = m;
        both = te - tb > 1;
      }
      // (a row that exists keeps itself)
      const bool aside = mine.hi >= 0 && *const_cast<volatile int*>(bad_item) > li;
      const float inv_l = 1.f / l_run;
      const int chunks = kDual ? 2 : 4, c0 = kDual ? 2 * x : 0;
      const uint32_t stage = sbase + L::kEpiOff + (warp - kSoftmaxWarp0) * 2048;
      // own O (a warpgroup without tiles, B of one key tile, has A's), and what
      // the guard put aside back into the O of the larger weight
      const uint32_t t_own = j0 < te ? t_o : t_lane + 256;
      if (__any_sync(0xffffffffu, aside)) {
        const bool to_own = j0 >= te || w >= w2;
        put_back<kBf16, kFormat>(args, tb, te, mine, item.head, c0, c0 + chunks, t_own,
                                 aside && to_own);
        if (both)
          put_back<kBf16, kFormat>(args, tb, te, mine, item.head, c0, c0 + chunks,
                                   t_lane + 256 + (x ^ 1) * 128, aside && !to_own);
      }
      // split: f32 rows of 512 bytes, their 16-byte units swizzled by the row: of
      // tile A over Q, of B over the first slots (at A's end Q is read no more,
      // at B's no slot is)
      const uint32_t part = sbase + (kDual ? 0 : x) * L::kPartOffB + row * 512;
#pragma unroll 1
      for (int c = c0; c < c0 + chunks; ++c) {
        uint32_t o[32];
        if constexpr (kDual) {
          uint32_t o2[32];
          tmem_ld32(t_own + 32 * c, o);
          if (both) tmem_ld32(t_lane + 256 + (x ^ 1) * 128 + 32 * c, o2);
          tmem_wait_ld();
          reg_fence32(o);
          const float a = j0 < te ? w : w2;
          if (both) {
            reg_fence32(o2);
#pragma unroll
            for (int i = 0; i < 32; ++i)
              o[i] = __float_as_uint(fmaf(__uint_as_float(o2[i]), w2, __uint_as_float(o[i]) * a));
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * a);
          }
          if (c == c0 + 1) {
            tc_fence_before();
            mbar_arrive(bar(L::kTaken + x));
          }
        } else {
          tmem_ld32(t_o + 32 * c, o);
          tmem_wait_ld();
          reg_fence32(o);
        }
        if constexpr (kSplit) {
#pragma unroll
          for (int v = 0; v < 8; ++v)
            st_shared_v4(part + (static_cast<uint32_t>(c * 8 + v) ^ ln) * 16, o[4 * v],
                         o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
        } else {
          // 32 dims at a time: the warp's 32 rows of 64 bytes through its 2 KB,
          // out as 64-byte runs, eight rows an instruction
          __syncwarp();  // the chunk before has been read
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const uint32_t* p = o + 8 * v;
            uint32_t y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              y[i] = pack2<kBf16>(__uint_as_float(p[2 * i]) * inv_l,
                                  __uint_as_float(p[2 * i + 1]) * inv_l);
            // a row's unit v at v ^ (row / 2) % 4: two rows share 128 bytes of banks
            st_shared_v4(stage + ln * 64 + (v ^ ((ln >> 1) & 3)) * 16, y[0], y[1], y[2], y[3]);
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int rw = 8 * i + (ln >> 2), r = sub * 32 + rw;
            const int rt = r / group, rh = r - rt * group;
            const int tok = first_token + rt;
            const uint4 v =
                ld_shared_v4(stage + rw * 64 + ((ln & 3) ^ ((rw >> 1) & 3)) * 16);
            if (r < tile_rows && tok < item.tokens)
              *reinterpret_cast<uint4*>(args.out +
                                        (static_cast<int64_t>(item.row0 + tok) * args.q_heads +
                                         item.head * group + rh) *
                                            kHeadDim +
                                        c * 32 + (ln & 3) * 8) = v;
          }
        }
      }
      if (kSplit && !(kDual && x == 1))
        *reinterpret_cast<float2*>(smem + L::kEpiOff + ((kDual ? 0 : x) * 128 + row) * 8) =
            make_float2(m_run, l_run);
      tc_fence_before();
      __syncwarp();
      if constexpr (kDual) {
        // the next item's P, and with it PV over O, only once both have read O
        if (!(ok = wait(bar(L::kTaken + (x ^ 1)), (ph >> 2) & 1u, kDevTimeoutOFinal)))
          break;
        ph ^= 4u;
      }
    }
  }

  tc_fence_before();
  __syncwarp();
  if constexpr (kSplit) {
    // the cluster's O, m and l are in shared memory: each CTA merges its share
    // of the rows, a warp a row
    cluster_sync();
    if (warp >= kSoftmaxWarp0 && warp < kSoftmaxWarp0 + 8) {
      const PrefixItem item = args.items[share.beg];
      const int rows = item.tokens * args.group;  // of the block, those of B after A's
      const int per = (rows + share.ranks - 1) / share.ranks;
      const int end = min(rows, share.rank * per + per);
      // two rows at a time, all their loads in flight together
      for (int i = share.rank * per + (warp - kSoftmaxWarp0) * 2; i < end; i += 16) {
        float2 ml[2];
        float4 v[2][kMaxSplit];
        int rr[2], x[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = min(i + h, end - 1);
          x[h] = r >= tile_rows ? 1 : 0;
          rr[h] = r - x[h] * tile_rows;
          ml[h] = make_float2(-INFINITY, 0.f);
          if (lane < share.ranks)
            ml[h] = ld_cluster_v2(
                mapa_shared(sbase + L::kEpiOff + (x[h] * 128 + rr[h]) * 8, lane));
          const uint32_t at = sbase + x[h] * L::kPartOffB + rr[h] * 512 +
                              (static_cast<uint32_t>(lane) ^ (rr[h] & 31)) * 16;
#pragma unroll
          for (int k = 0; k < kMaxSplit; ++k)
            if (k < share.ranks) v[h][k] = ld_cluster_v4(mapa_shared(at, k));
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (i + h >= end) break;
          float m = ml[h].x;
#pragma unroll
          for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
          m = __shfl_sync(0xffffffffu, m, 0);
          const float w = ml[h].x == -INFINITY ? 0.f : ex2(ml[h].x - m);
          float l = w * ml[h].y;
#pragma unroll
          for (int o = 4; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
          l = __shfl_sync(0xffffffffu, l, 0);
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int k = 0; k < kMaxSplit; ++k) {
            if (k >= share.ranks) break;
            const float wk = __shfl_sync(0xffffffffu, w, k);
            acc.x = fmaf(wk, v[h][k].x, acc.x);
            acc.y = fmaf(wk, v[h][k].y, acc.y);
            acc.z = fmaf(wk, v[h][k].z, acc.z);
            acc.w = fmaf(wk, v[h][k].w, acc.w);
          }
          const float inv_l = 1.f / l;
          uint2 y;
          y.x = pack2<kBf16>(acc.x * inv_l, acc.y * inv_l);
          y.y = pack2<kBf16>(acc.z * inv_l, acc.w * inv_l);
          const int rt = rr[h] / args.group, rh = rr[h] - rt * args.group;
          const int64_t tok = item.row0 + x[h] * args.tile_tokens + rt;
          *reinterpret_cast<uint2*>(
              args.out + (tok * args.q_heads + item.head * args.group + rh) * kHeadDim +
              lane * 4) = y;
        }
      }
    }
    __syncwarp();
    cluster_sync();  // no CTA leaves while its shared memory is read
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

template <bool kBf16, int kFormat, bool kSplit, bool kDual>
cudaError_t launch(const PrefixMaps& m, const PrefixArgs& args, int grid, int splits,
                   cudaStream_t stream) {
  static bool configured[kMaxDevices] = {};
  auto kernel = prefix_attention_kernel<kBf16, kFormat, kSplit, kDual>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             Layout<kFormat>::kSmemBytes);
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(Layout<kFormat>::kThreads);
  cfg.dynamicSmemBytes = Layout<kFormat>::kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(splits);
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  if (kSplit) {
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, kernel, m.q, m.k, m.v, m.pk, m.pv, args);
}

template <bool kBf16, int kFormat>
cudaError_t launch_format(const PrefixMaps& m, const PrefixArgs& a, int grid,
                          cudaStream_t stream) {
  const bool split = a.splits > 1;
  if (a.one_tile)
    return split ? launch<kBf16, kFormat, true, true>(m, a, grid, a.splits, stream)
                 : launch<kBf16, kFormat, false, true>(m, a, grid, a.splits, stream);
  return split ? launch<kBf16, kFormat, true, false>(m, a, grid, a.splits, stream)
               : launch<kBf16, kFormat, false, false>(m, a, grid, a.splits, stream);
}

template <bool kBf16>
cudaError_t launch_typed(const PrefixMaps& m, const PrefixArgs& a, int format, int grid,
                         cudaStream_t stream) {
  switch (format) {
    case kKvE4M3: return launch_format<kBf16, kKvE4M3>(m, a, grid, stream);
    case kKvInt8: return launch_format<kBf16, kKvInt8>(m, a, grid, stream);
    default: return launch_format<kBf16, kKvPlain>(m, a, grid, stream);
  }
}

}  // namespace

int prefix_active_clusters(int splits) {
  using L = Layout<kKvInt8>;
  auto kernel = prefix_attention_kernel<false, kKvInt8, true, true>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmemBytes) !=
      cudaSuccess)
    return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(splits);
  cfg.blockDim = dim3(L::kThreads);
  cfg.dynamicSmemBytes = L::kSmemBytes;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(splits);
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int n = 0;
  return cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) == cudaSuccess ? n : 0;
}

cudaError_t launch_prefix_attention(const PrefixMaps& maps, const PrefixArgs& args, int bf16,
                                    int format, int grid, cudaStream_t stream) {
  if (grid <= 0) return cudaSuccess;
  return bf16 ? launch_typed<true>(maps, args, format, grid, stream)
              : launch_typed<false>(maps, args, format, grid, stream);
}

}  // namespace qwa
