// Attention of a batch's rows over a shared prefix on the tensor cores (tcgen05), fp16 queries, D = 64 or 128.
//
// The rows (b, i) of all sequences, up to 128 at a time, meet every key of the prefix once: S = Q K^T and O += P V with
// 128-key tiles, one CTA on an SM for a part of the prefix, which it walks from the latest tile to the earliest (the
// mathematics is in fpa_decode.cuh). With R rows there are R flops a byte in fp16 and 2 R in int8, so for few rows the
// prefix's bytes bound it; at 128 rows and D = 128 a tile takes 1024 cycles of MMAs, as many of exponentials, and its
// 64 KB take 2.8k cycles at an SM's share of the HBM rate (1024 from L2). Where the rows fill half or a quarter of the 128 lanes, they stand there twice or
// four times, and each copy takes its half or quarter of the tile's keys (its P stays zero for the others), so that no
// warp idles; the copies' softmax states join at the end.
//
// Warps 0-3 and 4-7: two softmax groups; a thread is a row (a TMEM lane). Group g takes keys 64 g .. 64 g + 63 of every
// tile, with its own running maximum, sum and O, so the groups never wait for each other and one's exponentials run
// beside the other's products and minima; their states join at the end. Each group's S is double-buffered (P overwrites
// the buffer it came from), so a tile's S is ready when its turn comes. Warps 8-11 and 12-15: K and V into the ring of 128-byte-swizzled tiles; fp16
// by cp.async directly, int8 by cp.async into a raw ring that each thread reads back itself, converts to fp16 (exact)
// and stores. Plain loads rather than TMA, because the last page's slots past the prefix must come out as zeros
// whatever they hold, and because codes have to be converted on the way. Warp 16: the MMAs. Warps 17 and 18: the keys'
// field and scales, alternate tiles. Every wait is bounded.
//
// On a B200: 120 rows behind 16383 fp16 tokens, 16 heads of 128, 40 us (403 TFLOP/s; 3.2k cycles for a tile of 128 keys); 64 rows
// behind 8192 int8 tokens, 12 heads of 64, 16 us, of which 11 are the CTA's start and end.
#include <cuda_fp16.h>

#include <type_traits>

#include "fpa_decode.cuh"
#include "fpa_sm100.cuh"

namespace fpa {
namespace {

using namespace sm100;

constexpr int kTile = 128;
constexpr int kPrefixThreads = 640;
constexpr int kLoaders = 128;   // of K, and as many of V
constexpr int kWarpMma = 16, kWarpField = 17;
constexpr int kParStages = 4;

template <int D, bool kInt8>
struct PrefixCfg {
  static constexpr int BOXB = kTile * 128;                // a tile's 64 columns
  static constexpr int TILEB = D / 64 * BOXB;             // K or V of a tile in fp16
  static constexpr int SLOTS = kInt8 ? (D == 64 ? 6 : 3) : (D == 64 ? 8 : 5);
  // Barriers that a unit's slot is free again: one for each slot and kind (K, V) that stands there. With an odd number
  // of slots both kinds take turns in a slot, and a loader, which only waits for the unit before its own, would miss every
  // other phase of a barrier that they shared: V of tile k could then pass before V of tile k - 3 has been read.
  static constexpr int EMPTIES = SLOTS % 2 ? 2 * SLOTS : SLOTS;
  static constexpr int RAWB = kInt8 ? kTile * D : 0;      // K or V of a tile in codes
  static constexpr int RAWS = kInt8 ? (D == 64 ? 3 : 2) : 0;  // of K, and as many of V
  static constexpr int PARF = kInt8 ? 8 : 4;              // floats of a pair of keys
  static constexpr int PARB = kTile / 2 * PARF * 4;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_RING = OFF_Q + TILEB;
  static constexpr int OFF_RAW = OFF_RING + SLOTS * TILEB;
  static constexpr int OFF_PAR = OFF_RAW + 2 * RAWS * RAWB;
  static constexpr int OFF_ML = OFF_PAR + kParStages * PARB;  // the states' maxima and sums [2][256]
  static constexpr int OFF_BAR = OFF_ML + 512 * 4;
  static constexpr int NBAR = SLOTS + EMPTIES + 2 * kParStages + 10;
  static constexpr int SMEM = OFF_BAR + NBAR * 8 + 16 + 1024;
  static constexpr int COL_S = 0, COL_O = 2 * kTile;  // S of tile k: + 128 (k & 1), of group g: + 64 g; O: + D g
  static constexpr uint32_t IDESC_S = idesc_f16(kTile, kTile, 0);
  static constexpr uint32_t IDESC_O = idesc_f16(kTile, D, 1);
  static_assert(SMEM <= 227 * 1024, "shared memory");
  static_assert(256 * (D + 4) * 4 <= SLOTS * TILEB + 2 * RAWS * RAWB, "the states join in the ring's place");
};

__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}
__device__ __forceinline__ void st_shared16(uint32_t dst, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t src) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(src) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Codes 2i, 2i + 1 of a word of four (each with 128 added) as halves.
template <uint32_t kSel>
__device__ __forceinline__ uint32_t code_pair(uint32_t x) {
  const uint32_t y = __byte_perm(x, 0x64646464u, kSel);
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&y), __floats2half2_rn(1152.f, 1152.f));
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Address of 16-byte chunk c of row r in a tile of [D / 64][128 rows][128 bytes] with the 128-byte swizzle.
__device__ __forceinline__ uint32_t tile_chunk(int r, int c) {
  return uint32_t((c >> 3) * (kTile * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// REP: how often the rows stand in the 128 lanes.
template <int D, bool kInt8, int REP>
__global__ void __launch_bounds__(kPrefixThreads, 1) prefix_tc_kernel(const __grid_constant__ DecodeParams p) {
  using C = PrefixCfg<D, kInt8>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* empty = full + C::SLOTS;
  uint64_t* par_full = empty + C::EMPTIES;
  uint64_t* par_empty = par_full + kParStages;
  uint64_t* s_full = par_empty + kParStages;
  uint64_t* p_full = s_full + 2;
  uint64_t* o_ready = p_full + 4;
  uint64_t* q_full = o_ready + 2;
  uint64_t* o_done = q_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_done + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const CacheView& c = p.c;
  const int h = blockIdx.z, R = p.B * p.n;
  constexpr int RP = kTile / REP;  // lanes of one copy
  const int r0 = blockIdx.y * RP, rows = min(RP, R - r0);
  // This CTA's tiles [t0, t1), walked downwards.
  const int tiles = (p.prefix_len + kTile - 1) / kTile, S = gridDim.x;
  const int each = tiles / S, more = tiles - each * S;
  const int t0 = int(blockIdx.x) * each + min(int(blockIdx.x), more);
  const int nt = each + (int(blockIdx.x) < more ? 1 : 0), t1 = t0 + nt;
  auto prefix_level = [&]() {
    return level_at(c, p.prefix_table[(p.prefix_len - 1) >> c.page_shift], h, p.prefix_len - 1);
  };

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::SLOTS; ++i) mbar_init(full + i, kLoaders);
    for (int i = 0; i < C::EMPTIES; ++i) mbar_init(empty + i, 1);
    for (int i = 0; i < kParStages; ++i) {
      mbar_init(par_full + i, 32);
      mbar_init(par_empty + i, 256);
    }
    // P of group g, tile k: barrier 2 g + (k & 1). A warp can be a tile ahead of another of its group, but not two: S of
    // tile k + 2 follows P V of tile k, which needs every warp's P.
    for (int i = 0; i < 4; ++i) mbar_init(p_full + i, 128);
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(o_ready + i, 1);
    }
    mbar_init(q_full, 256);
    mbar_init(o_done, 1);
    fence_mbar_init();
  }
  if (warp == kWarpMma) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // The launch before this one (row_min) has waited for everything earlier, so the cache and the queries can be read
  // at once; only the softmax warps wait, for the rows' minima.

  // Registers: 96 a thread at launch (61440 in all); 136 for the two softmax warpgroups, 64 for the other three (59392).
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;" ::: "memory");
    if (warp < kWarpMma) {
      // ------------------------------------------------------------------------------------------- K and V ----
      const int kv = (warp - 8) >> 2, tid = threadIdx.x - 256 - kv * kLoaders;  // K or V
      constexpr int kRowB = kInt8 ? D : 2 * D, CPR = kRowB / 16, kPer = kTile * CPR / kLoaders;
      const char* pool = static_cast<const char*>(kv ? c.v : c.k);
      // A thread's chunks lie kRows rows apart (a multiple of 8), in kQuarters of the tile's four 32-key quarters, each
      // of which lies in one page: all four where kRows <= 32, else every other one.
      constexpr int kRows = kLoaders / CPR, kQuarters = kRows <= 32 ? 4 : 2;
      const int row0 = tid / CPR, ch = tid % CPR;
      int64_t base[kQuarters];   // pool index of the quarters of the current tile, or -1
      int pid[kQuarters];        // the next tile's table entries, looked up a tile ahead
      bool whole = false;        // every key of the current tile exists
      auto quarter = [&](int j) { return kRows <= 32 ? j : 2 * j + (row0 >> 5); };
      auto chunk_quarter = [](int i) { return kRows <= 32 ? (i * kRows) >> 5 : i; };
      constexpr int kInQuarter = kRows <= 32 ? kRows : 0;  // chunk i's row within its quarter: (i kInQuarter) & 31 + row0 & 31
      auto look_up = [&](int tile) {
#pragma unroll
        for (int j = 0; j < kQuarters; ++j) {
          const int pos = tile * kTile + quarter(j) * 32;
          pid[j] = tile >= 0 && pos < p.prefix_len ? p.prefix_table[pos >> c.page_shift] : 0;
        }
      };
      look_up(t1 - 1);
      // Tile k's chunks of this thread to dst, `step` bytes apart. Tiles are taken in order.
      auto copy_tile = [&](int k, uint32_t dst, auto step) {
        const int tile = t1 - 1 - k;
        whole = tile * kTile + kTile <= p.prefix_len;
#pragma unroll
        for (int j = 0; j < kQuarters; ++j) {
          const int pos = tile * kTile + quarter(j) * 32;
          base[j] = pos < p.prefix_len ? slot_in(c, pid[j], h, pos) : -1;
          whole = whole && base[j] >= 0;
        }
        look_up(tile - 1);
        const char* src = pool + (row0 & 31) * kRowB + ch * 16;
        if (whole) {
          const char* from[kQuarters];
#pragma unroll
          for (int j = 0; j < kQuarters; ++j) from[j] = src + base[j] * kRowB;
#pragma unroll
          for (int i = 0; i < kPer; ++i)
            cp16(dst + i * step, from[chunk_quarter(i)] + ((i * kInQuarter) & 31) * kRowB, true);
        } else {
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            const int64_t b0 = base[chunk_quarter(i)];
            const bool ok = b0 >= 0 && tile * kTile + i * kRows + row0 < p.prefix_len;
            cp16(dst + i * step, src + ((b0 < 0 ? 0 : b0) + ((i * kInQuarter) & 31)) * kRowB, ok);
          }
        }
      };
      // K of tile k is unit 2 k of the ring, V unit 2 k + 1.
      const uint32_t ring = smem_u32(smem + C::OFF_RING);
      bool ok = true;
      if constexpr (kInt8) {
        const uint32_t raw = smem_u32(smem + C::OFF_RAW) + kv * (C::RAWS * C::RAWB) + tid * 16;
        constexpr std::integral_constant<uint32_t, kLoaders * 16> step{};
#pragma unroll
        for (int k = 0; k < C::RAWS - 1; ++k) {
          if (k < nt) copy_tile(k, raw + k * C::RAWB, step);
          cp_commit();
        }
        for (int k = 0; k < nt; ++k) {
          const int kn = k + C::RAWS - 1;
          if (kn < nt) copy_tile(kn, raw + (kn % C::RAWS) * C::RAWB, step);
          cp_commit();
          cp_wait<C::RAWS - 1>();
          const int u = 2 * k + kv, slot = u % C::SLOTS;
          const int before = u - C::SLOTS;  // the unit whose place this one takes
          if (before >= 0) ok = mbar_wait(empty + before % C::EMPTIES, (before / C::EMPTIES) & 1, c.status, 71);
          if (!ok) break;
          const uint32_t from = raw + (k % C::RAWS) * C::RAWB, to = ring + slot * C::TILEB;
          const uint32_t to_a = to + tile_chunk(row0, 2 * ch), to_b = to + tile_chunk(row0, 2 * ch + 1);
          // Slots past the prefix hold zero bytes, which would be code -128: they are zero in fp16 too.
          const int live = p.prefix_len - (t1 - 1 - k) * kTile - row0;
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            uint4 w = ld_shared16(from + i * kLoaders * 16);
            if (i * kRows >= live) w = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
            st_shared16(to_a + i * kRows * 128, make_uint4(code_pair<0x4140>(w.x), code_pair<0x4342>(w.x),
                                                           code_pair<0x4140>(w.y), code_pair<0x4342>(w.y)));
            st_shared16(to_b + i * kRows * 128, make_uint4(code_pair<0x4140>(w.z), code_pair<0x4342>(w.z),
                                                           code_pair<0x4140>(w.w), code_pair<0x4342>(w.w)));
          }
          fence_async_proxy();
          mbar_arrive(full + slot);
        }
      } else {
        // A tile is handed over when kAhead younger ones are on their way, or when the ring is full, so that there is
        // nothing to fetch anyhow.
        constexpr int kAhead = C::SLOTS / 2 - 1;
        int handed = 0;
        auto hand_over = [&]() {
          fence_async_proxy();
          mbar_arrive(full + (2 * handed + kv) % C::SLOTS);
          ++handed;
        };
        for (int k = 0; k < nt; ++k) {
          const int u = 2 * k + kv, slot = u % C::SLOTS;
          if (u >= C::SLOTS) {
            const int before = u - C::SLOTS;  // the unit whose place this one takes
            uint64_t* const freed = empty + before % C::EMPTIES;
            const uint32_t parity = (before / C::EMPTIES) & 1;
            while (handed < k && !__all_sync(0xffffffffu, mbar_test_wait(freed, parity))) {
              if (k - handed > 1 && kAhead > 1)
                cp_wait<1>();  // all but the youngest
              else
                cp_wait<0>();
              hand_over();
            }
            ok = mbar_wait(freed, parity, c.status, 72);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
          }
          copy_tile(k, ring + slot * C::TILEB + tile_chunk(row0, ch), std::integral_constant<uint32_t, kRows * 128>{});
          cp_commit();
          if (k - handed >= kAhead) {
            cp_wait<kAhead>();
            hand_over();
          }
        }
        cp_wait<0>();
        while (ok && handed < nt) hand_over();
      }
      cp_wait<0>();
    } else if (warp == kWarpMma) {
      // ------------------------------------------------------------------------------------------------ MMA ----
      const bool leader = elect_one();
      constexpr uint32_t HI = desc_hi(8 * 128, kSwizzle128);
      const uint32_t lq = desc_lo(smem_u32(smem + C::OFF_Q), 16);
      const uint32_t lk = desc_lo(smem_u32(smem + C::OFF_RING), 16);
      const uint32_t lv = desc_lo(smem_u32(smem + C::OFF_RING), C::BOXB);
      auto issue_s = [&](int k) {
        const int slot = (2 * k) % C::SLOTS;
        const uint32_t lb = lk + uint32_t((slot * C::TILEB) >> 4);
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = uint32_t(((kk / 4) * C::BOXB + (kk % 4) * 32) >> 4);
            mma_ss(tmem + C::COL_S + (k & 1) * kTile, desc_make(lq + off, HI), desc_make(lb + off, HI), C::IDESC_S, kk > 0);
          }
          mma_commit(s_full + (k & 1));
          mma_commit(empty + (2 * k) % C::EMPTIES);
        }
        __syncwarp();
      };
      auto issue_pv = [&](int g, int k) {
        const int slot = (2 * k + 1) % C::SLOTS;
        const uint32_t lb = lv + uint32_t((slot * C::TILEB + g * 64 * 128) >> 4);
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_ts(tmem + C::COL_O + g * D, tmem + C::COL_S + (k & 1) * kTile + g * 64 + kk * 8,
                   desc_make(lb + uint32_t((kk * 16 * 128) >> 4), HI), C::IDESC_O, (k > 0 || kk > 0) ? 1u : 0u);
          mma_commit(o_ready + g);
          if (g == 1) mma_commit(empty + (2 * k + 1) % C::EMPTIES);
        }
        __syncwarp();
      };
      bool ok = mbar_wait(q_full, 0, c.status, 73);
      for (int k = 0; k < 2 && k < nt && ok; ++k) {
        ok = mbar_wait(full + (2 * k) % C::SLOTS, ((2 * k) / C::SLOTS) & 1, c.status, 74);
        if (!ok) break;
        tc_fence_after();
        issue_s(k);
      }
      for (int k = 0; k < nt && ok; ++k) {
        for (int g = 0; g < 2 && ok; ++g) {
          ok = mbar_wait(p_full + g * 2 + (k & 1), (k >> 1) & 1, c.status, 75);
          if (ok && g == 0) ok = mbar_wait(full + (2 * k + 1) % C::SLOTS, ((2 * k + 1) / C::SLOTS) & 1, c.status, 76);
          if (!ok) break;
          tc_fence_after();
          issue_pv(g, k);
        }
        if (ok && k + 2 < nt) {
          // MMAs run in the order they are issued: S takes P's place after P V has read it. The softmax has S of tile
          // k + 1 to work on meanwhile.
          ok = mbar_wait(full + (2 * k + 4) % C::SLOTS, ((2 * k + 4) / C::SLOTS) & 1, c.status, 77);
          if (!ok) break;
          tc_fence_after();
          issue_s(k + 2);
        }
      }
      mma_commit_w(o_done);
      mbar_wait(o_done, 0, c.status, 78);  // every MMA has completed before TMEM is released
    } else if (warp < kWarpField + 2) {
      // ----------------------------------------------------------------------- the keys' field and scales ----
      // Per key, with b' = beta log2(e) and lv = log2 of V's scale (0 in fp16): the bias plus lv of a row is the smaller
      // (b' < 0: the larger) of a = b' min(SUF - psi, 0) + lv and b' (M - level) + e, e = -b' (psi - level) + lv; -inf where
      // there is no key. The level is phi of the prefix's last token (see fpa_decode_mma.cu).
      const float bias = p.beta[h] * kLog2e, level = prefix_level();
      // Two warps take alternate tiles; each also reads the phi of the tiles between its own, for the minimum.
      const int first = warp - kWarpField;
      float mid = t1 * kTile < p.prefix_len ? later_min(c, p.prefix_table, h, t1 * kTile, p.prefix_len) : kInf;
      float4 f4, ps4, ks4, vs4, skip4;  // this tile's four keys of the lane; phi of the next tile's
      int64_t at = -1;
      const float4 none = make_float4(kInf, kInf, kInf, kInf), zero4 = make_float4(0.f, 0.f, 0.f, 0.f);
      auto slot4 = [&](int pid, int tile) -> int64_t {
        // Four keys a lane lie in one page, at a multiple of four (16 bytes in the float arrays).
        const int pos = tile * kTile + lane * 4;
        return tile >= t0 && pos < p.prefix_len ? slot_in(c, pid, h, pos) : -1;
      };
      auto page_of = [&](int tile) {
        const int pos = tile * kTile + lane * 4;
        return tile >= t0 && pos < p.prefix_len ? p.prefix_table[pos >> c.page_shift] : 0;
      };
      int tile = t1 - 1 - first;
      if (first == 1) {  // the first warp's first tile comes after this one's
        const int64_t s0 = slot4(page_of(t1 - 1), t1 - 1);
        float4 x = s0 >= 0 ? *reinterpret_cast<const float4*>(c.phi + s0) : none;
        const int left = p.prefix_len - (t1 - 1) * kTile - lane * 4;
        if (left < 4) x.w = kInf;
        if (left < 3) x.z = kInf;
        if (left < 2) x.y = kInf;
        float all;
        suffix_min(fminf(fminf(x.x, x.y), fminf(x.z, x.w)), all);
        mid = fminf(mid, all);
      }
      int pid = page_of(tile), pid_skip = page_of(tile - 1);  // a pair of tiles ahead of the values
      auto load = [&]() {
        at = slot4(pid, tile);
        const int64_t next = slot4(pid_skip, tile - 1);
        f4 = at >= 0 ? *reinterpret_cast<const float4*>(c.phi + at) : none;
        skip4 = next >= 0 ? *reinterpret_cast<const float4*>(c.phi + next) : none;  // never the last, partial tile
        ps4 = at >= 0 ? *reinterpret_cast<const float4*>(c.psi + at) : zero4;
        if constexpr (kInt8) {
          ks4 = at >= 0 ? *reinterpret_cast<const float4*>(c.ks + at) : zero4;
          vs4 = at >= 0 ? *reinterpret_cast<const float4*>(c.vs + at) : zero4;
        }
        pid = page_of(tile - 2);
        pid_skip = page_of(tile - 3);
      };
      load();
      for (int k = first; k < nt; k += 2) {
        const int st = k % kParStages;
        if (k >= kParStages && !mbar_wait(par_empty + st, ((k / kParStages) - 1) & 1, c.status, 79)) break;
        const int left = at < 0 ? 0 : p.prefix_len - tile * kTile - lane * 4;  // keys of this lane that exist
        float f[4] = {f4.x, f4.y, f4.z, f4.w}, ps[4] = {ps4.x, ps4.y, ps4.z, ps4.w};
        float ks[4], vs[4];
        if constexpr (kInt8) {
          ks[0] = ks4.x, ks[1] = ks4.y, ks[2] = ks4.z, ks[3] = ks4.w;
          vs[0] = vs4.x, vs[1] = vs4.y, vs[2] = vs4.z, vs[3] = vs4.w;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j >= left) {
            f[j] = kInf;
            ps[j] = 0.f;
            if constexpr (kInt8) ks[j] = vs[j] = 0.f;
          }
        }
        float all, all_skip;
        float suf = fminf(suffix_min(fminf(fminf(f[0], f[1]), fminf(f[2], f[3])), all), mid);
        all_skip = fminf(fminf(skip4.x, skip4.y), fminf(skip4.z, skip4.w));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all_skip = fminf(all_skip, __shfl_xor_sync(0xffffffffu, all_skip, o));
        mid = fminf(mid, fminf(all, all_skip));
        float a[4], e[4], fac[4], rv[4];
#pragma unroll
        for (int j = 3; j >= 0; --j) {
          const bool ok = j < left;
          float lv = 0.f;
          if constexpr (kInt8) {
            const float v = fmax_nan(vs[j], 0x1p-90f);
            fac[j] = ks[j] * p.scale2;
            lv = lg2(v);
            rv[j] = ok ? rcp_approx_f(v) : 0.f;
          }
          a[j] = ok ? fmaf(bias, fminf(suf - ps[j], 0.f), lv) : -kInf;
          e[j] = ok ? fmaf(-bias, ps[j] - level, lv) : -kInf;
          suf = fminf(suf, f[j]);
        }
        float* out = reinterpret_cast<float*>(smem + C::OFF_PAR + st * C::PARB);
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          const int pair = lane * 2 + j / 2;
          reinterpret_cast<float4*>(out)[pair] = make_float4(e[j], e[j + 1], a[j], a[j + 1]);
          if constexpr (kInt8) {
            reinterpret_cast<float2*>(out + kTile * 2)[pair] = make_float2(fac[j], fac[j + 1]);
            reinterpret_cast<float2*>(out + kTile * 3)[pair] = make_float2(rv[j], rv[j + 1]);
          }
        }
        mbar_arrive(par_full + st);
        tile -= 2;
        if (k + 2 < nt) load();
      }
    }
  } else {
    // ------------------------------------------------------------------------------------------- softmax ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 136;" ::: "memory");
    const int g = warp >> 2;
    {
      // Q into shared memory, each copy of the rows; rows that are not there are zero.
      const __half* q = static_cast<const __half*>(p.q) + h * p.sq.h;
      const uint32_t sq = smem_u32(smem + C::OFF_Q);
      constexpr int kAhead = D / 16;  // all of this thread's
      for (int e0 = threadIdx.x; e0 < kTile * (D / 8); e0 += kAhead * 256) {
        uint32_t x[kAhead][4];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
          const int e = e0 + a * 256, r = e / (D / 8), ch = e % (D / 8), lr = r % RP;
          const int i = r0 + min(lr, rows - 1), b = i / p.n;
          const __half* row = q + b * p.sq.b + (i - b * p.n) * p.sq.t + ch * 8 * p.sq.d;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (p.q_pairs) {
              x[a][j] = *reinterpret_cast<const uint32_t*>(row + 2 * j);
            } else {
              const __half2 v = __halves2half2(row[2 * j * p.sq.d], row[(2 * j + 1) * p.sq.d]);
              x[a][j] = *reinterpret_cast<const uint32_t*>(&v);
            }
            if (lr >= rows) x[a][j] = 0;
          }
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
          const int e = e0 + a * 256;
          st_shared16(sq + tile_chunk(e / (D / 8), e % (D / 8)), make_uint4(x[a][0], x[a][1], x[a][2], x[a][3]));
        }
      }
      fence_async_proxy();
      mbar_arrive(q_full);
    }
    const int lrow = (warp & 3) * 32 + lane;  // TMEM lane
    const int copy = lrow / RP, lr = lrow % RP;
    constexpr int CW = kTile / 2 / REP;       // this copy's keys of the group's half tile
    const int c0 = copy * CW;                 // within the half tile
    const bool busy = lr - lane < rows;       // some row of this warp exists (RP is a multiple of 32)
    const uint32_t tl = tmem + (uint32_t((warp & 3) * 32) << 16);
    const uint32_t tO = tl + C::COL_O + g * D;
    const float level = prefix_level();
    pdl_wait();  // row_min
    pdl_launch_dependents();
    const float low = lr < rows ? p.row_min[int64_t(h) * R + r0 + lr] : kInf;
    const float bias = p.beta[h] * kLog2e;
    const float2 low2 = make_float2(bias * (low - level), bias * (low - level)), sc2 = make_float2(p.scale2, p.scale2);
    float m = -kInf;
    float2 l2 = make_float2(0.f, 0.f);
    bool ok = true;
    auto walk = [&](auto negative) {
      auto nearer = [](float x, float y) { return decltype(negative)::value ? fmaxf(x, y) : fminf(x, y); };
      for (int k = 0; k < nt; ++k) {
        const int st = k % kParStages;
        ok = mbar_wait(par_full + st, (k / kParStages) & 1, c.status, 80);
        if (ok) ok = mbar_wait(s_full + (k & 1), (k >> 1) & 1, c.status, 81);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        if (busy) {
          const uint32_t tS = tl + C::COL_S + (k & 1) * kTile + g * 64;
          const float* par = reinterpret_cast<const float*>(smem + C::OFF_PAR + st * C::PARB);
          const int pair0 = (g * 64 + c0) >> 1;
          float s[CW];
          if constexpr (CW >= 32) {
#pragma unroll
            for (int i = 0; i < CW; i += 32) tmem_ld32(tS + c0 + i, s + i);
          } else {
            tmem_ld16(tS + c0, s);
          }
          tmem_ld_wait();
          float m4[4] = {-kInf, -kInf, -kInf, -kInf};
#pragma unroll
          for (int i = 0; i < CW; i += 2) {
            const int pair = pair0 + (i >> 1);
            const float4 x = reinterpret_cast<const float4*>(par)[pair];
            const float2 t = __fadd2_rn(low2, make_float2(x.x, x.y));
            const float2 b = make_float2(nearer(x.z, t.x), nearer(x.w, t.y));
            const float2 f2 = kInt8 ? reinterpret_cast<const float2*>(par + kTile * 2)[pair] : sc2;
            const float2 z = __ffma2_rn(make_float2(s[i], s[i + 1]), f2, b);
            s[i] = z.x;
            s[i + 1] = z.y;
            m4[(i >> 1) & 3] = fmax3f(m4[(i >> 1) & 3], z.x, z.y);
          }
          const float mt = fmaxf(fmax3f(m4[0], m4[1], m4[2]), m4[3]);
          // A new maximum only when it grows by more than 8 (log2 units).
          const bool grow = mt > m + 8.f;
          if (__any_sync(0xffffffffu, grow)) {
            const float mn = grow ? mt : m, alpha = grow ? state_weight(m, mn) : 1.f;
            m = mn;
            l2.x *= alpha;
            l2.y *= alpha;
            if (k > 0) {
              ok = mbar_wait(o_ready + g, (k - 1) & 1, c.status, 84);  // O holds the tiles before this one
              ok = __all_sync(0xffffffffu, ok);
              if (!ok) break;
              tc_fence_after();
#pragma unroll
              for (int cc = 0; cc < D; cc += 16) {
                float o[16];
                tmem_ld16(tO + cc, o);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] *= alpha;
                tmem_st16(tO + cc, reinterpret_cast<const uint32_t*>(o));
              }
            }
          }
          const float ref = m == -kInf ? 0.f : -m;
          const float2 ref2 = make_float2(ref, ref);
          uint32_t pk[CW / 2];
#pragma unroll
          for (int e = 0; e < CW; e += 2) {
            const float2 x = __fadd2_rn(make_float2(s[e], s[e + 1]), ref2);
            const float2 pp = make_float2(ex2(x.x), ex2(x.y));
            if constexpr (kInt8)
              l2 = __ffma2_rn(pp, reinterpret_cast<const float2*>(par + kTile * 3)[pair0 + (e >> 1)], l2);
            else
              l2 = __fadd2_rn(l2, pp);
            pk[e / 2] = pack2(pp.x, pp.y);
          }
          if constexpr (CW == 64) {
            tmem_st32(tS, pk);
          } else {
            // The keys of the other copies count nothing here.
            const uint32_t zero[16] = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < REP; ++j) {
              if constexpr (CW == 32) {
                if (j != copy) tmem_st16(tS + j * 16, zero);
              } else {
                if (j != copy) tmem_st8(tS + j * 8, zero);
              }
            }
            if constexpr (CW == 32)
              tmem_st16(tS + c0 / 2, pk);
            else
              tmem_st8(tS + c0 / 2, pk);
          }
          tmem_st_wait();
        }
        tc_fence_before();
        mbar_arrive(par_empty + st);
        mbar_arrive(p_full + g * 2 + (k & 1));
      }
    };
    if (bias < 0.f)
      walk(std::true_type{});
    else
      walk(std::false_type{});
    // The states of both groups and all copies, in the ring's place once every MMA has completed.
    mbar_wait(o_done, 0, c.status, 82);
    tc_fence_after();
    float* sO = reinterpret_cast<float*>(smem + C::OFF_RING);  // [state][D + 4]
    float* ml = reinterpret_cast<float*>(smem + C::OFF_ML);
    const int state = g * kTile + lrow;  // = (g REP + copy) RP + lr
    ml[state] = m;
    ml[256 + state] = l2.x + l2.y;
    asm volatile("bar.sync 1, 256;" ::: "memory");
    float M = -kInf, l = 0.f;
#pragma unroll
    for (int s = 0; s < 2 * REP; ++s) M = fmaxf(M, ml[s * RP + lr]);
#pragma unroll
    for (int s = 0; s < 2 * REP; ++s) l += state_weight(ml[s * RP + lr], M) * ml[256 + s * RP + lr];
    const float w = state_weight(m, M);
    if (busy) {
#pragma unroll
      for (int cc = 0; cc < D; cc += 32) {
        float o[32];
        tmem_ld32(tO + cc, o);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; e += 4)
          *reinterpret_cast<float4*>(sO + state * (D + 4) + cc + e) =
              make_float4(o[e] * w, o[e + 1] * w, o[e + 2] * w, o[e + 3] * w);
      }
    }
    tc_fence_before();
    asm volatile("bar.sync 1, 256;" ::: "memory");
    const int64_t out = (int64_t(h) * R + r0) * p.chunks + blockIdx.x;  // of row 0; rows are p.chunks apart
    if (g == 0 && copy == 0 && lr < rows)
      *reinterpret_cast<float2*>(p.part_ml + (out + int64_t(lr) * p.chunks) * 2) = make_float2(M, l);
#pragma unroll 2
    for (int e = threadIdx.x; e < rows * (D / 4); e += 256) {
      const int r = e / (D / 4), d = e % (D / 4) * 4;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int s = 0; s < 2 * REP; ++s) {
        const float4 x = *reinterpret_cast<const float4*>(sO + (s * RP + r) * (D + 4) + d);
        o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
      }
      *reinterpret_cast<float4*>(p.part_o + (out + int64_t(r) * p.chunks) * D + d) = o;
    }
  }
  __syncthreads();
  if (warp == kWarpMma) tmem_dealloc(tmem, 512);
}

// How often the rows stand in the 128 lanes: as often as they fit. Whole calls behind 8192 tokens, 12 heads, us with 4 / 2 /
// 1 copies: int8 D = 64, 32 rows 18.6 / 19.3 / 21.6, 64 rows - / 21.1 / 22.9; fp16 D = 128, 32 rows 20.9 / 20.7 / 22.2.
template <int D, bool kInt8>
cudaError_t launch_rep(const DecodeParams& p, cudaStream_t s) {
  const int R = p.B * p.n;
  auto kernel = R <= 32 ? prefix_tc_kernel<D, kInt8, 4> : R <= 64 ? prefix_tc_kernel<D, kInt8, 2> : prefix_tc_kernel<D, kInt8, 1>;
  const cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), PrefixCfg<D, kInt8>::SMEM);
  if (e != cudaSuccess) return e;
  return launch_pdl(kernel, dim3(p.chunks, prefix_tc_row_tiles(R), p.c.H), dim3(kPrefixThreads), PrefixCfg<D, kInt8>::SMEM, s, p);
}

}  // namespace

int prefix_tc_row_tiles(int64_t rows) { return int((rows + kTile - 1) / kTile); }

cudaError_t launch_prefix_tc(const DecodeParams& p, bool int8, cudaStream_t s) {
  if (p.c.D == 64) return int8 ? launch_rep<64, true>(p, s) : launch_rep<64, false>(p, s);
  return int8 ? launch_rep<128, true>(p, s) : launch_rep<128, false>(p, s);
}

}  // namespace fpa
