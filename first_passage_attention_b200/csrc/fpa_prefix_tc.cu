// Attention of a batch's rows over a shared prefix on the tensor cores (tcgen05), fp16 queries, D = 64 or 128.
//
// The rows (b, i) of all sequences, up to 128 at a time, meet every key of the prefix once: S = Q K^T and O += P V with
// 128-key tiles, one CTA on an SM for a part of the prefix, which it walks from the latest tile to the earliest (the
// mathematics is in fpa_decode.cuh). With R rows there are R flops a byte in fp16 and 2 R in int8, so up to about 128
// rows the prefix's bytes bound it and beyond that the softmax's instructions do, about 7 for a (row, key) pair. Against
// that, two softmax groups of 128 threads (a thread is a row is a TMEM lane) take alternate tiles, each with its own S,
// running maximum, sum and O in TMEM, and their states join at the end. Where the rows fill half or a quarter of the
// 128 lanes, they stand there twice or four times, and each copy takes its half or quarter of the tile's keys (its P
// is zero for the others), so that no warp idles; the copies' states join like the groups'.
//
// Warps 0-3 and 4-7: softmax groups. Warps 8-11: K and V into the ring of 128-byte-swizzled tiles; fp16 by cp.async
// directly, int8 by cp.async into a raw ring that each thread reads back itself, converts to fp16 (exact) and stores.
// Plain loads rather than TMA, because the last page's slots past the prefix must come out as zeros whatever they
// hold, and because codes have to be converted on the way. Warp 12: the MMAs. Warp 13: per tile the keys' a, psi and
// scales, with the running minimum of phi. Every wait is bounded.
#include <cuda_fp16.h>

#include "fpa_decode.cuh"
#include "fpa_sm100.cuh"

namespace fpa {
namespace {

using namespace sm100;

constexpr int kTile = 128;
constexpr int kPrefixThreads = 512;
constexpr int kLoaders = 128;
constexpr int kParStages = 4;

template <int D, bool kInt8>
struct PrefixCfg {
  static constexpr int BOXB = kTile * 128;                // a tile's 64 columns
  static constexpr int TILEB = D / 64 * BOXB;             // K or V of a tile in fp16
  static constexpr int SLOTS = kInt8 ? (D == 64 ? 6 : 4) : (D == 64 ? 8 : 5);
  static constexpr int RAWB = kInt8 ? kTile * D : 0;      // K or V of a tile in codes
  static constexpr int RAWS = kInt8 ? (D == 64 ? 4 : 3) : 0;
  static constexpr int PARF = kInt8 ? 10 : 6;             // floats of a pair of keys
  static constexpr int PARB = kTile / 2 * PARF * 4;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_RING = OFF_Q + TILEB;
  static constexpr int OFF_RAW = OFF_RING + SLOTS * TILEB;
  static constexpr int OFF_PAR = OFF_RAW + RAWS * RAWB;
  static constexpr int OFF_ML = OFF_PAR + kParStages * PARB;  // [2][256] maxima and sums of the states
  static constexpr int OFF_BAR = OFF_ML + 2 * 256 * 4;
  static constexpr int NBAR = 2 * SLOTS + 2 * kParStages + 2 + 2 + 2;
  static constexpr int SMEM = OFF_BAR + NBAR * 8 + 16 + 1024;
  static constexpr int COL_S = 0, COL_O = 2 * kTile;      // of group g: + 128 g, + D g; P over the first half of S
  static constexpr uint32_t IDESC_S = idesc_f16(kTile, kTile, 0);
  static constexpr uint32_t IDESC_O = idesc_f16(kTile, D, 1);
  static_assert(SMEM <= 227 * 1024, "shared memory");
  static_assert(256 * (D + 1) * 4 <= SLOTS * TILEB + RAWS * RAWB, "the states join in the ring's place");
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
  uint64_t* par_full = empty + C::SLOTS;
  uint64_t* par_empty = par_full + kParStages;
  uint64_t* s_full = par_empty + kParStages;
  uint64_t* p_full = s_full + 2;
  uint64_t* q_full = p_full + 2;
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

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::SLOTS; ++i) {
      mbar_init(full + i, kLoaders);
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < kParStages; ++i) {
      mbar_init(par_full + i, 32);
      mbar_init(par_empty + i, 128);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(s_full + g, 1);
      mbar_init(p_full + g, 128);
    }
    mbar_init(q_full, 256);
    mbar_init(o_done, 1);
    fence_mbar_init();
  }
  if (warp == 12) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // The launch before this one (row_min) has waited for everything earlier, so the cache and the queries can be read
  // at once; only the softmax warps wait, for the rows' minima.

  // Registers: 128 a thread at launch; 184 for the softmax warpgroups, 72 for the others.
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;" ::: "memory");
    if (warp < 12) {
      // ------------------------------------------------------------------------------------------- K and V ----
      const int tid = threadIdx.x - 256;
      constexpr int kRowB = kInt8 ? D : 2 * D, CPR = kRowB / 16, kPer = kTile * CPR / kLoaders;
      const int units = 2 * nt;  // K then V of each tile
      int64_t base[4];           // pool index of each 32-key quarter of the current tile, or -1
      // Unit u's chunks of this thread: chunk i is row (i 128 + tid) / CPR, so 128 / CPR rows apart.
      auto copy_unit = [&](int u, uint32_t dst_base) {
        const int tile = t1 - 1 - (u >> 1);
        if ((u & 1) == 0) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int pos = tile * kTile + q * 32;
            base[q] = pos < p.prefix_len ? slot_of(c, p.prefix_table, h, pos) : -1;
          }
        }
        const char* src = static_cast<const char*>((u & 1) ? c.v : c.k);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int idx = i * kLoaders + tid, row = idx / CPR, ch = idx % CPR;
          const int64_t b0 = base[(i * (kLoaders / CPR)) >> 5];  // rows of one i stay within 32 keys
          const bool ok = b0 >= 0 && tile * kTile + row < p.prefix_len;
          const char* from = src + ((b0 < 0 ? 0 : b0) + (row & 31)) * kRowB + ch * 16;
          cp16(dst_base + (kInt8 ? uint32_t(idx * 16) : tile_chunk(row, ch)), from, ok);
        }
      };
      const uint32_t ring = smem_u32(smem + C::OFF_RING);
      bool ok = true;
      if constexpr (kInt8) {
        const uint32_t raw = smem_u32(smem + C::OFF_RAW);
#pragma unroll
        for (int u = 0; u < C::RAWS - 1; ++u) {
          if (u < units) copy_unit(u, raw + u * C::RAWB);
          cp_commit();
        }
        for (int u = 0; u < units; ++u) {
          const int un = u + C::RAWS - 1;
          if (un < units) copy_unit(un, raw + (un % C::RAWS) * C::RAWB);
          cp_commit();
          cp_wait<C::RAWS - 1>();
          const int slot = u % C::SLOTS;
          if (u >= C::SLOTS) ok = mbar_wait(empty + slot, ((u / C::SLOTS) - 1) & 1, c.status, 71);
          if (!ok) break;
          const uint32_t from = raw + (u % C::RAWS) * C::RAWB, to = ring + slot * C::TILEB;
          // Slots past the prefix hold zero bytes, which would be code -128: they are zero in fp16 too.
          const int tile = t1 - 1 - (u >> 1);
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            const int idx = i * kLoaders + tid, row = idx / CPR, ch = idx % CPR;
            const uint4 w = ld_shared16(from + idx * 16);
            const bool live = tile * kTile + row < p.prefix_len;
            uint4 a = make_uint4(code_pair<0x4140>(w.x), code_pair<0x4342>(w.x), code_pair<0x4140>(w.y), code_pair<0x4342>(w.y));
            uint4 b = make_uint4(code_pair<0x4140>(w.z), code_pair<0x4342>(w.z), code_pair<0x4140>(w.w), code_pair<0x4342>(w.w));
            if (!live) a = b = make_uint4(0, 0, 0, 0);
            st_shared16(to + tile_chunk(row, 2 * ch), a);
            st_shared16(to + tile_chunk(row, 2 * ch + 1), b);
          }
          fence_async_proxy();
          mbar_arrive(full + slot);
        }
      } else {
        // Up to kAhead units in flight beyond the one that is handed over.
        constexpr int kAhead = C::SLOTS - 2;
        int sent = 0;
        for (int u = 0; u < units + kAhead && ok; ++u) {
          if (u < units) {
            const int slot = u % C::SLOTS;
            if (u >= C::SLOTS) ok = mbar_wait(empty + slot, ((u / C::SLOTS) - 1) & 1, c.status, 72);
            if (!ok) break;
            copy_unit(u, ring + slot * C::TILEB);
          }
          cp_commit();
          if (u >= kAhead) {
            cp_wait<kAhead>();
            fence_async_proxy();
            mbar_arrive(full + sent % C::SLOTS);
            ++sent;
          }
        }
      }
      cp_wait<0>();
    } else if (warp == 12) {
      // ------------------------------------------------------------------------------------------------ MMA ----
      const bool leader = elect_one();
      constexpr uint32_t HI = desc_hi(8 * 128, kSwizzle128);
      const uint32_t lq = desc_lo(smem_u32(smem + C::OFF_Q), 16);
      const uint32_t lk = desc_lo(smem_u32(smem + C::OFF_RING), 16);
      const uint32_t lv = desc_lo(smem_u32(smem + C::OFF_RING), C::BOXB);
      auto issue_s = [&](int k) {
        const int slot = (2 * k) % C::SLOTS;
        const uint32_t lb = lk + uint32_t(slot * (C::TILEB >> 4));
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = uint32_t(((kk / 4) * C::BOXB + (kk % 4) * 32) >> 4);
            mma_ss(tmem + C::COL_S + (k & 1) * kTile, desc_make(lq + off, HI), desc_make(lb + off, HI), C::IDESC_S, kk > 0);
          }
          mma_commit(empty + slot);
          mma_commit(s_full + (k & 1));
        }
        __syncwarp();
      };
      auto issue_pv = [&](int k) {
        const int slot = (2 * k + 1) % C::SLOTS;
        const uint32_t lb = lv + uint32_t(slot * (C::TILEB >> 4));
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < kTile / 16; ++kk)
            mma_ts(tmem + C::COL_O + (k & 1) * D, tmem + C::COL_S + (k & 1) * kTile + kk * 8,
                   desc_make(lb + uint32_t((kk * 16 * 128) >> 4), HI), C::IDESC_O, (k > 1 || kk > 0) ? 1u : 0u);
          mma_commit(empty + slot);
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
        ok = mbar_wait(p_full + (k & 1), (k >> 1) & 1, c.status, 75);
        if (ok) ok = mbar_wait(full + (2 * k + 1) % C::SLOTS, ((2 * k + 1) / C::SLOTS) & 1, c.status, 76);
        if (!ok) break;
        tc_fence_after();
        issue_pv(k);
        if (k + 2 < nt) {
          // The MMAs run in the order they are issued: S takes P's place after P V has read it.
          ok = mbar_wait(full + (2 * k + 4) % C::SLOTS, ((2 * k + 4) / C::SLOTS) & 1, c.status, 77);
          if (!ok) break;
          tc_fence_after();
          issue_s(k + 2);
        }
      }
      mma_commit_w(o_done);
      mbar_wait(o_done, 0, c.status, 78);  // every MMA has completed before TMEM is released
    } else if (warp == 13) {
      // ----------------------------------------------------------------------- the keys' field and scales ----
      float mid = t1 * kTile < p.prefix_len ? later_min(c, p.prefix_table, h, t1 * kTile, p.prefix_len) : kInf;
      float f[4], ps[4], ks[4], vs[4];
      int64_t at = -1;
      auto load = [&](int tile) {
        // Four keys a lane, which lie in one page.
        const int pos = tile * kTile + lane * 4;
        at = pos < p.prefix_len ? slot_of(c, p.prefix_table, h, pos) : -1;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool ok = at >= 0 && pos + j < p.prefix_len;
          f[j] = ok ? c.phi[at + j] : kInf;
          ps[j] = ok ? c.psi[at + j] : 0.f;
          if constexpr (kInt8) {
            ks[j] = ok ? c.ks[at + j] : 0.f;
            vs[j] = ok ? c.vs[at + j] : 0.f;
          }
        }
      };
      load(t1 - 1);
      for (int k = 0; k < nt; ++k) {
        const int st = k % kParStages, tile = t1 - 1 - k;
        if (k >= kParStages && !mbar_wait(par_empty + st, ((k / kParStages) - 1) & 1, c.status, 79)) break;
        float all;
        float suf = fminf(suffix_min(fminf(fminf(f[0], f[1]), fminf(f[2], f[3])), all), mid);
        mid = fminf(mid, all);
        float a[4], fac[4], lv[4], rv[4];
#pragma unroll
        for (int j = 3; j >= 0; --j) {
          const bool ok = at >= 0 && tile * kTile + lane * 4 + j < p.prefix_len;
          a[j] = ok ? fminf(suf - ps[j], 0.f) : 0.f;
          suf = fminf(suf, f[j]);
          lv[j] = ok ? 0.f : -kInf;
          if constexpr (kInt8) {
            const float v = fmaxf(vs[j], 0x1p-90f);
            fac[j] = ks[j] * p.scale2;
            if (ok) lv[j] = lg2(v);
            rv[j] = ok ? rcp_approx_f(v) : 0.f;
          }
        }
        float* out = reinterpret_cast<float*>(smem + C::OFF_PAR + st * C::PARB);
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          const int pair = lane * 2 + j / 2;
          reinterpret_cast<float4*>(out)[pair] = make_float4(-ps[j], -ps[j + 1], a[j], a[j + 1]);
          if constexpr (kInt8) {
            reinterpret_cast<float4*>(out + kTile * 2)[pair] = make_float4(fac[j], fac[j + 1], lv[j], lv[j + 1]);
            reinterpret_cast<float2*>(out + kTile * 4)[pair] = make_float2(rv[j], rv[j + 1]);
          } else {
            reinterpret_cast<float2*>(out + kTile * 2)[pair] = make_float2(lv[j], lv[j + 1]);
          }
        }
        mbar_arrive(par_full + st);
        if (k + 1 < nt) load(tile - 1);
      }
    }
  } else {
    // ------------------------------------------------------------------------------------------- softmax ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 184;" ::: "memory");
    const int g = warp >> 2;
    {
      // Q into shared memory, each copy of the rows; rows that are not there are zero.
      const __half* q = static_cast<const __half*>(p.q) + h * p.sq.h;
      const uint32_t sq = smem_u32(smem + C::OFF_Q);
      for (int e = threadIdx.x; e < kTile * (D / 8); e += 256) {
        const int r = e / (D / 8), ch = e % (D / 8), lr = r % RP;
        uint4 w = make_uint4(0, 0, 0, 0);
        if (lr < rows) {
          const int i = r0 + lr, b = i / p.n;
          const __half* row = q + b * p.sq.b + (i - b * p.n) * p.sq.t + ch * 8 * p.sq.d;
          uint32_t x[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (p.q_pairs) {
              x[j] = *reinterpret_cast<const uint32_t*>(row + 2 * j);
            } else {
              const __half2 v = __halves2half2(row[2 * j * p.sq.d], row[(2 * j + 1) * p.sq.d]);
              x[j] = *reinterpret_cast<const uint32_t*>(&v);
            }
          }
          w = make_uint4(x[0], x[1], x[2], x[3]);
        }
        st_shared16(sq + tile_chunk(r, ch), w);
      }
      fence_async_proxy();
      mbar_arrive(q_full);
    }
    const int lrow = (warp & 3) * 32 + lane;  // TMEM lane
    const int copy = lrow / RP, lr = lrow % RP;
    constexpr int CW = kTile / REP;           // this copy's keys of a tile
    const int c0 = copy * CW;
    const bool busy = lr - lane < rows;       // some row of this warp exists (RP is a multiple of 32)
    const uint32_t tl = tmem + (uint32_t((warp & 3) * 32) << 16);
    const uint32_t tS = tl + C::COL_S + g * kTile, tO = tl + C::COL_O + g * D;
    pdl_wait();  // row_min
    pdl_launch_dependents();
    const float low = lr < rows ? p.row_min[int64_t(h) * R + r0 + lr] : kInf;
    const float bias = p.beta[h] * kLog2e;
    const float2 low2 = make_float2(low, low), bias2 = make_float2(bias, bias), sc2 = make_float2(p.scale2, p.scale2);
    float m = -kInf;
    float2 l2 = make_float2(0.f, 0.f);
    bool ok = true;
    for (int k = g; k < nt && ok; k += 2) {
      const int st = k % kParStages;
      ok = mbar_wait(par_full + st, (k / kParStages) & 1, c.status, 80);
      if (ok) ok = mbar_wait(s_full + g, (k >> 1) & 1, c.status, 81);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      if (busy) {
        const float* par = reinterpret_cast<const float*>(smem + C::OFF_PAR + st * C::PARB);
        float s[CW];
#pragma unroll
        for (int i = 0; i < CW; i += 32) tmem_ld32(tS + c0 + i, s + i);
        tmem_ld_wait();
        float m4[4] = {-kInf, -kInf, -kInf, -kInf};
#pragma unroll
        for (int i = 0; i < CW; i += 2) {
          const int pair = (c0 + i) >> 1;
          const float4 x = reinterpret_cast<const float4*>(par)[pair];
          const float2 t = __fadd2_rn(low2, make_float2(x.x, x.y));
          const float2 b = make_float2(fminf(x.z, t.x), fminf(x.w, t.y));
          float2 z;
          if constexpr (kInt8) {
            const float4 y = reinterpret_cast<const float4*>(par + kTile * 2)[pair];
            z = __ffma2_rn(make_float2(s[i], s[i + 1]), make_float2(y.x, y.y), __ffma2_rn(bias2, b, make_float2(y.z, y.w)));
          } else {
            const float2 lv = reinterpret_cast<const float2*>(par + kTile * 2)[pair];
            z = __ffma2_rn(make_float2(s[i], s[i + 1]), sc2, __ffma2_rn(bias2, b, lv));
          }
          s[i] = z.x;
          s[i + 1] = z.y;
          m4[(i >> 1) & 3] = fmax3f(m4[(i >> 1) & 3], z.x, z.y);
        }
        const float mt = fmaxf(fmax3f(m4[0], m4[1], m4[2]), m4[3]);
        // A new maximum only when it grows by more than 8 (log2 units); O holds the sums up to this group's last tile.
        const bool grow = mt > m + 8.f;
        if (__any_sync(0xffffffffu, grow)) {
          const float mn = grow ? mt : m, alpha = grow ? state_weight(m, mn) : 1.f;
          m = mn;
          l2.x *= alpha;
          l2.y *= alpha;
          if (k > 1) {
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
#pragma unroll
        for (int cc = 0; cc < CW; cc += 32) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 x = __fadd2_rn(make_float2(s[cc + e], s[cc + e + 1]), ref2);
            const float2 pp = make_float2(ex2(x.x), ex2(x.y));
            if constexpr (kInt8)
              l2 = __ffma2_rn(pp, reinterpret_cast<const float2*>(par + kTile * 4)[(c0 + cc + e) >> 1], l2);
            else
              l2 = __fadd2_rn(l2, pp);
            pk[e / 2] = pack2(pp.x, pp.y);
          }
          tmem_st16(tS + (c0 + cc) / 2, pk);
        }
        if constexpr (REP > 1) {
          // The other copies' keys count nothing here.
          const uint32_t zero[16] = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
          for (int cc = 0; cc < kTile; cc += 32)
            if (cc / CW != copy) tmem_st16(tS + cc / 2, zero);
        }
        tmem_st_wait();
      }
      tc_fence_before();
      mbar_arrive(par_empty + st);
      mbar_arrive(p_full + g);
    }
    // The states of both groups and all copies, in the ring's place once every MMA has completed.
    if (ok) ok = mbar_wait(o_done, 0, c.status, 82);
    ok = __all_sync(0xffffffffu, ok);
    tc_fence_after();
    float* sO = reinterpret_cast<float*>(smem + C::OFF_RING);
    float* ml = reinterpret_cast<float*>(smem + C::OFF_ML);
    const int state = (g * REP + copy) * RP + lr;  // = g 128 + lrow
    const bool any = ok && g < nt;                 // this group has had a tile
    ml[state] = any ? m : -kInf;
    ml[256 + state] = any ? l2.x + l2.y : 0.f;
#pragma unroll 1
    for (int cc = 0; cc < D; cc += 32) {
      float o[32];
      if (any) {
        tmem_ld32(tO + cc, o);
        tmem_ld_wait();
      }
#pragma unroll
      for (int e = 0; e < 32; ++e) sO[state * (D + 1) + cc + e] = any ? o[e] : 0.f;
    }
    tc_fence_before();
    asm volatile("bar.sync 1, 256;" ::: "memory");
    for (int e = threadIdx.x; e < rows * D; e += 256) {
      const int r = e / D, d = e - r * D;
      float M = -kInf, l = 0.f, o = 0.f;
#pragma unroll
      for (int s = 0; s < 2 * REP; ++s) M = fmaxf(M, ml[s * RP + r]);
#pragma unroll
      for (int s = 0; s < 2 * REP; ++s) {
        const float w = state_weight(ml[s * RP + r], M);
        l += w * ml[256 + s * RP + r];
        o += w * sO[(s * RP + r) * (D + 1) + d];
      }
      const int64_t at = (int64_t(h) * R + r0 + r) * p.chunks + blockIdx.x;
      p.part_o[at * D + d] = o;
      if (d == 0) {
        p.part_ml[at * 2] = M;
        p.part_ml[at * 2 + 1] = l;
      }
    }
  }
  __syncthreads();
  if (warp == 12) tmem_dealloc(tmem, 512);
}

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
