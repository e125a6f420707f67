// Decode attention for fp16 queries over an fp16 or int8 cache, on the tensor cores (mma.sync m16n8k16).
//
// The products are S^T = K Q^T (16 keys x 16 d times 16 d x 8 rows) and O^T = V^T P^T (16 d x 16 keys times 16 keys x 8
// rows): the keys, which are many, fill the instruction's 16 rows, and the query rows, which are few, its 8 columns.
// With at most 16 rows there are at most 32 flops a byte, a tenth of what would make the tensor cores' rate matter,
// so the loads decide: the fragments come straight from global memory into registers. Lane (g, t) = (lane / 4, lane
// % 4) needs, of K, some four elements of key g for each 16-d step: which ones is free as long as Q agrees, so it
// takes consecutive ones (16 bytes at a time, a full 64-byte run per key and four lanes). Of V it needs, for each 16-d
// tile, two columns of the keys 2t, 2t + 1, 2t + 8, 2t + 9: it takes D / 8 consecutive columns. P passes from the
// accumulators' layout to the operand's with movmatrix. No shared memory, no barrier, on the way of K and V.
//
// int8: codes become fp16 exactly (0x6400 | (code + 128) is 1152 + code); K's scale multiplies the finished product,
// and V's goes into the exponent. With lv = log2 vs, P' = 2^(z + lv - m) <= 2^8 for m = max(z + lv) as of its last
// update, l = sum P' / vs and o = sum P' code / l: the factors fp16 holds are scaled to the largest contribution
// whatever the scales are, and the cost is that of the plain softmax. P' is rounded to fp16 (2^-11 relative, as the
// training kernels round P); sums and states stay in fp32. The maximum is updated only when it grows by more than 8
// (in log2 units), decided by the whole warp.
#include <cuda_fp16.h>

#include "fpa_decode.cuh"

namespace fpa {
namespace {

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Two halves from bytes (lo, hi) of codes with 128 added: `sel` picks byte 0 / 1 or 2 / 3 of x.
template <uint32_t kSel>
__device__ __forceinline__ uint32_t codes_to_half2(uint32_t x) {
  const uint32_t y = __byte_perm(x, 0x64646464u, kSel);
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&y), __floats2half2_rn(1152.f, 1152.f));
  return *reinterpret_cast<const uint32_t*>(&h);
}

// kBytes (2, 4, 8 or a multiple of 16) from global memory that this kernel only reads once.
template <int kBytes, int kStride>
__device__ __forceinline__ void load_words(const char* p, uint32_t* w) {
  if constexpr (kBytes == 2) {
    unsigned short x;
    asm volatile("ld.global.nc.L1::no_allocate.u16 %0, [%1];" : "=h"(x) : "l"(p));
    w[0] = x;
  } else if constexpr (kBytes == 4) {
    asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(w[0]) : "l"(p));
  } else if constexpr (kBytes == 8) {
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
  } else {
#pragma unroll
    for (int j = 0; j < kBytes / 16; ++j)
      asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w[4 * j]), "=r"(w[4 * j + 1]), "=r"(w[4 * j + 2]), "=r"(w[4 * j + 3])
                   : "l"(p + j * kStride));
  }
}

template <int D_, bool kInt8, int NT>
struct MmaCore {
  static constexpr int D = D_, W = 4, NQ = 8 * NT;
  static constexpr int ES = kInt8 ? 1 : 2;             // bytes of a stored element
  static constexpr int KB = D / 4 * ES, KV = KB < 16 ? KB : 16;   // bytes of a key for a lane; of one load
  static constexpr int VB = D / 8 * ES, VV = VB < 16 ? VB : 16;
  static constexpr int KW = KB / 4, VW = VB < 4 ? 1 : VB / 4;     // 32-bit words
  static constexpr int KE = KV / ES, VE = VV / ES;                // elements of one load
  static constexpr int KS = D / 16, MT = D / 16;
  static constexpr int SUB = D * ES <= 128 ? 2 : 1;    // 16-key blocks loaded and worked on at a time
  static constexpr int STEPS = 2 / SUB;
  // Registers of the fragments and accumulators decide how many CTAs an SM can hold.
  static constexpr int kRegs = SUB * (2 * KW + 4 * VW) + NT * (2 * KS + 4 * MT);
  static constexpr int kMinBlocks = kRegs <= 72 ? 4 : kRegs <= 112 ? 3 : 2;
  static constexpr int kScratchFloats = W * 32 * 5;
  using Out = __half;

  uint32_t kf[SUB][2][KW], vf[SUB][4][VW], qf[NT][KS][2];
  float o[MT][NT][4], m[NT][2], l[NT][2], low[NT][2];
  float4* par;  // per key of the tile: a, psi, factor of the product, log2 of V's scale (-inf: no such key)
  float* rvs;   // 1 / V's scale
  int g, t;

  __device__ __forceinline__ MmaCore(const DecodeParams&, const Job&, float* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    g = lane >> 2;
    t = lane & 3;
    par = reinterpret_cast<float4*>(scratch) + warp * 32;
    rvs = scratch + W * 32 * 4 + warp * 32;
  }

  __device__ __forceinline__ void load_k(const CacheView& c, int64_t slot, int sub, int key, int lim) {
    // Key `key` (of the block's g, g + 8) sits at pool index `slot`; beyond `lim` nothing is touched.
#pragma unroll
    for (int i = 0; i < KW; ++i) kf[sub][key][i] = 0;
    if (key * 8 + g < lim) load_words<KB, 4 * KV>(static_cast<const char*>(c.k) + slot * (D * ES) + t * KV, kf[sub][key]);
  }
  __device__ __forceinline__ void load_v(const CacheView& c, int64_t slot, int sub, int i, int lim) {
#pragma unroll
    for (int j = 0; j < VW; ++j) vf[sub][i][j] = 0;
    if ((i >> 1) * 8 + 2 * t + (i & 1) < lim)
      load_words<VB, 8 * VV>(static_cast<const char*>(c.v) + slot * (D * ES) + g * VV, vf[sub][i]);
  }
  // The blocks of step st of the tile at pool index `base` with `lim` keys.
  __device__ __forceinline__ void load_k_step(const CacheView& c, int64_t base, int st, int lim) {
#pragma unroll
    for (int sub = 0; sub < SUB; ++sub)
#pragma unroll
      for (int key = 0; key < 2; ++key) {
        const int first = (st * SUB + sub) * 16;
        load_k(c, base + first + key * 8 + g, sub, key, lim - first);
      }
  }
  __device__ __forceinline__ void load_v_step(const CacheView& c, int64_t base, int st, int lim) {
#pragma unroll
    for (int sub = 0; sub < SUB; ++sub)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int first = (st * SUB + sub) * 16;
        load_v(c, base + first + (i >> 1) * 8 + 2 * t + (i & 1), sub, i, lim - first);
      }
  }

  template <bool kPrefix>
  __device__ __forceinline__ void load_q(const DecodeParams& p, const Job& job) {
    const __half* q = static_cast<const __half*>(p.q) + job.h * p.sq.h + (kPrefix ? 0 : job.b * p.sq.b);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = nt * 8 + g;
      const bool ok = r < job.rows;
      int i = job.r0 + (ok ? r : 0);
      const __half* row = q;
      if (kPrefix) {
        const int b = i / p.n;
        i -= b * p.n;
        row += b * p.sq.b;
      }
      row += i * p.sq.t;
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const int idx = 4 * s + 2 * w, d = (idx / KE * 4 + t) * KE + idx % KE;
          uint32_t x;
          if (p.q_pairs) {
            x = *reinterpret_cast<const uint32_t*>(row + d);
          } else {
            const __half2 h = __halves2half2(row[d * p.sq.d], row[(d + 1) * p.sq.d]);
            x = *reinterpret_cast<const uint32_t*>(&h);
          }
          qf[nt][s][w] = ok ? x : 0u;
        }
    }
  }

  // S^T of one 16-key block.
  __device__ __forceinline__ void scores(int sub, float (&z)[NT][4]) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) z[nt][i] = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      uint32_t a[4];
      if constexpr (kInt8) {
        const uint32_t x = kf[sub][0][s] ^ 0x80808080u, y = kf[sub][1][s] ^ 0x80808080u;
        a[0] = codes_to_half2<0x4140>(x);
        a[1] = codes_to_half2<0x4140>(y);
        a[2] = codes_to_half2<0x4342>(x);
        a[3] = codes_to_half2<0x4342>(y);
      } else {
        a[0] = kf[sub][0][2 * s];
        a[1] = kf[sub][1][2 * s];
        a[2] = kf[sub][0][2 * s + 1];
        a[3] = kf[sub][1][2 * s + 1];
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma16816(z[nt], a, qf[nt][s][0], qf[nt][s][1]);
    }
  }

  // Softmax of N blocks of scores (z + lv in log2 units) and their products with V.
  template <int N>
  __device__ __forceinline__ void accumulate(float (&z)[N][NT][4], const float (&rv)[N][2]) {
    bool grow = false;
    float top[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float x = -kInf;
#pragma unroll
        for (int b = 0; b < N; ++b) x = fmaxf(x, fmaxf(z[b][nt][q], z[b][nt][q + 2]));
        top[nt][q] = x;
        grow |= x > m[nt][q] + 8.f;
      }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          float x = fmaxf(top[nt][q], m[nt][q]);
#pragma unroll
          for (int o_ = 4; o_ < 32; o_ <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o_));
          const float f = state_weight(m[nt][q], x);
          m[nt][q] = x;
          l[nt][q] *= f;
#pragma unroll
          for (int j = 0; j < MT; ++j) {
            o[j][nt][q] *= f;
            o[j][nt][q + 2] *= f;
          }
        }
    }
    uint32_t pb[N][NT][2];
#pragma unroll
    for (int b = 0; b < N; ++b)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float ref = m[nt][i & 1] == -kInf ? 0.f : m[nt][i & 1];  // a row that has seen nothing yet
          e[i] = ex2(z[b][nt][i] - ref);
          if constexpr (kInt8)
            l[nt][i & 1] = fmaf(e[i], rv[b][i >> 1], l[nt][i & 1]);
          else
            l[nt][i & 1] += e[i];
        }
        pb[b][nt][0] = transpose8x8(pack_half2(e[0], e[1]));
        pb[b][nt][1] = transpose8x8(pack_half2(e[2], e[3]));
      }
#pragma unroll
    for (int b = 0; b < N; ++b) {
      if constexpr (kInt8) {
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          const uint32_t k0 = vf[b][0][w] ^ 0x80808080u, k1 = vf[b][1][w] ^ 0x80808080u;
          const uint32_t k2 = vf[b][2][w] ^ 0x80808080u, k3 = vf[b][3][w] ^ 0x80808080u;
#pragma unroll
          for (int half = 0; half < (MT < 2 ? 1 : 2); ++half) {
            const uint32_t x = half ? __byte_perm(k0, k1, 0x7362) : __byte_perm(k0, k1, 0x5140);
            const uint32_t y = half ? __byte_perm(k2, k3, 0x7362) : __byte_perm(k2, k3, 0x5140);
            const uint32_t a[4] = {codes_to_half2<0x4140>(x), codes_to_half2<0x4342>(x), codes_to_half2<0x4140>(y),
                                   codes_to_half2<0x4342>(y)};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816(o[2 * w + half][nt], a, pb[b][nt][0], pb[b][nt][1]);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          const uint32_t a[4] = {__byte_perm(vf[b][0][j], vf[b][1][j], 0x5410), __byte_perm(vf[b][0][j], vf[b][1][j], 0x7632),
                                 __byte_perm(vf[b][2][j], vf[b][3][j], 0x5410), __byte_perm(vf[b][2][j], vf[b][3][j], 0x7632)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816(o[j][nt], a, pb[b][nt][0], pb[b][nt][1]);
        }
      }
    }
  }

  template <bool kPrefix>
  __device__ __forceinline__ void run(const DecodeParams& p, const Job& job) {
    const CacheView& c = p.c;
    const int lane = threadIdx.x & 31;
    // The first loads of the run go out before anything else.
    int tile = job.t1 - 1;
    int64_t base = -1, next = -1;
    int lim = 0;
    float phi = kInf, psi = 0.f, ks = 0.f, vs = 0.f;
    if (tile >= job.t0) {
      base = slot_of(c, job.table, job.h, tile * 32);
      if (tile > job.t0) next = slot_of(c, job.table, job.h, tile * 32 - 32);
      lim = base < 0 ? 0 : min(32, job.end - tile * 32);
      load_k_step(c, base, 0, lim);
      load_v_step(c, base, 0, lim);
      if (lane < lim) {
        phi = c.phi[base + lane];
        psi = c.psi[base + lane];
        if (kInt8) {
          ks = c.ks[base + lane];
          vs = c.vs[base + lane];
        }
      }
    }
    load_q<kPrefix>(p, job);
    NewTokens nw{kInf, 0.f, kInf, -1, 0};
    if constexpr (!kPrefix) nw = load_new(c, job.table, job.h, job.end, job.n_new);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        m[nt][q] = -kInf;
        l[nt][q] = 0.f;
        const int r = nt * 8 + 2 * t + q;
        if constexpr (kPrefix) {
          low[nt][q] = r < job.rows ? p.row_min[int64_t(job.h) * (p.B * p.n) + job.r0 + r] : kInf;
        } else {
          const int i = job.r0 + r - job.lead;
          const float x = __shfl_sync(0xffffffffu, nw.low, i & 31);
          low[nt][q] = i >= 0 && i < job.n_new ? x : kInf;
        }
#pragma unroll
        for (int j = 0; j < MT; ++j) o[j][nt][q] = o[j][nt][q + 2] = 0.f;
      }
    if (tile >= job.t0) {
      float mid = job.t1 * 32 < job.end ? later_min(c, job.table, job.h, job.t1 * 32, job.end) : kInf;
      for (; tile >= job.t0; --tile) {
        float all;
        const float suf = fminf(suffix_min(phi, all), mid);
        mid = fminf(mid, all);
        const bool ok = lane < lim;
        __syncwarp();
        float lv = ok ? 0.f : -kInf;
        if constexpr (kInt8) {
          const float v = fmaxf(vs, 0x1p-90f);
          if (ok) lv = lg2(v);
          rvs[lane] = rcp_approx_f(v);
        }
        par[lane] = make_float4(ok ? fminf(suf - psi, 0.f) : 0.f, psi, ok ? (kInt8 ? ks : 1.f) * p.scale2 : 0.f, lv);
        __syncwarp();
        // The next tile's field and scales, and the page after it.
        const int64_t here = base;
        const int lim_here = lim;
        base = next;
        lim = tile > job.t0 && base >= 0 ? 32 : 0;
        next = tile - 1 > job.t0 ? slot_of(c, job.table, job.h, tile * 32 - 64) : -1;
        phi = kInf;
        psi = ks = vs = 0.f;
        if (lane < lim) {
          phi = c.phi[base + lane];
          psi = c.psi[base + lane];
          if (kInt8) {
            ks = c.ks[base + lane];
            vs = c.vs[base + lane];
          }
        }
#pragma unroll
        for (int st = 0; st < STEPS; ++st) {
          float z[SUB][NT][4], rv[SUB][2];
#pragma unroll
          for (int sub = 0; sub < SUB; ++sub) scores(sub, z[sub]);
          if (st + 1 < STEPS)
            load_k_step(c, here, st + 1, lim_here);
          else
            load_k_step(c, base, 0, lim);
#pragma unroll
          for (int sub = 0; sub < SUB; ++sub)
#pragma unroll
            for (int key = 0; key < 2; ++key) {
              const int at = (st * SUB + sub) * 16 + key * 8 + g;
              const float4 x = par[at];
              rv[sub][key] = kInt8 ? rvs[at] : 1.f;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                  const float b = fminf(x.x, low[nt][q] - x.y);
                  float& zz = z[sub][nt][2 * key + q];
                  zz = fmaf(zz, x.z, fmaf(job.bias, b, x.w));
                }
            }
          accumulate<SUB>(z, rv);
          if (st + 1 < STEPS)
            load_v_step(c, here, st + 1, lim_here);
          else
            load_v_step(c, base, 0, lim);
        }
      }
    }
    if constexpr (!kPrefix)
      if (job.last) run_new(p, job, nw);
  }

  // The newest tokens among themselves: one block of up to 16 keys, whose range minima are taken pair by pair.
  __device__ __forceinline__ void run_new(const DecodeParams& p, const Job& job, const NewTokens& nw) {
    const CacheView& c = p.c;
#pragma unroll
    for (int key = 0; key < 2; ++key) {
      const int64_t slot = __shfl_sync(0xffffffffu, nw.slot, key * 8 + g);
      load_k(c, slot, 0, key, slot >= 0 ? 16 : 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t slot = __shfl_sync(0xffffffffu, nw.slot, (i >> 1) * 8 + 2 * t + (i & 1));
      load_v(c, slot, 0, i, slot >= 0 ? 16 : 0);
    }
    float z[1][NT][4], rv[1][2];
    scores(0, z[0]);
#pragma unroll
    for (int key = 0; key < 2; ++key) {
      const int j = key * 8 + g;
      const int64_t slot = __shfl_sync(0xffffffffu, nw.slot, j);
      float f = p.scale2, lv = 0.f;
      rv[0][key] = 1.f;
      if constexpr (kInt8) {
        if (slot >= 0) {
          const float v = fmaxf(c.vs[slot], 0x1p-90f);
          f *= c.ks[slot];
          lv = lg2(v);
          rv[0][key] = rcp_approx_f(v);
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int i = job.r0 + nt * 8 + 2 * t + q - job.lead;
          const float b = new_pair(nw, j, i);
          float& zz = z[0][nt][2 * key + q];
          zz = slot >= 0 && j <= i ? fmaf(zz, f, fmaf(job.bias, b, lv)) : -kInf;
        }
    }
    float (&zz)[1][NT][4] = z;
    accumulate<1>(zz, rv);
  }

  __device__ __forceinline__ void store(float* sm, float* sl, float* sO, int rows) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float x = l[nt][q];
#pragma unroll
        for (int o_ = 4; o_ < 32; o_ <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o_);
        const int r = nt * 8 + 2 * t + q;
        if (r < rows) {
          if (g == 0) {
            sm[r] = m[nt][q];
            sl[r] = x;
          }
#pragma unroll
          for (int j = 0; j < MT; ++j) {
            const int i = 2 * j, d = (i / VE * 8 + g) * VE + i % VE;
            *reinterpret_cast<float2*>(sO + r * D + d) = make_float2(o[j][nt][q], o[j][nt][q + 2]);
          }
        }
      }
  }
};

template <bool kInt8>
cudaError_t launch_for(const DecodeParams& p, bool prefix, int splits, cudaStream_t s) {
  // 16 rows at a time where there are more than 8, except at D = 256, whose accumulators leave no registers for them.
  const bool wide = (prefix ? p.B * p.n : p.n) > 8;
  switch (p.c.D) {
#define FPA_CASE(D)                                                                            \
  case D:                                                                                      \
    return wide ? launch_decode_core<MmaCore<D, kInt8, 2>>(p, prefix, splits, s)               \
                : launch_decode_core<MmaCore<D, kInt8, 1>>(p, prefix, splits, s);
    FPA_CASE(16)
    FPA_CASE(32)
    FPA_CASE(64)
    FPA_CASE(128)
#undef FPA_CASE
    default:
      return launch_decode_core<MmaCore<256, kInt8, 1>>(p, prefix, splits, s);
  }
}

}  // namespace

cudaError_t launch_decode_mma(const DecodeParams& p, bool int8, bool prefix, int splits, cudaStream_t s) {
  return int8 ? launch_for<true>(p, prefix, splits, s) : launch_for<false>(p, prefix, splits, s);
}

}  // namespace fpa
