// Decode attention for fp16 queries over an fp16 or int8 cache, on the tensor cores (mma.sync m16n8k16).
//
// The products are S^T = K Q^T (16 keys x 16 d times 16 d x 8 rows) and O^T = V^T P^T (16 d x 16 keys times 16 keys x 8
// rows): the keys, which are many, fill the instruction's 16 rows, and the query rows, which are few, its 8 columns.
// With at most 16 rows there are at most 32 flops a byte, a tenth of what would make the tensor cores' rate matter;
// the bytes bound it, then the instructions that turn them into fragments. Every warp keeps a ring of its own in
// shared memory, filled by cp.async kStages - 1 blocks of keys ahead: enough bytes in flight on an SM however few
// CTAs it holds, no register held by a pending load, and no barrier between warps. Fragments come out with ldmatrix:
// plain for K; transposed for V, where the transposition of pairs of bytes also brings together the codes of two keys
// that an int8 fragment needs side by side. The 16-byte chunks of a row are permuted in shared memory so that the
// eight rows of a matrix lie in different banks. P passes from the accumulators' layout to the operand's with movmatrix.
//
// int8: a stored byte is u = code + 128. K's bytes are used as they are: with a zero byte above, u is the fp16
// subnormal u 2^-24, exactly, and the accumulator starts at -128 2^-24 sum_d q_d, which takes the offset out again;
// K's scale multiplies the finished product. (The offset's products are of the size of the others: float32 loses
// nothing that matters.) V's bytes become code exactly (0x6400 | u is 1024 + u), since sums over many keys would
// cancel; V's scale goes into the exponent. With lv = log2 vs, P' = 2^(z + lv - m) <= 2^8 for m = max(z + lv) as of its
// last update, l = sum P' / vs and o = sum P' code / l: the factors fp16 holds are scaled to the largest contribution
// whatever the scales are, at the cost of the plain softmax. P' is rounded to fp16 (2^-11 relative, as the training
// kernels round P); sums and states stay in fp32. The maximum is updated only when it grows by more than 8 (in log2
// units), decided by the whole warp.
#include <cuda_fp16.h>

#include "fpa_decode.cuh"
#include "fpa_sm100.cuh"

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

// Four (two) 8 x 8 matrices of 16-bit elements, the rows at the lanes' addresses.
template <bool kTrans>
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  if constexpr (kTrans)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool kTrans>
__device__ __forceinline__ void ldmatrix2(uint32_t addr, uint32_t (&r)[4]) {
  if constexpr (kTrans)
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr) : "memory");
}

// 16 (4) bytes to shared memory; zeros without touching the source where `ok` is false.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(ok ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Two codes as halves, from the bytes of x that kSel picks.
template <uint32_t kSel>
__device__ __forceinline__ uint32_t codes_to_half2(uint32_t x) {
  const uint32_t y = __byte_perm(x, 0x64646464u, kSel);
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&y), __floats2half2_rn(1152.f, 1152.f));
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <int D_, bool kInt8, int NT>
struct MmaCore {
  static constexpr int D = D_, NQ = 8 * NT;
  static constexpr int ES = kInt8 ? 1 : 2;              // bytes of a stored element
  static constexpr int RB = D * ES;                     // ... of a row
  static constexpr int CPR = RB / 16;                   // 16-byte chunks of a row
  static constexpr int SUB = RB <= 128 ? 2 : 1;         // 16-key blocks handled together
  static constexpr int kKeys = 16 * SUB;
  static constexpr int KS = D / 16, MT = D / 16;
  static constexpr int kArray = kKeys * RB;             // bytes of K (and of V) in a stage
  static constexpr int kStage = 2 * kArray + (kInt8 ? 4 : 2) * kKeys * 4;
  // Two stages leave room for more warps, which gain more than a third stage (fp16 D = 128, 16 heads, 4 x 16383
  // tokens, 5 rows: 64 us against 69); at D = 256 in fp16 few warps fit either way (48 us with three, 60 with two).
  static constexpr int kStages = RB < 512 ? 2 : 3;
  static constexpr int kRingBytes = kStages * kStage;   // of a warp
  static constexpr int kCtaFloats = 0, kWarpFloats = kMaxNew * kMaxNew;  // keys' values, or the new pairs
  static_assert(kWarpFloats >= kKeys * 4, "scratch");
  static constexpr int kMinBlocks = D * NT <= 64 ? (RB <= 64 ? 5 : 4) : D * NT <= 128 ? 3 : 2;
  static constexpr int kManyBlocks = 16;  // of a warp: enough that a second round of CTAs pays its start-up
  using Out = __half;

  uint32_t qf[NT][KS][2];
  float o[MT][NT][4], m[NT][2], l[NT][2], low[NT][2], zero[NT][2];
  float4* par;    // per key of the block: see field_of
  float sign;     // of beta (1 for 0)
  uint32_t ring;  // this warp's stages
  int lane, g, t;

  __device__ __forceinline__ MmaCore(const DecodeParams&, const Job&, float* scratch, char* rings) {
    const int warp = threadIdx.x >> 5;
    lane = threadIdx.x & 31;
    g = lane >> 2;
    t = lane & 3;
    par = reinterpret_cast<float4*>(scratch + warp * kWarpFloats);
    ring = static_cast<uint32_t>(__cvta_generic_to_shared(rings)) + warp * kRingBytes;
  }

  // Byte offset of 16-byte chunk c of a row: bits of the chunk's number are flipped by the row's place among the eight
  // rows that a matrix reads at once. Stages start at multiples of 128 bytes and rows are powers of two, so for a
  // fixed row, chunk c lies at chunk_at(row, c0) ^ 16 (c ^ c0) for any c0 < 8 with c < 8.
  __device__ __forceinline__ static constexpr int swizzle(int row) {
    constexpr int kLine = RB < 128 ? 128 / RB : 1, kMask = (CPR < 8 ? CPR : 8) - 1;
    return (row / kLine) & kMask;
  }
  __device__ __forceinline__ static int chunk_at(int row, int c) { return (row * CPR + (c ^ swizzle(row))) * 16; }
  // Address of chunk (even c) + `odd` of a row whose chunk `odd` is at `at`.
  __device__ __forceinline__ static uint32_t chunk_from(uint32_t at, int c) { return (at ^ ((c & 7) * 16)) + (c >> 3) * 128; }

  // A block of keys that lie one after the other from pool index `base` on, `lim` of them.
  __device__ __forceinline__ void fetch(const CacheView& c, uint32_t st, int64_t base, int lim) {
    const char* k = static_cast<const char*>(c.k) + base * RB + lane * 16;
    const char* v = static_cast<const char*>(c.v) + base * RB + lane * 16;
    // The lane's chunk of every 512 bytes: its row moves by whole groups of rows, which flip other bits.
    const uint32_t at = st + chunk_at(lane / CPR, lane % CPR);
    if (lim == kKeys) {
#pragma unroll
      for (int i = 0; i < kKeys * CPR; i += 32) {
        const uint32_t to = (at ^ (swizzle(i / CPR) * 16)) + i * 16;
        copy16(to, k + i * 16, true);
        copy16(to + kArray, v + i * 16, true);
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < kKeys * CPR; i += 32) {
        const uint32_t to = (at ^ (swizzle(i / CPR) * 16)) + i * 16;
        copy16(to, k + i * 16, (i + lane) / CPR < lim);
        copy16(to + kArray, v + i * 16, (i + lane) / CPR < lim);
      }
    }
    if (lane < kKeys) fetch_field(c, st, base + lane, lane < lim);
  }
  __device__ __forceinline__ void fetch_field(const CacheView& c, uint32_t st, int64_t slot, bool ok) {
    const uint32_t at = st + 2 * kArray + lane * 4;
    copy4(at, c.phi + slot, ok);
    copy4(at + kKeys * 4, c.psi + slot, ok);
    if constexpr (kInt8) {
      copy4(at + 2 * kKeys * 4, c.ks + slot, ok);
      copy4(at + 3 * kKeys * 4, c.vs + slot, ok);
    }
  }
  // The newest tokens, which may lie in two pages: each key at its own place.
  __device__ __forceinline__ void fetch_new(const CacheView& c, uint32_t st, const NewTokens& nw) {
#pragma unroll 1
    for (int i = 0; i < kKeys * CPR; i += 32) {
      const int idx = i + lane, row = idx / CPR, ch = idx % CPR, at = chunk_at(row, ch);
      const int64_t slot = __shfl_sync(0xffffffffu, nw.slot, row & 31);
      copy16(st + at, static_cast<const char*>(c.k) + (slot < 0 ? 0 : slot) * RB + ch * 16, slot >= 0);
      copy16(st + kArray + at, static_cast<const char*>(c.v) + (slot < 0 ? 0 : slot) * RB + ch * 16, slot >= 0);
    }
    if (lane < kKeys) fetch_field(c, st, nw.slot < 0 ? 0 : nw.slot, nw.slot >= 0);
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
          // fp16: elements 2t, 2t + 1 and 2t + 8, 2t + 9 of the 16; int8: the four that a 32-bit word holds.
          const int d = s * 16 + (kInt8 ? 4 * t + 2 * w : 2 * t + 8 * w);
          __half2 x;
          if (p.q_pairs)
            x = *reinterpret_cast<const __half2*>(row + d);
          else
            x = __halves2half2(row[d * p.sq.d], row[(d + 1) * p.sq.d]);
          if (!ok) x = __floats2half2_rn(0.f, 0.f);
          qf[nt][s][w] = *reinterpret_cast<const uint32_t*>(&x);
        }
    }
  }
  // What the accumulators of the scores start at, for the rows of this lane's columns.
  __device__ __forceinline__ void sum_q() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if constexpr (kInt8) {
        float sum = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const __half2 x = *reinterpret_cast<const __half2*>(&qf[nt][s][w]);
            sum += __low2float(x) + __high2float(x);
          }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
        for (int c = 0; c < 2; ++c) zero[nt][c] = -128.f * 0x1p-24f * __shfl_sync(0xffffffffu, sum, (2 * t + c) * 4);
      } else {
        zero[nt][0] = zero[nt][1] = 0.f;
      }
    }
  }

  // S^T of one 16-key block (int8: times 2^-24).
  __device__ __forceinline__ void scores(uint32_t st, int sub, float (&z)[NT][4]) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) z[nt][i] = zero[nt][i & 1];
    const uint32_t at = st + sub * 16 * RB + chunk_at(lane & 15, KS == 1 && kInt8 ? 0 : lane >> 4);
    if constexpr (kInt8) {
      // A matrix of eight rows by 16 codes; four of them are two steps of 16 d.
#pragma unroll
      for (int s = 0; s < KS; s += 2) {
        uint32_t x[4];
        if constexpr (KS == 1)
          ldmatrix2<false>(at, x);
        else
          ldmatrix4<false>(chunk_from(at, s), x);
#pragma unroll
        for (int w = 0; w < (KS == 1 ? 1 : 2); ++w) {
          const uint32_t a[4] = {__byte_perm(x[2 * w], 0, 0x4140), __byte_perm(x[2 * w + 1], 0, 0x4140),
                                 __byte_perm(x[2 * w], 0, 0x4342), __byte_perm(x[2 * w + 1], 0, 0x4342)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816(z[nt], a, qf[nt][s + w][0], qf[nt][s + w][1]);
        }
      }
    } else {
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        uint32_t a[4];
        ldmatrix4<false>(chunk_from(at, 2 * s), a);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma16816(z[nt], a, qf[nt][s][0], qf[nt][s][1]);
      }
    }
  }

  // O^T += V^T P^T for one 16-key block.
  __device__ __forceinline__ void values(uint32_t st, int sub, const uint32_t (&pb)[NT][2]) {
    const uint32_t v = st + kArray + sub * 16 * RB;
    if constexpr (kInt8) {
      // Transposed as 16-bit pairs: lane (g, t) gets columns 2g, 2g + 1 of the keys 2t, 2t + 1.
      const uint32_t at = v + chunk_at(lane & 15, MT == 1 ? 0 : lane >> 4);
#pragma unroll
      for (int j = 0; j < MT; j += 2) {
        uint32_t x[4];
        if constexpr (MT == 1)
          ldmatrix2<true>(at, x);
        else
          ldmatrix4<true>(chunk_from(at, j), x);
#pragma unroll
        for (int w = 0; w < (MT == 1 ? 1 : 2); ++w) {
          const uint32_t a[4] = {codes_to_half2<0x4240>(x[2 * w]), codes_to_half2<0x4341>(x[2 * w]),
                                 codes_to_half2<0x4240>(x[2 * w + 1]), codes_to_half2<0x4341>(x[2 * w + 1])};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816(o[j + w][nt], a, pb[nt][0], pb[nt][1]);
        }
      }
    } else {
      // Matrices in the order (keys 0-7, d 0-7), (0-7, 8-15), (8-15, 0-7), (8-15, 8-15).
      const uint32_t at = v + chunk_at((lane & 7) + ((lane >> 4) << 3), (lane >> 3) & 1);
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        uint32_t a[4];
        ldmatrix4<true>(chunk_from(at, 2 * j), a);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma16816(o[j][nt], a, pb[nt][0], pb[nt][1]);
      }
    }
  }

  // Softmax of a block's scores (z + lv in log2 units, less ref) and their products with V.
  __device__ __forceinline__ void accumulate(uint32_t st, float2 (&z)[SUB][NT][2], const float (&rv)[SUB][2]) {
    float top[NT][2];
    bool grow = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      top[nt][0] = top[nt][1] = -kInf;
#pragma unroll
      for (int b = 0; b < SUB; ++b) {
        top[nt][0] = sm100::fmax3f(top[nt][0], z[b][nt][0].x, z[b][nt][1].x);
        top[nt][1] = sm100::fmax3f(top[nt][1], z[b][nt][0].y, z[b][nt][1].y);
      }
      // A row that has seen nothing yet (m = -inf, ref = 0) takes any maximum.
#pragma unroll
      for (int q = 0; q < 2; ++q) grow |= top[nt][q] > (m[nt][q] == -kInf ? -kInf : 8.f);
    }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float shift[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const float ref = m[nt][q] == -kInf ? 0.f : m[nt][q];
          float x = fmaxf(top[nt][q] + ref, m[nt][q]);
#pragma unroll
          for (int o_ = 4; o_ < 32; o_ <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o_));
          const float f = state_weight(m[nt][q], x);
          shift[q] = ref - (x == -kInf ? 0.f : x);
          m[nt][q] = x;
          l[nt][q] *= f;
#pragma unroll
          for (int j = 0; j < MT; ++j) {
            o[j][nt][q] *= f;
            o[j][nt][q + 2] *= f;
          }
        }
#pragma unroll
        for (int b = 0; b < SUB; ++b)
#pragma unroll
          for (int key = 0; key < 2; ++key) z[b][nt][key] = __fadd2_rn(z[b][nt][key], make_float2(shift[0], shift[1]));
      }
    }
    uint32_t pb[SUB][NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float2 sum = make_float2(l[nt][0], l[nt][1]);
#pragma unroll
      for (int b = 0; b < SUB; ++b)
#pragma unroll
        for (int key = 0; key < 2; ++key) {
          const float2 e = make_float2(ex2(z[b][nt][key].x), ex2(z[b][nt][key].y));
          sum = kInt8 ? __ffma2_rn(e, make_float2(rv[b][key], rv[b][key]), sum) : __fadd2_rn(sum, e);
          pb[b][nt][key] = transpose8x8(pack_half2(e.x, e.y));
        }
      l[nt][0] = sum.x;
      l[nt][1] = sum.y;
    }
#pragma unroll
    for (int b = 0; b < SUB; ++b) values(st, b, pb[b]);
  }

  // This lane's key of the stage: its field and scales. With b' = beta log2(e), the bias plus lv of a row is b' min(a_s,
  // M - psi_s) + lv, which times the sign of b' is min(a, low + e) for a = |b'| a_s + sign lv, e = -|b'| (psi_s - level) +
  // sign lv and the row's low = |b'| (M - level); sign f is the product's factor. No such key: a = e = -sign inf. The level
  // is phi of the first new token (of the prefix's last token), which M is near to, and psi_s too wherever the bias is
  // small: what is rounded here is then of the bias's own size, however far from zero the walk stands.
  struct Field {
    float phi, psi, f, lv, rv;
  };
  __device__ __forceinline__ Field field_of(const DecodeParams& p, uint32_t st, bool ok) {
    auto word = [&](int i) {
      float x;
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(st + 2 * kArray + (i * kKeys + lane) * 4) : "memory");
      return x;
    };
    Field f{kInf, 0.f, 0.f, -kInf, 1.f};
    if (ok) {
      f.phi = word(0);
      f.psi = word(1);
      f.f = p.scale2;
      f.lv = 0.f;
      if constexpr (kInt8) {
        const float v = fmax_nan(word(3), 0x1p-90f);
        f.f *= word(2) * 0x1p24f;
        f.lv = lg2(v);
        f.rv = rcp_approx_f(v);
        if (v != v) f.rv = 1.f;  // NaN reaches the rows that see the key through lv, and no other
      }
    }
    return f;
  }

  // The newest tokens' values in fp16 may hold infinities and NaN, which a product with a weight of zero would bring to the
  // rows that do not see the token. Such elements count as zeros in the tile's products (true if there are any) ...
  __device__ __forceinline__ bool clear_wild(uint32_t st) {
    const uint32_t v = st + kArray + lane * 16;
    auto load = [](uint32_t at) {
      uint4 w;
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(at) : "memory");
      return w;
    };
    __half2 sum = __floats2half2_rn(0.f, 0.f);
#pragma unroll 4
    for (int i = 0; i < kArray; i += 512) {
      const uint4 w = load(v + i);
      const __half2* h = reinterpret_cast<const __half2*>(&w);
#pragma unroll
      for (int j = 0; j < 4; ++j) sum = __hfma2(h[j], __floats2half2_rn(0.f, 0.f), sum);
    }
    if (!__any_sync(0xffffffffu, __low2float(sum) != 0.f || __high2float(sum) != 0.f)) return false;
    auto finite = [](uint32_t x) {
      return ((x & 0x7c00u) == 0x7c00u ? 0u : x & 0xffffu) | ((x & 0x7c000000u) == 0x7c000000u ? 0u : x & 0xffff0000u);
    };
#pragma unroll 1
    for (int i = 0; i < kArray; i += 512) {
      const uint4 w = load(v + i);
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(v + i), "r"(finite(w.x)), "r"(finite(w.y)), "r"(finite(w.z)),
                   "r"(finite(w.w)) : "memory");
    }
    __syncwarp();
    return true;
  }
  // ... and join the rows that see them afterwards: z[key * kMaxNew + row] are their scores, -inf where masked.
  __device__ __forceinline__ void add_wild(const CacheView& c, const NewTokens& nw, const float* z) {
#pragma unroll 1
    for (int k = 0; k < nw.nn; ++k) {
      const int64_t slot = __shfl_sync(0xffffffffu, nw.slot, k);
      if (slot < 0) continue;
      const __half* v = static_cast<const __half*>(c.v) + slot * D + g;
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float x = __half2float(v[j * 16 + half * 8]);
          if (fabsf(x) < kInf) continue;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const float s = z[k * kMaxNew + nt * 8 + 2 * t + q];
              if (s != -kInf) o[j][nt][q + 2 * half] += x * ex2(s - m[nt][q]);
            }
        }
    }
  }

  template <bool kPrefix>
  __device__ __forceinline__ void run(const DecodeParams& p, const Job& job) {
    const CacheView& c = p.c;
    // The run's blocks from the latest to the earliest. First the table's entries that the start needs, all at once,
    // with the queries; then all that they lead to: two dependent trips to memory instead of one for each use.
    const int history = job.t1 - job.t0, total = history + (job.last ? 1 : 0);
    int next = job.t1 - 1;  // next block to fetch
    const int pid0 = history > 0 ? job.table[(next * kKeys) >> c.page_shift] : -1;
    const int pid1 = history > 1 ? job.table[((next - 1) * kKeys) >> c.page_shift] : -1;
    const int pid2 = kStages == 3 && history > 2 ? job.table[((next - 2) * kKeys) >> c.page_shift] : -1;
    const int pid_level = kPrefix ? job.table[(job.end - 1) >> c.page_shift] : -1;
    const int pid_new = !kPrefix && lane < job.n_new ? job.table[(job.end + lane) >> c.page_shift] : -1;
    LaterMin later;
    later.ids(c, job.table, job.t1 * kKeys, history > 0 ? job.end : 0);
    load_q<kPrefix>(p, job);
    int64_t base = -1;
    // Keys of the blocks on their way, the earliest first: none of a block whose page lies outside the pool.
    int lims[kStages - 1] = {};
    auto fetch_block = [&](int i, int& lim) {
      lim = base < 0 ? 0 : min(kKeys, job.end - next * kKeys);
      fetch(c, ring + (i % kStages) * kStage, base < 0 ? 0 : base, lim);
      --next;
    };
    auto fetch_next = [&](int i) {
      // Block i of the run into its stage; the place of the one after it, where that lies in another page, is looked
      // up meanwhile.
      fetch_block(i, lims[kStages - 2]);
      if (i + 1 < history) {
        if (((next + 1) * kKeys & ((1 << c.page_shift) - 1)) != 0 && base >= 0)
          base -= kKeys;
        else
          base = slot_of(c, job.table, job.h, next * kKeys);
      }
    };
    if (history > 0) {
      base = slot_in(c, pid0, job.h, next * kKeys);
      fetch_block(0, lims[0]);
    }
    if (history > 0 || !job.last) copy_commit();  // else the newest tokens' place is not known yet
    if constexpr (kStages == 3) {
      if (history > 1) {
        base = slot_in(c, pid1, job.h, next * kKeys);
        fetch_block(1, lims[1 % (kStages - 1)]);
      }
      if (history > 1 || !job.last) copy_commit();
      if (history > 2) base = slot_in(c, pid2, job.h, next * kKeys);
    } else {
      if (history > 1) base = slot_in(c, pid1, job.h, next * kKeys);
    }
    NewTokens nw{kInf, 0.f, kInf, -1, 0};
    if constexpr (!kPrefix) nw = load_new(c, pid_new, job.h, job.end, job.n_new);
    later.values(c, job.h);
    float level;
    if constexpr (kPrefix) {
      level = level_at(c, pid_level, job.h, job.end - 1);
    } else {
      level = __shfl_sync(0xffffffffu, nw.phi, 0);
      if (!(fabsf(level) < kInf)) level = 0.f;  // no new token, or a page outside the pool
    }
    sum_q();
    nw.low = prefix_min(nw.phi);
    sign = job.bias < 0.f ? -1.f : 1.f;
    const float strength = fabsf(job.bias);
    if (job.last && history < kStages - 1) {
      // Few blocks: the newest tokens' block and the empty groups after it.
      for (int i = history; i < kStages - 1; ++i) {
        if (i == history) fetch_new(c, ring + (i % kStages) * kStage, nw);
        copy_commit();
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        m[nt][q] = -kInf;
        l[nt][q] = 0.f;
        const int r = nt * 8 + 2 * t + q;
        float x;
        if constexpr (kPrefix) {
          x = r < job.rows ? p.row_min[int64_t(job.h) * (p.B * p.n) + job.r0 + r] : kInf;
        } else {
          const int i = job.r0 + r - job.lead;
          x = __shfl_sync(0xffffffffu, nw.low, i & 31);
          if (i < 0 || i >= job.n_new) x = kInf;
        }
        // strength 0: the bias is 0 whatever the minimum is (not 0 times infinity).
        low[nt][q] = strength == 0.f ? 0.f : strength * (x - level);
#pragma unroll
        for (int j = 0; j < MT; ++j) o[j][nt][q] = o[j][nt][q + 2] = 0.f;
      }
    float mid = later.finish(c, job.table, job.h);
    bool wild = false;
    for (int i = 0; i < total; ++i) {
      copy_wait<kStages - 2>();
      __syncwarp();
      const int lim = lims[0];
#pragma unroll
      for (int j = 1; j < kStages - 1; ++j) lims[j - 1] = lims[j];
      if (i + kStages - 1 < history)
        fetch_next(i + kStages - 1);
      else if (job.last && i + kStages - 1 == history)
        fetch_new(c, ring + ((i + kStages - 1) % kStages) * kStage, nw);
      copy_commit();
      const uint32_t st = ring + (i % kStages) * kStage;
      float s[SUB][NT][4], rv[SUB][2];
      float2 z[SUB][NT][2];  // per key g, g + 8 of each 16: rows 2t and 2t + 1
#pragma unroll
      for (int sub = 0; sub < SUB; ++sub) scores(st, sub, s[sub]);
      float2 ref[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        ref[nt] = make_float2(m[nt][0] == -kInf ? 0.f : -m[nt][0], m[nt][1] == -kInf ? 0.f : -m[nt][1]);
      const float2 sign2 = make_float2(sign, sign);
      if (i < history) {
        const Field f = field_of(p, st, lane < lim);
        float all;
        const float suf = fminf(suffix_min(f.phi, all), mid);
        mid = fminf(mid, all);
        if (lane < kKeys)
          par[lane] = make_float4(fmaf(-strength, f.psi - level, sign * f.lv), fmaf(strength, fminf(suf - f.psi, 0.f), sign * f.lv),
                                  sign * f.f, f.rv);
        __syncwarp();
#pragma unroll
        for (int sub = 0; sub < SUB; ++sub)
#pragma unroll
          for (int key = 0; key < 2; ++key) {
            const float4 x = par[sub * 16 + key * 8 + g];
            rv[sub][key] = x.w;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const float2 t2 = __fadd2_rn(make_float2(low[nt][0], low[nt][1]), make_float2(x.x, x.x));
              const float2 b = make_float2(fminf(x.y, t2.x), fminf(x.y, t2.y));
              const float2 zz = __ffma2_rn(make_float2(s[sub][nt][2 * key], s[sub][nt][2 * key + 1]), make_float2(x.z, x.z), b);
              z[sub][nt][key] = __ffma2_rn(zz, sign2, ref[nt]);
            }
          }
      } else {
        // The newest tokens among themselves.
        const Field f = field_of(p, st, lane < kKeys && nw.slot >= 0);
        float* pairs = reinterpret_cast<float*>(par);
        fill_pairs(nw, pairs);
#pragma unroll
        for (int sub = 0; sub < SUB; ++sub)
#pragma unroll
          for (int key = 0; key < 2; ++key) {
            const int j = sub * 16 + key * 8 + g;
            const float ff = __shfl_sync(0xffffffffu, f.f, j & 31), lv = __shfl_sync(0xffffffffu, f.lv, j & 31);
            rv[sub][key] = __shfl_sync(0xffffffffu, f.rv, j & 31);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float zz[2];
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const int i_ = job.r0 + nt * 8 + 2 * t + q - job.lead;
                zz[q] = -kInf;
                if (j < job.n_new && j <= i_ && i_ < job.n_new)
                  zz[q] = fmaf(s[sub][nt][2 * key + q], ff, fmaf(job.bias, pairs[j * kMaxNew + i_], lv));
              }
              z[sub][nt][key] = __fadd2_rn(make_float2(zz[0], zz[1]), ref[nt]);
            }
          }
        if constexpr (!kPrefix && !kInt8) wild = clear_wild(st);
        if (wild) {  // the pairs' place takes the scores (the newest tokens are the first 16 keys)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int key = 0; key < 2; ++key) {
              float* at = pairs + (key * 8 + g) * kMaxNew + nt * 8 + 2 * t;
              at[0] = z[0][nt][key].x - ref[nt].x;
              at[1] = z[0][nt][key].y - ref[nt].y;
            }
        }
      }
      accumulate(st, z, rv);
      __syncwarp();
    }
    copy_wait<0>();
    if constexpr (!kPrefix && !kInt8) {
      if (wild) add_wild(c, nw, reinterpret_cast<const float*>(par));
    }
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
            float* at = sO + r * D + j * 16;
            at[kInt8 ? 2 * g : g] = o[j][nt][q];
            at[kInt8 ? 2 * g + 1 : g + 8] = o[j][nt][q + 2];
          }
        }
      }
  }
};

template <bool kInt8>
cudaError_t launch_for(const DecodeParams& p, bool prefix, cudaStream_t s, int& launches) {
  // 16 rows at a time where there are more than 8, so that the keys are read and converted once: 16 x 12 (sequence, head)
  // pairs of 4096 int8 tokens, D = 64, 16 rows 34 us against 52 in two groups of 8; 4 x 16 of 16383, fp16 D = 128 106 against
  // 146 (short calls differ by little: 72 pairs of 1000 tokens 12.7 against 11.5). Not at D = 256, whose accumulators
  // leave no registers for them.
  const bool wide = (prefix ? p.B * p.n : p.n) > 8;
  switch (p.c.D) {
#define FPA_CASE(D)                                                                            \
  case D:                                                                                      \
    return wide ? launch_decode_core<MmaCore<D, kInt8, 2>>(p, prefix, s, launches)               \
                : launch_decode_core<MmaCore<D, kInt8, 1>>(p, prefix, s, launches);
    FPA_CASE(16)
    FPA_CASE(32)
    FPA_CASE(64)
    FPA_CASE(128)
#undef FPA_CASE
    default:
      return launch_decode_core<MmaCore<256, kInt8, 1>>(p, prefix, s, launches);
  }
}

}  // namespace

cudaError_t launch_decode_mma(const DecodeParams& p, bool int8, bool prefix, cudaStream_t s, int& launches) {
  return int8 ? launch_for<true>(p, prefix, s, launches) : launch_for<false>(p, prefix, s, launches);
}

}  // namespace fpa
