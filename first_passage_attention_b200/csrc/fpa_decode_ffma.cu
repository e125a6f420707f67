// Decode attention in float32 (FFMA), over a float32 or int8 cache, and the minima that a prefix pass needs.
//
// A warp takes 32 keys at a time. Scores: lane (g, t) = (lane / 4, lane % 4) holds a quarter of key g of eight, in
// runs of four elements that the four lanes of a key read side by side; two shuffles finish a product. The softmax has
// one key per lane, and the product with V one run of D / 32 columns per lane, P coming from shared memory four keys
// at a time. Everything is float32: this is the path of float32 models, whose tolerance rules out fp16 operands.
#include "fpa_decode.cuh"

namespace fpa {
namespace {

template <int D_, bool kInt8, int NR>
struct FfmaCore {
  static constexpr int D = D_, NQ = NR;
  static constexpr int CPL = D < 32 ? 1 : D / 32;   // columns of V for a lane
  static constexpr int CV = CPL < 4 ? CPL : 4;      // ... of one load
  static constexpr int KG = D < 32 ? 32 / D : 1;    // lanes that share a column take every KG-th key
  static constexpr int kMinBlocks = NR * CPL + D / 4 <= 64 ? 4 : 2;
  static constexpr int kKeys = 32, kRingBytes = 0;
  static constexpr int kCtaFloats = NR * D, kWarpFloats = NR * 32;
  using Out = float;

  float o[NR][CPL], m[NR], l[NR];
  float* qs;  // [NR][D]
  float* ss;  // [NR][32], this warp's scores and probabilities
  int lane, g, t;

  __device__ __forceinline__ FfmaCore(const DecodeParams&, const Job&, float* scratch, char*) {
    lane = threadIdx.x & 31;
    g = lane >> 2;
    t = lane & 3;
    qs = scratch;
    ss = scratch + NR * D + (threadIdx.x >> 5) * NR * 32;
  }

  __device__ __forceinline__ static int column(int j) { return (j / CV * 32 + (threadIdx.x & 31)) * CV + j % CV; }

  // Four elements d .. d + 3 of the key at pool index `slot` (codes for int8).
  __device__ __forceinline__ static float4 load4(const void* base, int64_t slot, int d) {
    if constexpr (kInt8) {
      const uchar4 x = __ldg(reinterpret_cast<const uchar4*>(static_cast<const char*>(base) + slot * D + d));
      return make_float4(x.x - 128, x.y - 128, x.z - 128, x.w - 128);
    } else {
      return __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(base) + slot * D + d));
    }
  }

  // V of one key, this lane's columns.
  __device__ __forceinline__ static void load_v(const void* base, int64_t slot, float (&v)[CPL]) {
    if constexpr (CV == 4) {
#pragma unroll
      for (int j = 0; j < CPL; j += 4) {
        const float4 x = load4(base, slot, column(j));
        v[j] = x.x, v[j + 1] = x.y, v[j + 2] = x.z, v[j + 3] = x.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
        const int64_t at = slot * D + (D < 32 ? (threadIdx.x & (D - 1)) : column(j));
        v[j] = kInt8 ? float(__ldg(static_cast<const unsigned char*>(base) + at) - 128) : __ldg(static_cast<const float*>(base) + at);
      }
    }
  }

  // Softmax of one key per lane (z = ss[r][lane] * f + bias(r) + lv) and the products with V of `n` keys whose pool
  // indices are slot(0), slot(1), ...
  template <class Bias, class Slot>
  __device__ __forceinline__ void accumulate(const CacheView& c, float f, float lv, float rv, int n, Bias bias, Slot slot) {
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const float b = bias(r);
      const float z = lv == -kInf || b == -kInf ? -kInf : fmaf(ss[r * 32 + lane], f, b + lv);
      if (__any_sync(0xffffffffu, z > m[r] + 8.f)) {
        float x = fmaxf(z, m[r]);
#pragma unroll
        for (int o_ = 16; o_ > 0; o_ >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o_));
        const float w = state_weight(m[r], x);
        m[r] = x;
        l[r] *= w;
#pragma unroll
        for (int j = 0; j < CPL; ++j) o[r][j] *= w;
      }
      const float e = ex2(z - (m[r] == -kInf ? 0.f : m[r]));
      l[r] = fmaf(e, rv, l[r]);
      ss[r * 32 + lane] = e;
    }
    __syncwarp();
    if constexpr (KG > 1) {
      for (int k = lane / D; k < n; k += KG) {
        const int64_t at = slot(k);
        if (at < 0) continue;
        float v[CPL];
        load_v(c.v, at, v);
#pragma unroll
        for (int r = 0; r < NR; ++r) o[r][0] = fmaf(ss[r * 32 + k], v[0], o[r][0]);
      }
    } else {
#pragma unroll 2
      for (int k = 0; k < n; k += 4) {
        float v[4][CPL];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int64_t at = k + i < n ? slot(k + i) : -1;
#pragma unroll
          for (int j = 0; j < CPL; ++j) v[i][j] = 0.f;
          if (at >= 0) load_v(c.v, at, v[i]);
        }
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          const float4 e = *reinterpret_cast<const float4*>(ss + r * 32 + k);
#pragma unroll
          for (int j = 0; j < CPL; ++j) {
            float x = o[r][j];
            x = fmaf(e.x, v[0][j], x);
            x = fmaf(e.y, v[1][j], x);
            x = fmaf(e.z, v[2][j], x);
            o[r][j] = fmaf(e.w, v[3][j], x);
          }
        }
      }
    }
    __syncwarp();
  }

  // Scores of 8 keys (this lane's key g at pool index `at`, or -1) into columns first .. first + 7.
  __device__ __forceinline__ void scores(const CacheView& c, int64_t at, int first) {
    float4 k[D / 16];
#pragma unroll
    for (int j = 0; j < D / 16; ++j) k[j] = at >= 0 ? load4(c.k, at, (j * 4 + t) * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        const float4 q = *reinterpret_cast<const float4*>(qs + r * D + (j * 4 + t) * 4);
        s = fmaf(q.x, k[j].x, s);
        s = fmaf(q.y, k[j].y, s);
        s = fmaf(q.z, k[j].z, s);
        s = fmaf(q.w, k[j].w, s);
      }
      s += __shfl_xor_sync(0xffffffffu, s, 1);
      s += __shfl_xor_sync(0xffffffffu, s, 2);
      if (t == (r & 3)) ss[r * 32 + first + g] = s;
    }
  }

  template <bool kPrefix>
  __device__ __forceinline__ void run(const DecodeParams& p, const Job& job) {
    const CacheView& c = p.c;
    for (int e = threadIdx.x; e < NR * D; e += blockDim.x) {
      const int r = e / D, d = e - r * D;
      float x = 0.f;
      if (r < job.rows) {
        int i = job.r0 + r, b = job.b;
        if (kPrefix) {
          b = i / p.n;
          i -= b * p.n;
        }
        x = static_cast<const float*>(p.q)[b * p.sq.b + job.h * p.sq.h + i * p.sq.t + d * p.sq.d];
      }
      qs[e] = x;
    }
    __syncthreads();
    NewTokens nw{kInf, 0.f, kInf, -1, 0};
    if constexpr (!kPrefix) {
      nw = load_new(c, lane < job.n_new ? job.table[(job.end + lane) >> c.page_shift] : -1, job.h, job.end, job.n_new);
      nw.low = prefix_min(nw.phi);
    }
    float low[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      m[r] = -kInf;
      l[r] = 0.f;
#pragma unroll
      for (int j = 0; j < CPL; ++j) o[r][j] = 0.f;
      if constexpr (kPrefix) {
        low[r] = r < job.rows ? p.row_min[int64_t(job.h) * (p.B * p.n) + job.r0 + r] : kInf;
      } else {
        const int i = job.r0 + r - job.lead;
        const float x = __shfl_sync(0xffffffffu, nw.low, i & 31);
        low[r] = i >= 0 && i < job.n_new ? x : kInf;
      }
    }
    if (job.t1 > job.t0) {
      float mid = job.t1 * 32 < job.end ? later_min(c, job.table, job.h, job.t1 * 32, job.end) : kInf;
      for (int tile = job.t1 - 1; tile >= job.t0; --tile) {
        const int64_t base = slot_of(c, job.table, job.h, tile * 32);
        const int lim = base < 0 ? 0 : min(32, job.end - tile * 32);
        const bool ok = lane < lim;
        const float phi = ok ? c.phi[base + lane] : kInf, psi = ok ? c.psi[base + lane] : 0.f;
        float f = p.scale2, lv = ok ? 0.f : -kInf, rv = 1.f;
        if (kInt8 && ok) {
          const float v = fmaxf(c.vs[base + lane], 0x1p-90f);
          f *= c.ks[base + lane];
          lv = lg2(v);
          rv = 1.f / v;
        }
        float all;
        const float suf = fminf(suffix_min(phi, all), mid);
        mid = fminf(mid, all);
        const float a = fminf(suf - psi, 0.f);
#pragma unroll
        for (int first = 0; first < 32; first += 8) scores(c, first + g < lim ? base + first + g : -1, first);
        __syncwarp();
        accumulate(
            c, f, lv, rv, lim, [&](int r) { return ok ? job.bias * fminf(a, low[r] - psi) : 0.f; },
            [&](int k) { return base + k; });
      }
    }
    if constexpr (!kPrefix) {
      if (job.last && job.n_new > 0) {
#pragma unroll
        for (int first = 0; first < 32; first += 8) {
          const int64_t at = __shfl_sync(0xffffffffu, nw.slot, first + g);
          scores(c, at, first);
        }
        __syncwarp();
        float f = p.scale2, lv = nw.slot >= 0 ? 0.f : -kInf, rv = 1.f;
        if (kInt8 && nw.slot >= 0) {
          const float v = fmaxf(c.vs[nw.slot], 0x1p-90f);
          f *= c.ks[nw.slot];
          lv = lg2(v);
          rv = 1.f / v;
        }
        accumulate(
            c, f, lv, rv, job.n_new,
            [&](int r) {
              const int i = job.r0 + r - job.lead;
              const float x = new_pair(nw, lane, i);
              return lane <= i ? job.bias * x : -kInf;
            },
            [&](int k) { return slot_of(c, job.table, job.h, job.end + k); });
      }
    }
  }

  __device__ __forceinline__ void store(float* sm, float* sl, float* sO, int rows) {
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      float x = l[r];
#pragma unroll
      for (int o_ = 16; o_ > 0; o_ >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o_);
      if constexpr (KG > 1) {
#pragma unroll
        for (int o_ = D; o_ < 32; o_ <<= 1) o[r][0] += __shfl_xor_sync(0xffffffffu, o[r][0], o_);
      }
      if (r < rows) {
        if (lane == 0) {
          sm[r] = m[r];
          sl[r] = x;
        }
#pragma unroll
        for (int j = 0; j < CPL; ++j) sO[r * D + (D < 32 ? (lane & (D - 1)) : column(j))] = o[r][j];
      }
    }
  }
};

template <bool kInt8>
cudaError_t launch_for(const DecodeParams& p, bool prefix, cudaStream_t s) {
  const int rows = prefix ? p.B * p.n : p.n;
  switch (p.c.D) {
#define FPA_CASE(D)                                                                                  \
  case D:                                                                                            \
    return rows == 1  ? launch_decode_core<FfmaCore<D, kInt8, 1>>(p, prefix, s)              \
           : rows < 5 ? launch_decode_core<FfmaCore<D, kInt8, 4>>(p, prefix, s)              \
                      : launch_decode_core<FfmaCore<D, kInt8, 8>>(p, prefix, s);
    FPA_CASE(16)
    FPA_CASE(32)
    FPA_CASE(64)
    FPA_CASE(128)
    FPA_CASE(256)
#undef FPA_CASE
    default:
      return cudaErrorInvalidValue;
  }
}

// row_min[h][b * n + r]: minimum of phi over the sequence's own tokens up to row r. A warp per (sequence, head).
__global__ void __launch_bounds__(128) row_min_kernel(const __grid_constant__ DecodeParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int i = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (i >= p.B * p.c.H) return;
  const int b = i / p.c.H, h = i - b * p.c.H;
  const int32_t* table = p.table + b * p.table_stride;
  const int cap = int(min(int64_t(p.max_pages) << p.c.page_shift, int64_t(INT32_MAX)));
  const int L = min(max(p.lengths[b], 0), cap), Lb = max(L - p.n, 0), nn = L - Lb, lead = p.n - nn;
  const int pid = lane < nn ? table[(Lb + lane) >> p.c.page_shift] : -1;
  LaterMin own;
  own.ids(p.c, table, 0, Lb);
  NewTokens nw = load_new(p.c, pid, h, Lb, nn);
  own.values(p.c, h);
  nw.low = prefix_min(nw.phi);
  const float before = own.finish(p.c, table, h);
  if (lane < p.n) {
    float* out = p.row_min + int64_t(h) * (p.B * p.n) + b * p.n;
    if (lane < lead) out[lane] = kInf;
    if (lane < nn) out[lead + lane] = fminf(before, nw.low);
  }
}

}  // namespace

cudaError_t launch_decode_ffma(const DecodeParams& p, bool int8, bool prefix, cudaStream_t s) {
  return int8 ? launch_for<true>(p, prefix, s) : launch_for<false>(p, prefix, s);
}

cudaError_t launch_row_min(const DecodeParams& p, cudaStream_t s) {
  return launch_pdl(row_min_kernel, dim3((p.B * p.c.H + 3) / 4), dim3(128), 0, s, p);
}

}  // namespace fpa
