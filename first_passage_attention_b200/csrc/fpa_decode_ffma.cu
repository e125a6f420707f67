// Decode attention in float32 (FFMA), over a float32 or int8 cache, and the minima that a prefix pass needs.
//
// A warp takes 32 keys at a time. Scores: lane (g, t) = (lane / 4, lane % 4) holds a quarter of key g of eight, in
// runs of four elements that the four lanes of a key read side by side; two shuffles finish a product. The softmax has
// one key per lane, and the product with V one run of D / 32 columns per lane, P coming from shared memory four keys
// at a time. K and V come through a ring of the warp's own, eight rows to a stage, filled by cp.async kStages - 1 stages
// ahead; rows are padded so that the lanes of a key and of its neighbour read different banks. Everything is float32:
// this is the path of float32 models, whose tolerance rules out fp16 operands.
//
// What bounds it: for several rows the latency of shared memory, not FFMA: a float4 of a query serves four products and a
// row's product ends in two shuffles for every eight keys. 8 rows of 8 x 8 pairs of up to 4096 tokens of 64 take 65 us, 4.4
// times their bytes, with 9 warps on an SM, 27 % of the issue slots, 29 % of the shared-memory pipe and 17 % of the HBM rate
// busy; the first stalls are waits for shared memory. Short calls (8 x 8 pairs of up to 1000 tokens of 32, 3 rows, 13 us): one
// look-up more in series than the fp16 kernel at the start, one tile a warp, and the join of 32 states.
#include "fpa_decode.cuh"

namespace fpa {
namespace {

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

template <int D_, bool kInt8, int NR>
struct FfmaCore {
  static constexpr int D = D_, NQ = NR, kKeys = 32;
  static constexpr int CPL = D < 32 ? 1 : D / 32;   // columns of V for a lane
  static constexpr int CV = CPL < 4 ? CPL : 4;      // ... side by side
  static constexpr int KG = D < 32 ? 32 / D : 1;    // lanes that share a column take every KG-th key
  static constexpr int RB = kInt8 ? D : 4 * D;      // bytes of a row
  static constexpr int kPitch = RB + (kInt8 ? 16 : D < 32 ? 0 : 64);
  static constexpr int kStage = 8 * kPitch;         // eight rows of K or of V
  static constexpr int kStages = kStage <= 2560 ? 6 : kStage <= 4608 ? 5 : 2;  // so that at least two CTAs fit an SM
  static constexpr int kRingBytes = kStages * kStage;
  static constexpr int kMinBlocks = NR * CPL + D / 4 <= 64 ? 4 : 2;
  static constexpr int kCtaFloats = NR * D;
  static constexpr int kScores = NR * 32, kSlots = 64;  // probabilities; the new tokens' pool indices (int64)
  static constexpr int kWarpFloats = kScores + kSlots + kMaxNew * kMaxNew;
  static constexpr int kManyBlocks = NR * D >= 512 ? 2 : 16;  // a block of many products outweighs a start-up sooner
  using Out = float;
  static_assert(kStages <= 8, "at most one tile ahead");

  float o[NR][CPL], m[NR], l[NR];
  float* qs;         // [NR][D]
  float* ss;         // [NR][32], this warp's scores and probabilities
  int64_t* slots;    // [32]
  float* pairs;      // [kMaxNew][kMaxNew]
  char* ring_ptr;
  uint32_t ring;
  int lane, g, t;

  __device__ __forceinline__ FfmaCore(const DecodeParams&, const Job&, float* scratch, char* rings) {
    lane = threadIdx.x & 31;
    g = lane >> 2;
    t = lane & 3;
    qs = scratch;
    ss = scratch + kCtaFloats + (threadIdx.x >> 5) * kWarpFloats;
    slots = reinterpret_cast<int64_t*>(ss + kScores);
    pairs = ss + kScores + kSlots;
    ring_ptr = rings + (threadIdx.x >> 5) * kRingBytes;
    ring = static_cast<uint32_t>(__cvta_generic_to_shared(ring_ptr));
  }

  __device__ __forceinline__ static int column(int j) { return (j / CV * 32 + (threadIdx.x & 31)) * CV + j % CV; }

  // Four elements d .. d + 3 of a row in shared memory (codes for int8).
  __device__ __forceinline__ static float4 load4(const char* row, int d) {
    if constexpr (kInt8) {
      const uchar4 x = *reinterpret_cast<const uchar4*>(row + d);
      return make_float4(x.x - 128, x.y - 128, x.z - 128, x.w - 128);
    } else {
      return *reinterpret_cast<const float4*>(row + 4 * d);
    }
  }

  // V of one row, this lane's columns.
  __device__ __forceinline__ static void load_v(const char* row, float (&v)[CPL]) {
    if constexpr (CV == 4) {
#pragma unroll
      for (int j = 0; j < CPL; j += 4) {
        const float4 x = load4(row, column(j));
        v[j] = x.x, v[j + 1] = x.y, v[j + 2] = x.z, v[j + 3] = x.w;
      }
    } else if constexpr (CV == 2) {
      const int d = column(0);
      if constexpr (kInt8) {
        const uchar2 x = *reinterpret_cast<const uchar2*>(row + d);
        v[0] = x.x - 128, v[1] = x.y - 128;
      } else {
        const float2 x = *reinterpret_cast<const float2*>(row + 4 * d);
        v[0] = x.x, v[1] = x.y;
      }
    } else {
      const int d = threadIdx.x & (D < 32 ? D - 1 : 31);
      v[0] = kInt8 ? float(static_cast<unsigned char>(row[d])) - 128.f : reinterpret_cast<const float*>(row)[d];
    }
  }

  // Eight rows into stage i: row r at pool index slot(r), zeros where that is negative.
  template <class Slot>
  __device__ __forceinline__ void fetch(const void* pool, int i, Slot slot) {
    const uint32_t st = ring + (i % kStages) * kStage;
    constexpr int kChunks = RB / 16;
#pragma unroll
    for (int e0 = 0; e0 < 8 * kChunks; e0 += 32) {
      const int e = e0 + lane, r = e / kChunks, c = e % kChunks;
      if (8 * kChunks < 32 && e >= 8 * kChunks) break;
      const int64_t at = slot(r);
      copy16(st + r * kPitch + c * 16, static_cast<const char*>(pool) + (at < 0 ? 0 : at) * RB + c * 16, at >= 0);
    }
  }

  // Scores of the eight keys in stage i into columns first .. first + 7.
  __device__ __forceinline__ void scores(int i, int first) {
    const char* row = ring_ptr + (i % kStages) * kStage + g * kPitch;
    float4 k[D / 16];
#pragma unroll
    for (int j = 0; j < D / 16; ++j) k[j] = load4(row, (j * 4 + t) * 4);
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

  // Softmax of one key per lane: z = ss[r][lane] f + bias(r) + lv; no key where lv (or the bias) is -inf.
  template <class Bias>
  __device__ __forceinline__ void softmax(float f, float lv, float rv, Bias bias) {
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
  }

  // O += P V of the eight keys in stage i, columns first .. first + 7 of P.
  __device__ __forceinline__ void values(int i, int first) {
    const char* rows = ring_ptr + (i % kStages) * kStage;
    if constexpr (KG > 1) {
#pragma unroll
      for (int k0 = 0; k0 < 8; k0 += KG) {
        const int k = k0 + lane / D;
        float v[CPL];
        load_v(rows + k * kPitch, v);
#pragma unroll
        for (int r = 0; r < NR; ++r) o[r][0] = fmaf(ss[r * 32 + first + k], v[0], o[r][0]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; k += 4) {
        float v[4][CPL];
#pragma unroll
        for (int j = 0; j < 4; ++j) load_v(rows + (k + j) * kPitch, v[j]);
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          const float4 e = *reinterpret_cast<const float4*>(ss + r * 32 + first + k);
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
  }

  // The same for the newest tokens, n of them in the tile. Some rows do not see all of these keys: what they do not see stays
  // out of their sums even where it is not finite.
  __device__ __forceinline__ void values_new(int i, int first, int n) {
    const char* rows = ring_ptr + (i % kStages) * kStage;
#pragma unroll 1
    for (int k0 = 0; k0 < min(8, n - first); k0 += KG) {
      const int k = k0 + (KG > 1 ? lane / D : 0);
      float v[CPL];
      load_v(rows + k * kPitch, v);
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const float e = ss[r * 32 + first + k];
#pragma unroll
        for (int j = 0; j < CPL; ++j) o[r][j] = e == 0.f ? o[r][j] : fmaf(e, v[j], o[r][j]);
      }
    }
  }

  template <bool kPrefix>
  __device__ __forceinline__ void run(const DecodeParams& p, const Job& job) {
    const CacheView& c = p.c;
    // The run: history tiles from the latest to the earliest, then the newest tokens' tile. Stages 8 k .. 8 k + 3 hold
    // K of tile k, 8 k + 4 .. 8 k + 7 its V, eight rows each.
    const int history = job.t1 - job.t0, total = history + (job.last ? 1 : 0);
    int64_t base = -1;   // of the tile being fetched
    int lim = 0;
    float phi = kInf, psi = 0.f, ks = 0.f, vs = 0.f;  // this lane's key of the tile being fetched
    auto fetch_stage = [&](int i) {
      const int tile = i >> 3, part = i & 7;
      const void* pool = part < 4 ? c.k : c.v;
      const int first = (part & 3) * 8;
      if (tile < history) {
        if (part == 0) {
          const int at = (job.t1 - 1 - tile) * kKeys;
          base = slot_of(c, job.table, job.h, at);
          lim = base < 0 ? 0 : min(kKeys, job.end - at);
          phi = kInf, psi = ks = vs = 0.f;
          if (lane < lim) {
            phi = c.phi[base + lane];
            psi = c.psi[base + lane];
            if (kInt8) {
              ks = c.ks[base + lane];
              vs = c.vs[base + lane];
            }
          }
        }
        fetch(pool, i, [&](int r) { return first + r < lim ? base + first + r : int64_t(-1); });
      } else if (tile < total) {
        fetch(pool, i, [&](int r) { return slots[first + r]; });
      }
    };
    LaterMin later;
    later.ids(c, job.table, job.t1 * kKeys, history > 0 ? job.end : 0);
    NewTokens nw{kInf, 0.f, kInf, -1, 0};
    if constexpr (!kPrefix)
      nw = load_new(c, lane < job.n_new ? job.table[(job.end + lane) >> c.page_shift] : -1, job.h, job.end, job.n_new);
    later.values(c, job.h);
    slots[lane] = nw.slot;
    __syncwarp();
#pragma unroll 1
    for (int i = 0; i < kStages - 1; ++i) {
      fetch_stage(i);
      copy_commit();
    }
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
    nw.low = prefix_min(nw.phi);
    fill_pairs(nw, pairs);
    __syncthreads();
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
    float mid = later.finish(c, job.table, job.h);
    auto next = [&](int i) {
      // Stage i has landed; the one before it is free for what comes kStages - 1 later.
      copy_wait<kStages - 2>();
      __syncwarp();
      fetch_stage(i + kStages - 1);
      copy_commit();
    };
    for (int k = 0; k < total; ++k) {
      // The tile's field, before the fetches go on to the next tile's.
      // (A single row has no such tile: its own key is the history's last.)
      const bool fresh = NR > 1 && k >= history, ok = fresh ? nw.slot >= 0 : lane < lim;
      float f_phi = phi, f_psi = psi, f_ks = ks, f_vs = vs;
      if (fresh) {
        f_ks = f_vs = 0.f;
        if (kInt8 && ok) {
          f_ks = c.ks[nw.slot];
          f_vs = c.vs[nw.slot];
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        next(8 * k + j);
        scores(8 * k + j, j * 8);
      }
      __syncwarp();
      float f = p.scale2, lv = ok ? 0.f : -kInf, rv = 1.f;
      if (kInt8 && ok) {
        const float v = fmax_nan(f_vs, 0x1p-90f);
        f *= f_ks;
        lv = lg2(v);
        rv = v != v ? 1.f : 1.f / v;  // NaN reaches the rows that see the key through lv, and no other
      }
      if (!fresh) {
        float all;
        const float suf = fminf(suffix_min(ok ? f_phi : kInf, all), mid);
        mid = fminf(mid, all);
        const float a = fminf(suf - f_psi, 0.f);
        softmax(f, lv, rv, [&](int r) { return ok ? job.bias * fminf(a, low[r] - f_psi) : 0.f; });
      } else {
        softmax(f, lv, rv, [&](int r) {
          const int i = job.r0 + r - job.lead;
          return lane <= i && i < job.n_new ? job.bias * pairs[lane * kMaxNew + i] : -kInf;
        });
      }
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        next(8 * k + 4 + j);
        if (fresh)
          values_new(8 * k + 4 + j, j * 8, job.n_new);
        else
          values(8 * k + 4 + j, j * 8);
      }
    }
    copy_wait<0>();
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

template <int D, bool kInt8>
cudaError_t launch_groups(const DecodeParams& p, bool prefix, cudaStream_t s, int& launches) {
  const int group = ffma_group(D, prefix ? p.B * p.n : p.n);
  if (group == 1) return launch_decode_core<FfmaCore<D, kInt8, 1>>(p, prefix, s, launches);
  if constexpr (D <= 64) {
    if (group == 8) return launch_decode_core<FfmaCore<D, kInt8, 8>>(p, prefix, s, launches);
  }
  return launch_decode_core<FfmaCore<D, kInt8, 4>>(p, prefix, s, launches);
}

template <bool kInt8>
cudaError_t launch_for(const DecodeParams& p, bool prefix, cudaStream_t s, int& launches) {
  switch (p.c.D) {
    case 16: return launch_groups<16, kInt8>(p, prefix, s, launches);
    case 32: return launch_groups<32, kInt8>(p, prefix, s, launches);
    case 64: return launch_groups<64, kInt8>(p, prefix, s, launches);
    case 128: return launch_groups<128, kInt8>(p, prefix, s, launches);
    case 256: return launch_groups<256, kInt8>(p, prefix, s, launches);
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
  const int cap = int(min(int64_t(p.max_pages) << p.c.page_shift, int64_t(kMaxPositions)));
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

cudaError_t launch_decode_ffma(const DecodeParams& p, bool int8, bool prefix, cudaStream_t s, int& launches) {
  return int8 ? launch_for<true>(p, prefix, s, launches) : launch_for<false>(p, prefix, s, launches);
}

cudaError_t launch_row_min(const DecodeParams& p, cudaStream_t s) {
  return launch_pdl(row_min_kernel, dim3((p.B * p.c.H + 3) / 4), dim3(128), 0, s, p);
}

}  // namespace fpa
