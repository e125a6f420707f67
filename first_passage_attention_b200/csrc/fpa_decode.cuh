// Attention of the newest tokens over the paged cache: the parts that the tensor-core and the FFMA kernels share.
//
// Row r of a sequence of L tokens stands at t = L - n + r and sees the keys s <= t with the logits
//     z_ts = q_t k_s / sqrt(D) + beta min(0, min_{s<u<=t} phi_u - psi_s),   z_tt without the bias.
// With Lb = L - n, the range minimum of a history key s < Lb splits into SUF_s = min_{s<u<Lb} phi_u, which all rows
// share, and M_r = min_{Lb<=u<=t} phi_u, so the bias is beta min(a_s, M_r - psi_s) with a_s = min(0, SUF_s - psi_s);
// the pairs among the n newest tokens get their minimum one by one (with n = 1 the row's own key joins the history as
// its last: the empty range leaves it no bias). A prefix shared by the batch is the same thing once
// more: its keys' SUF ends at the prefix's end and M_r is the minimum over the row's own tokens.
//
// What bounds it: the bytes of the cache, and for short histories a chain of look-ups (length, table, values) of about
// 2 us. A CTA of up to four warps takes a (sequence, head, row group) or, as one of up to 8 CTAs of a cluster, a part
// of its history; every warp walks its own consecutive run of 16- or 32-key blocks from the latest
// to the earliest, so that SUF is a running minimum that the warp carries in a register, and no warp waits for
// another until the end. What lies after a warp's run enters through the page minima (phi_min), four bytes a page and
// head. The softmax states (m, l, O) of the warps join in shared memory, those of the cluster's CTAs through
// distributed shared memory: no atomics, a fixed order, one launch (two where a last round would stay mostly empty).
//
// On a B200, whole calls in a graph: 4 x 16 pairs of up to 16383 fp16 tokens of 128, 5 rows, 65 us, 5.5 TB/s; 64 x 12 of up to
// 2048 tokens of 64, one row, over the same lengths in fp16 45.6 us, 6.0 TB/s, and in int8 32.7 us, 4.5 TB/s; 12 heads of
// 1000 fp16 tokens 6.7 us; float32, 8 x 8 of up to 1000 tokens of 32, 3 rows, 13 us.
#pragma once

#include "fpa_serve.h"

namespace fpa {

constexpr int kMaxWarps = 4;     // of a CTA
constexpr int kMinSorted = 16, kMaxSorted = 64;  // sequences that a launch puts in the order of their lengths

// Index of slot `pos` of head h in the pool's [n_pages, H, page_size] arrays, given its page's id, or -1 where the id
// lies outside the pool (recorded in the status word).
__device__ __forceinline__ int64_t slot_in(const CacheView& c, int pid, int h, int pos) {
  if (unsigned(pid) >= unsigned(c.n_pages)) {
    report_bad_page(c.status, kSiteDecode);
    return -1;
  }
  return ((int64_t(pid) * c.H + h) << c.page_shift) + (pos & ((1 << c.page_shift) - 1));
}
__device__ __forceinline__ int64_t slot_of(const CacheView& c, const int32_t* table, int h, int pos) {
  return slot_in(c, table[pos >> c.page_shift], h, pos);
}

// phi of a position whose page's id is given; 0 where that lies outside the pool or phi is not finite. What M and psi are
// counted from where they are scaled apart from each other: the walk may stand anywhere, the bias is made of differences.
__device__ __forceinline__ float level_at(const CacheView& c, int pid, int h, int pos) {
  if (unsigned(pid) >= unsigned(c.n_pages)) return 0.f;
  const float x = c.phi[((int64_t(pid) * c.H + h) << c.page_shift) + (pos & ((1 << c.page_shift) - 1))];
  return fabsf(x) < kInf ? x : 0.f;
}

// The warp's minimum of phi over the positions [from, to) of a sequence: whole pages through phi_min, the rest from
// phi itself. In three steps, so that the table's entries, and then the values, of this and of the caller's other
// look-ups travel together.
struct LaterMin {
  int from, to, e1, e2, p0, p1;  // [from, e1) of a first page, pages p0 .. p1 - 1, [e2, to) of a last page
  int pid_a, pid_p, pid_z;
  float x;

  __device__ __forceinline__ void ids(const CacheView& c, const int32_t* table, int from_, int to_) {
    const int lane = threadIdx.x & 31, page = 1 << c.page_shift;
    from = from_;
    to = max(from_, to_);
    e1 = min(to, (from + page - 1) & -page);
    p0 = e1 >> c.page_shift;
    p1 = max(p0, to >> c.page_shift);
    e2 = max(e1, p1 << c.page_shift);
    pid_a = from < e1 ? table[from >> c.page_shift] : -1;
    pid_p = p0 + lane < p1 ? table[p0 + lane] : -1;
    pid_z = e2 < to ? table[e2 >> c.page_shift] : -1;
  }
  __device__ __forceinline__ static float part(const CacheView& c, int pid, int h, int s0, int s1) {
    float x = kInf;
    if (unsigned(pid) < unsigned(c.n_pages)) {
      const float* f = c.phi + ((int64_t(pid) * c.H + h) << c.page_shift);
      for (int s = s0 + (threadIdx.x & 31); s < s1; s += 32) x = fminf(x, f[s & ((1 << c.page_shift) - 1)]);
    }
    return x;
  }
  __device__ __forceinline__ void values(const CacheView& c, int h) {
    x = unsigned(pid_p) < unsigned(c.n_pages) ? c.pmin[int64_t(pid_p) * c.H + h] : kInf;
    x = fminf(x, fminf(part(c, pid_a, h, from, e1), part(c, pid_z, h, e2, to)));
  }
  __device__ __forceinline__ float finish(const CacheView& c, const int32_t* table, int h) {
#pragma unroll 4
    for (int pg = p0 + 32 + (threadIdx.x & 31); pg < p1; pg += 32) {
      const int pid = table[pg];
      if (unsigned(pid) < unsigned(c.n_pages)) x = fminf(x, c.pmin[int64_t(pid) * c.H + h]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x = fminf(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
  }
};
__device__ __forceinline__ float later_min(const CacheView& c, const int32_t* table, int h, int from, int to) {
  LaterMin m;
  m.ids(c, table, from, to);
  m.values(c, h);
  return m.finish(c, table, h);
}

// Minimum over the lanes' x of the lanes strictly after this one (+inf for lane 31); `all` gets the warp's minimum.
__device__ __forceinline__ float suffix_min(float x, float& all) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const float y = __shfl_down_sync(0xffffffffu, x, o);
    if (lane + o < 32) x = fminf(x, y);
  }
  all = __shfl_sync(0xffffffffu, x, 0);
  const float y = __shfl_down_sync(0xffffffffu, x, 1);
  return lane < 31 ? y : kInf;
}

// Running minimum over the lanes up to and including this one.
__device__ __forceinline__ float prefix_min(float x) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const float y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x = fminf(x, y);
  }
  return x;
}

// The newest tokens of a sequence, one per lane (lanes >= nn hold nothing).
struct NewTokens {
  float phi, psi;  // +inf, 0 on the empty lanes
  float low;       // min of phi over the new tokens up to this lane's (filled by the caller: prefix_min(phi))
  int64_t slot;    // pool index, or -1
  int nn;
};

__device__ __forceinline__ NewTokens load_new(const CacheView& c, int pid, int h, int Lb, int nn) {
  const int lane = threadIdx.x & 31;
  NewTokens t{kInf, 0.f, kInf, -1, nn};
  if (lane < nn) t.slot = slot_in(c, pid, h, Lb + lane);
  if (t.slot >= 0) {
    t.phi = c.phi[t.slot];
    t.psi = c.psi[t.slot];
  }
  return t;
}

// The newest tokens' pairs: table[j * kMaxNew + i] = min(0, min_{j<u<=i} phi_u - psi_j) for j < i, 0 for j == i. Lane j
// fills row j with a running minimum.
__device__ __forceinline__ void fill_pairs(const NewTokens& t, float* table) {
  const int lane = threadIdx.x & 31;
  float m = kInf;
  for (int i = 0; i < t.nn; ++i) {
    const float f = __shfl_sync(0xffffffffu, t.phi, i);
    if (i > lane) m = fminf(m, f);
    if (lane < t.nn) table[lane * kMaxNew + i] = fminf(m - t.psi, 0.f);
  }
  __syncwarp();
}

// The sequence of rank r when the batch is ordered by falling length (to one part in 32 of cap; equal ones in the
// batch's order), the same in every warp of the grid. The rank's length is found bit by bit, by counting.
__device__ __forceinline__ int by_length(const int32_t* lengths, int B, int r, int cap) {
  const int lane = threadIdx.x & 31;
  const int shift = max(0, 27 - __clz(cap));
  int x[kMaxSorted / 32];
#pragma unroll
  for (int i = 0; i < kMaxSorted / 32; ++i)
    x[i] = i * 32 + lane < B ? min(max(lengths[i * 32 + lane], 0), cap) >> shift : -1;
  int at = 0;  // largest value that more than r sequences reach
#pragma unroll
  for (int bit = 16; bit > 0; bit >>= 1) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < kMaxSorted / 32; ++i) n += __popc(__ballot_sync(0xffffffffu, x[i] >= at + bit));
    if (n > r) at += bit;
  }
#pragma unroll
  for (int i = 0; i < kMaxSorted / 32; ++i) r -= __popc(__ballot_sync(0xffffffffu, x[i] > at));
  int b = 0;
#pragma unroll
  for (int i = 0; i < kMaxSorted / 32; ++i) {
    const unsigned m = __ballot_sync(0xffffffffu, x[i] == at);
    const unsigned who = __ballot_sync(0xffffffffu, x[i] == at && __popc(m & ((1u << lane) - 1)) == r);
    if (who) b = i * 32 + __ffs(who) - 1;
    r -= __popc(m);
  }
  return __reduce_max_sync(0xffffffffu, b);  // the same in every lane, and known to be
}

// What one CTA works on.
struct Job {
  const int32_t* table;
  int h, b;
  int rows;           // rows of this group
  int r0;             // first row: of the sequence's n (decode) or of the head's R (prefix)
  int end;            // history keys [0, end)
  int t0, t1;         // this warp's blocks of Core::kKeys keys
  int n_new;          // new tokens in the cache (decode)
  int lead;           // rows of the sequence that stand before its first token
  bool last;          // this warp also takes the tile of the new tokens
  float bias;         // beta log2(e)
};

__device__ __forceinline__ uint32_t cluster_addr(const void* p, int rank) {
  uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(p)), r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}
__device__ __forceinline__ float cluster_ld(uint32_t addr) {
  float x;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(addr) : "memory");
  return x;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// Weight of a softmax state with maximum m in a joint one with maximum M (0 for an empty state).
__device__ __forceinline__ float state_weight(float m, float M) { return m == -kInf ? 0.f : ex2(m - M); }

// Dynamic shared memory of a CTA: the warps' rings, whose place the joining of their states takes over at the end;
// the cores' scratch, of the CTA and of each warp; the states' maxima and sums.
template <class Core>
__host__ __device__ constexpr int decode_warp_bytes() {
  return Core::kRingBytes > Core::NQ * Core::D * 4 ? Core::kRingBytes : Core::NQ * Core::D * 4;
}
template <class Core>
__host__ __device__ constexpr int decode_smem_bytes(int warps) {
  return warps * decode_warp_bytes<Core>() +
         (Core::kCtaFloats + warps * (Core::kWarpFloats + 2 * Core::NQ) + 2 * Core::NQ) * 4;
}

// Core: the arithmetic of one warp over a run of keys (see fpa_decode_mma.cu, fpa_decode_ffma.cu).
// kPrefix: the rows (b, i) of the whole batch against the prefix, partial results to the workspace.
// kSorted: the batch's sequences in the order of their lengths, the longest first.
template <class Core, bool kPrefix, bool kSorted>
__global__ void __launch_bounds__(kMaxWarps * 32, Core::kMinBlocks) decode_kernel(const __grid_constant__ DecodeParams p) {
  extern __shared__ __align__(128) float smem[];
  constexpr int NQ = Core::NQ, D = Core::D;
  const int W = blockDim.x >> 5;
  float* sO = smem;                 // [W][NQ][D]
  float* scratch = smem + W * (decode_warp_bytes<Core>() / 4);
  float* sm = scratch + Core::kCtaFloats + W * Core::kWarpFloats;  // [W][NQ]
  float* sl = sm + W * NQ;          // [W][NQ]
  float* cm = sl + W * NQ;          // [NQ]
  float* cl = cm + NQ;              // [NQ]
  const int warp = threadIdx.x >> 5;
  const int S = gridDim.x, rank = blockIdx.x;
  // A prefix pass before this kernel has waited for everything before it, so only its own results are still open:
  // the wait then moves to where they are read.
  const bool behind = !kPrefix && p.prefix_len > 0;
  // The same holds for a second launch behind the first one, which has waited too (or is late itself, behind a prefix
  // pass that has); its wait at the end leaves whatever comes after this launch behind both.
  const bool late = !kPrefix && (behind || p.follows);
  if (!late) pdl_wait();
  if (!late || p.followed) pdl_launch_dependents();
  Job job;
  int R = p.n;
  if constexpr (kPrefix) {
    job.h = blockIdx.z;
    job.b = 0;
    job.table = p.prefix_table;
    job.end = p.prefix_len;
    job.n_new = 0;
    job.lead = 0;
    job.r0 = blockIdx.y * NQ;
    R = p.B * p.n;
  } else {
    job.h = blockIdx.y / p.groups;
    job.r0 = (blockIdx.y - job.h * p.groups) * NQ;
    const int cap = int(min(int64_t(p.max_pages) << p.c.page_shift, int64_t(kMaxPositions)));
    job.b = kSorted ? by_length(p.lengths, p.B, p.first + blockIdx.z, cap) : p.first + blockIdx.z;
    job.table = p.table + job.b * p.table_stride;
    int L = p.lengths[job.b];
    if (L < 0 || L > cap) {
      report_bad_page(p.c.status, kSiteDecode);
      L = min(max(L, 0), cap);
    }
    job.end = max(L - p.n, 0);
    job.n_new = L - job.end;
    job.lead = p.n - job.n_new;
    if (p.n == 1) {
      // One row: its own key is the last of the history, whose empty range leaves no bias.
      job.end = L;
      job.n_new = 0;
    }
  }
  job.rows = min(NQ, R - job.r0);
  job.bias = p.beta[job.h] * kLog2e;
  {
    const int tiles = (job.end + Core::kKeys - 1) / Core::kKeys, units = S * W, u = rank * W + warp;
    const int each = tiles / units, more = tiles - each * units;
    job.t0 = u * each + min(u, more);
    job.t1 = job.t0 + each + (u < more ? 1 : 0);
    job.last = job.n_new > 0 && u == units - 1;
  }
  Core core(p, job, scratch, reinterpret_cast<char*>(smem));
  core.template run<kPrefix>(p, job);
  if (Core::kRingBytes > 0) __syncthreads();  // every warp is done with its ring
  core.store(sm + warp * NQ, sl + warp * NQ, sO + warp * NQ * D, job.rows);
  __syncthreads();
  // The CTA's state: maxima and sums per row, O in the first warp's place.
  if (int(threadIdx.x) < job.rows) {
    float M = -kInf, l = 0.f;
    for (int w = 0; w < W; ++w) M = fmaxf(M, sm[w * NQ + threadIdx.x]);
    for (int w = 0; w < W; ++w) l += sl[w * NQ + threadIdx.x] * state_weight(sm[w * NQ + threadIdx.x], M);
    cm[threadIdx.x] = M;
    cl[threadIdx.x] = l;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < job.rows * D; e += W * 32) {
    const int r = e / D;
    const float M = cm[r];
    float o = 0.f;
    for (int w = 0; w < W; ++w) o += sO[w * NQ * D + e] * state_weight(sm[w * NQ + r], M);
    if constexpr (kPrefix) {
      const int64_t at = (int64_t(job.h) * R + job.r0 + r) * p.chunks + rank;
      p.part_o[at * D + (e - r * D)] = o;
      if (e == r * D) {
        p.part_ml[at * 2] = M;
        p.part_ml[at * 2 + 1] = cl[r];
      }
    } else {
      sO[e] = o;
    }
  }
  if constexpr (!kPrefix) {
    if (late) pdl_wait();
    if (S > 1)
      cluster_barrier();
    else
      __syncthreads();
    using O = typename Core::Out;
    O* out = static_cast<O*>(p.o) + job.b * p.so.b + job.h * p.so.h;
    for (int e = rank * W * 32 + threadIdx.x; e < job.rows * D; e += S * W * 32) {
      const int r = e / D, d = e - r * D, row = job.r0 + r;
      float M = -kInf;
      const int64_t pre = ((int64_t(job.h) * p.B + job.b) * p.n + row) * p.chunks;
      for (int c = 0; c < S; ++c) M = fmaxf(M, S > 1 ? cluster_ld(cluster_addr(cm + r, c)) : cm[r]);
      if (behind)
        for (int c = 0; c < p.chunks; ++c) M = fmaxf(M, p.part_ml[(pre + c) * 2]);
      float l = 0.f, o = 0.f;
      for (int c = 0; c < S; ++c) {
        const float w = state_weight(S > 1 ? cluster_ld(cluster_addr(cm + r, c)) : cm[r], M);
        l += w * (S > 1 ? cluster_ld(cluster_addr(cl + r, c)) : cl[r]);
        o += w * (S > 1 ? cluster_ld(cluster_addr(sO + e, c)) : sO[e]);
      }
      if (behind)
        for (int c = 0; c < p.chunks; ++c) {
          const float w = state_weight(p.part_ml[(pre + c) * 2], M);
          l += w * p.part_ml[(pre + c) * 2 + 1];
          o += w * p.part_o[(pre + c) * D + d];
        }
      // Rows before the sequence's first token see nothing, nor does a row whose keys all lie in pages outside the pool.
      out[row * p.so.t + d * p.so.d] = from_f32<O>(row < job.lead || l == 0.f ? 0.f : o / l);
    }
    if (S > 1) cluster_barrier();  // the other CTAs have read this one's shared memory
  }
}

// Grid and launch of one pass. chunks (prefix): CTAs that share the prefix.
//
// CTAs of four warps for each (sequence, head, row group): 1, 2, 4 or 8 (a cluster), as many as run at once on the GPU. An
// eighth of the places is left free, since clusters do not fill the SMs of a GPC exactly: 72 units of 400 tokens, fp16 D =
// 128, three CTAs on an SM, take 8.3 us with 4 CTAs each, 14.2 with 6 (432 of 444 places), where some wait for a second
// round. Twice as many where every warp then still has kManyBlocks blocks: a second round evens out long work (64 units
// of 16383 tokens, 5 rows: 71 us with 4, 68 with 8).
//
// Where the CTAs do not all run at once, the batch goes in the order of its lengths, so that the short sequences come last
// (in the batch's order / sorted, lengths drawn evenly up to the given one): 64 x 12 pairs, 2048 tokens of 64, fp16 41.8 /
// 36.2 us, int8 32.3 / 33.4 and 34.0 / 32.9 in two drawings; 48 x 16, 4096 of 128, int8 79 / 62; the own parts of 64 x 12, 512 of
// 64, int8, behind a prefix 32.4 / 28.8 (whole call). Equal lengths pay for the search: 38.2 / 39.4 in fp16. Fewer than 16
// sequences gain nothing (12 x 16, 8000 of 128, fp16, 5 rows: 84.3 / 85.3), and more than 64 little (100 x 8, 1500 of 64:
// 24.6 / 23.9 when handed over in order).
//
// What a last, partly filled round holds goes in a launch of its own with up to four CTAs each, whose CTAs start as the
// first launch's end (one launch / two; table as wide as the lengths): 64 x 12, 2048 int8 tokens of 64, all of them 52.9 /
// 45.6 us, uneven 31.3 / 29.4; 40 x 12 in fp16 55.0 / 47.5 and 25.1 / 26.8; 28 x 16 of 128, fp16, 5 rows, 97 / 84 and 48.1 / 49.8. Not
// for short runs (64 x 12 of 512: 19.8 / 19.5 and 12.5 / 14.3) or many rounds (130 x 12: 87 / 79 and 48 / 51).
template <class Core>
cudaError_t launch_decode_core(DecodeParams p, bool prefix, cudaStream_t s, int& launches) {
  const int rows = prefix ? p.B * p.n : p.n;
  p.groups = (rows + Core::NQ - 1) / Core::NQ;
  const int64_t units = int64_t(p.c.H) * p.groups * (prefix ? 1 : p.B);
  const int64_t len = prefix ? p.prefix_len : int64_t(p.max_pages) << p.c.page_shift;
  const int64_t blocks = (len + Core::kKeys - 1) / Core::kKeys;
  const int W = int(blocks < kMaxWarps ? blocks : kMaxWarps);
  int splits = prefix ? p.chunks : 1;
  bool sorted = false;
  int rest = 0, rest_splits = 0;
  if (!prefix) {
    const int by_smem = (228 * 1024) / (decode_smem_bytes<Core>(W) + 1024);
    const int64_t places = int64_t(sm_count()) * (by_smem < Core::kMinBlocks ? by_smem : Core::kMinBlocks);
    while (splits < 8 && units * splits * 2 <= places * 7 / 8 && blocks >= int64_t(splits) * 2 * W) splits *= 2;
    if (splits < 8 && units * splits <= places && blocks >= int64_t(splits) * 2 * W * Core::kManyBlocks)
      splits *= 2;
    sorted = p.B >= kMinSorted && p.B <= kMaxSorted && units * splits > places;
    const int64_t each = int64_t(p.c.H) * p.groups, round = places / (each * splits);
    if (round > 0 && p.B > round && p.B <= kMaxSorted && blocks >= int64_t(splits) * W * 8) {
      rest = int(p.B % round);
      rest_splits = splits;
      while (rest_splits < 4 && each * rest * rest_splits * 2 <= places * 7 / 8) rest_splits *= 2;
      if (rest_splits == splits) rest = 0;
    }
  }
  const int smem = decode_smem_bytes<Core>(W);
  auto kernel = prefix ? decode_kernel<Core, true, false>
                       : sorted ? decode_kernel<Core, false, true> : decode_kernel<Core, false, false>;
  if (smem > 48 * 1024) {
    const cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
    if (e != cudaSuccess) return e;
  }
  auto launch = [&](int count, int splits_) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = prefix ? dim3(splits_, p.groups, p.c.H) : dim3(splits_, p.c.H * p.groups, count);
    cfg.blockDim = dim3(W * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (!prefix && splits_ > 1) {
      attr[1].id = cudaLaunchAttributeClusterDimension;
      attr[1].val.clusterDim.x = splits_;
      attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
      cfg.numAttrs = 2;
    }
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
    launches += e == cudaSuccess;
    return e;
  };
  if (rest > 0) {
    p.followed = true;
    const cudaError_t e = launch(p.B - rest, splits);
    if (e != cudaSuccess) return e;
    p.first = p.B - rest;
    p.followed = false;
    p.follows = true;
    return launch(rest, rest_splits);
  }
  return launch(p.B, splits);
}

}  // namespace fpa
