// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Draft i is accepted while u_i q_i(x_i) < p_i(x_i). With a drafts accepted, the next token is a sample of the
// normalised residual max(p_a - q_a, 0) (of p_a when all drafts were accepted, or when the residual vanishes): for noise
// e_v from the exponential distribution, argmax_v w_v / e_v has the distribution w / sum w, so the weights need no
// sum, and each score is one subtraction and one division, rounded once each: the token does not depend on how the
// vocabulary is cut up.
//
// Bound by the bytes of three rows of V per sequence, and by latency when sequences are few: a cluster of CTAs shares a
// sequence, every CTA finds `a` itself (a few gathers), takes a part of the vocabulary, four entries to a load and
// eight in flight per thread, and leaves its best (score, index) in shared memory, which all compare through distributed shared
// memory. A thread divides only where w > 0.999 best e, without which w / e cannot reach its best so far. The target's
// own scores are looked at in a second pass, in the rare case that the first finds nothing.
//
// On a B200, in a graph: 64 sequences of 50304 float32 entries, 7 drafts, 12.6 us, 3.1 TB/s (fp16 12.3); one sequence
// 6.1 us.
#include "fpa_serve.h"

namespace fpa {
namespace {

constexpr int kThreads = 512;
constexpr int kAhead = 2;  // fours of entries whose loads a thread has in flight

struct VerifyParams {
  const void* p;
  const void* q;
  int64_t pb, pt, qb, qt;
  const int64_t* draft;
  int64_t db, dt;
  const float* u;
  int64_t ub, ut;
  const float* noise;
  int64_t nb;
  const int32_t* lens;
  int32_t* accepted;
  int64_t* tokens;
  int n, V;
};

// The thread's best entry so far, as a key: scores are >= 0, so their bits order as they do; the complement of the index
// lets the lowest index win a tie. Entries come with rising index, so a later one never wins a tie here.
struct Best {
  float score;
  unsigned long long key;
  __device__ __forceinline__ void take(float w, float n, int v) {
    if (w > 0.f && !(w < score * n * 0.999f)) {
      const float s = __fdiv_rn(w, n);
      if (s > score || (key == 0 && s >= 0.f)) {
        score = s;
        key = (static_cast<unsigned long long>(__float_as_uint(s) + 1u) << 32) | (0xffffffffu - unsigned(v));
      }
    }
  }
};

// Four consecutive entries, 16 or 8 bytes.
__device__ __forceinline__ void load4(const float* p, float (&x)[4]) {
  const float4 v = *reinterpret_cast<const float4*>(p);
  x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}
__device__ __forceinline__ void load4(const __half* p, float (&x)[4]) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
  x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}

// Best of the row w = pr - qr (qr null: pr) over e; the thread is number `first` of `step`. Rows that start at multiples of
// four entries' bytes are read four at a time, their last V % 4 entries by the first threads; others one at a time.
template <typename T>
__device__ __forceinline__ unsigned long long scan_row(const T* pr, const T* qr, const float* e, int V, int first, int step) {
  Best best{0.f, 0};
  const uintptr_t at = reinterpret_cast<uintptr_t>(pr) | reinterpret_cast<uintptr_t>(qr);
  int v0 = 0;
  if (at % (4 * sizeof(T)) == 0 && reinterpret_cast<uintptr_t>(e) % 16 == 0) {
    v0 = V & ~3;
    for (int i0 = first * 4; i0 < v0; i0 += kAhead * step * 4) {
      float w[kAhead][4], q[kAhead][4], n[kAhead][4];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int v = i0 + i * step * 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[i][j] = q[i][j] = n[i][j] = 0.f;
        if (v < v0) {
          load4(pr + v, w[i]);
          load4(e + v, n[i]);
          if (qr) load4(qr + v, q[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) best.take(__fsub_rn(w[i][j], q[i][j]), n[i][j], i0 + i * step * 4 + j);
    }
  }
  for (int i0 = v0 + first; i0 < V; i0 += 4 * kAhead * step) {
    float w[4 * kAhead], n[4 * kAhead];
#pragma unroll
    for (int i = 0; i < 4 * kAhead; ++i) {
      const int v = i0 + i * step;
      w[i] = n[i] = 0.f;
      if (v < V) {
        w[i] = to_f32(pr[v]);
        n[i] = e[v];
        if (qr) w[i] = __fsub_rn(w[i], to_f32(qr[v]));
      }
    }
#pragma unroll
    for (int i = 0; i < 4 * kAhead; ++i) best.take(w[i], n[i], i0 + i * step);
  }
  return best.key;
}

// Best key of the block, in every thread; `red` holds one key per warp.
__device__ __forceinline__ unsigned long long block_best(unsigned long long k, unsigned long long* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = k;
  __syncthreads();
  k = (threadIdx.x & 31) < kThreads / 32 ? red[threadIdx.x & 31] : 0ull;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
  __syncthreads();
  return k;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) verify_kernel(const __grid_constant__ VerifyParams a) {
  __shared__ unsigned long long red[kThreads / 32], best[2];
  __shared__ int first;
  pdl_wait();
  pdl_launch_dependents();
  const int S = gridDim.x, rank = blockIdx.x, b = blockIdx.y;
  const T* P = static_cast<const T*>(a.p) + b * a.pb;
  const T* Q = static_cast<const T*>(a.q) + b * a.qb;
  const int n = a.lens ? min(max(a.lens[b], 0), a.n) : a.n;
  if (threadIdx.x < 32) {
    // The first refused draft: 32 at a time.
    int acc = n;
    for (int i0 = 0; i0 < n && acc == n; i0 += 32) {
      const int i = i0 + int(threadIdx.x);
      bool refuse = false;
      if (i < n) {
        const int64_t x = a.draft[b * a.db + i * a.dt];
        refuse = x < 0 || x >= a.V ||
                 !(__fmul_rn(a.u[b * a.ub + i * a.ut], to_f32(Q[i * a.qt + x])) < to_f32(P[i * a.pt + x]));
      }
      const unsigned m = __ballot_sync(0xffffffffu, refuse);
      if (m) acc = i0 + __ffs(m) - 1;
    }
    if (threadIdx.x == 0) first = acc;
  }
  __syncthreads();
  const int acc = first;
  const T* pr = P + acc * a.pt;
  const T* qr = acc < n ? Q + acc * a.qt : nullptr;  // all accepted: the target's own probabilities
  const float* e = a.noise + b * a.nb;
  // The best of the residual; where it is nowhere positive, of the target's probabilities.
  unsigned long long k = 0;
  for (int pass = 0; pass < 2; ++pass) {
    if (pass == 1) {
      if (k || !qr) break;  // the same in every thread of the cluster
      qr = nullptr;
    }
    k = block_best(scan_row(pr, qr, e, a.V, rank * kThreads + int(threadIdx.x), S * kThreads), red);
    if (S > 1) {
      if (threadIdx.x == 0) best[pass] = k;
      cluster_sync();
      k = 0;
      for (int c = 0; c < S; ++c) {
        uint32_t at;
        unsigned long long x;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(best + pass))), "r"(c));
        asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(x) : "r"(at) : "memory");
        k = max(k, x);
      }
      cluster_sync();
    }
  }
  if (rank == 0 && threadIdx.x < 32) {
    // Nothing positive anywhere (all zeros or NaN): the lowest index.
    const int64_t next = k ? int64_t(0xffffffffu - unsigned(k)) : 0;
    for (int i = threadIdx.x; i <= a.n; i += 32)
      a.tokens[int64_t(b) * (a.n + 1) + i] = i < acc ? a.draft[b * a.db + i * a.dt] : i == acc ? next : -1;
    if (threadIdx.x == 0) a.accepted[b] = acc;
  }
}

int invalid(const char* msg) {
  set_last_error(msg);
  return FPA_ERR_INVALID_ARGUMENT;
}

}  // namespace
}  // namespace fpa

using namespace fpa;

extern "C" FPA_API int fpa_verify(const FpaVerifyArgs* a, void* stream) {
  if (a == nullptr) return invalid("null argument block");
  if (a->dtype != FPA_DTYPE_F16 && a->dtype != FPA_DTYPE_F32) return invalid("fpa_verify: p and q must be fp16 or fp32");
  if (a->B <= 0 || a->n < 0 || a->V <= 0) return invalid("fpa_verify: B and V must be positive and n not negative");
  if (!a->p || !a->noise || !a->accepted || !a->tokens || (a->n > 0 && (!a->q || !a->draft || !a->u)))
    return invalid("fpa_verify: null tensor pointer");
  if (a->B > 65535) {
    set_last_error("fpa_verify: B above 65535 is not supported");
    return FPA_ERR_UNSUPPORTED;
  }
  VerifyParams p{a->p, a->q, a->p_stride[0], a->p_stride[1], a->q_stride[0], a->q_stride[1], a->draft, a->draft_stride[0],
                 a->draft_stride[1], a->u, a->u_stride[0], a->u_stride[1], a->noise, a->noise_stride, a->draft_lens,
                 a->accepted, a->tokens, a->n, a->V};
  // Up to 8 CTAs for a sequence, while all CTAs run at once (two on an SM) and every thread keeps an entry. For 64
  // sequences of 50304 entries, two waves of CTAs take 36 us.
  int S = 1;
  while (S < 8 && a->B * S <= sm_count() && S * kThreads < a->V) S *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(S, a->B);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = S;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = S > 1 ? 2 : 1;
  const cudaError_t e = a->dtype == FPA_DTYPE_F16 ? cudaLaunchKernelEx(&cfg, verify_kernel<__half>, p)
                                                  : cudaLaunchKernelEx(&cfg, verify_kernel<float>, p);
  if (e != cudaSuccess) {
    set_last_error(std::string("fpa_verify: ") + cudaGetErrorString(e));
    return FPA_ERR_CUDA;
  }
  return FPA_OK;
}
