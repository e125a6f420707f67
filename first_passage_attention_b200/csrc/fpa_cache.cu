// The paged cache: tokens quantised as they are written, and read back.
//
// Both are one pass over the data and bound by its bytes, short calls by a chain of look-ups. Eight elements of a row
// belong to one lane (16 bytes of fp16), D / 8 lanes to a row; a thread has the loads of several rows in flight. int8: the
// row's largest magnitude `top` by shuffles, scale = top / 127, code = rint((127 x) / top): for fp16 inputs 127 x is
// exact in float32 and the quotient of two 18- and 11-bit integers never comes closer to a half without being one than
// float32 resolves, so every code is the correctly rounded one. The quotient is taken as a product with 127 / top, which
// is off by less than 2^-14 for |quotient| <= 127, and as a division only where the product lies that close to a half.
// Rounding and conversion go through sums with 1.5 2^23 (codes sit in the sum's low bits): conversion instructions run
// at a quarter of the rate. Stored is code + 128. A block of the append owns one page of one (sequence, head): it alone
// writes the page's minimum of phi.
//
// On a B200: 8 x 16 (sequence, head) pairs of 16383 int8 tokens of 128 read back as fp16 in 230 us, 6.3 TB/s, and fp16 tokens
// (up to 16383) as they are in 316 us, 5.9 TB/s; 64 x 12 pairs of up to 2048 fp16 tokens of 64 appended as int8 in 184 us,
// 2.3 TB/s, where neither pipe is full (issue slots 54 %, HBM 26 % of nominal, 46 % of the warps): at this page size a block
// loads its rows once, converts them and stores them, and the wait for the loads is not covered; 4 x 16 of up to 16383 fp16
// tokens of 128 as they are in 183 us, 4.7 TB/s; 32 x 12 single tokens in 3.5 us.
#include "fpa_serve.h"
#include "fpa_sm100.cuh"

namespace fpa {
namespace {

constexpr int kReadThreads = 128;
constexpr int kMaxThreads = 256;
constexpr int kAhead = 4;  // rows whose loads a thread has in flight

// Codes + 128 of eight elements of type T from their row's largest magnitude, four to a word.
template <typename T>
__device__ __forceinline__ uint2 encode8(const float (&x)[8], float top) {
  constexpr float kRound = 12582912.f + 128.f;  // 1.5 2^23: a sum with it is rounded to an integer, even on ties
  const float k = 127.f * rcp_approx_f(top);
  uint32_t w[8];
  float off = 0.f;  // largest distance from an integer
  const float2 k2 = make_float2(k, k), round2 = make_float2(kRound, kRound), back2 = make_float2(-kRound, -kRound);
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const float2 c = __fmul2_rn(make_float2(x[j], x[j + 1]), k2), r = __fadd2_rn(c, round2);
    const float2 i = __fadd2_rn(r, back2), d = __ffma2_rn(i, make_float2(-1.f, -1.f), c);
    off = sm100::fmax3f(off, fabsf(d.x), fabsf(d.y));
    w[j] = __float_as_uint(r.x);
    w[j + 1] = __float_as_uint(r.y);
  }
  // Near a half, or the reciprocal leaves float32's normal range, or NaN (codes 0).
  if (!(off < 0.5f - 0x1p-14f) || !(top < 0x1p100f)) {
    // 127 x would leave float32 for its largest rows: both sides are scaled down there, which is exact where it matters.
    const float down = sizeof(T) == 2 || top < 0x1p100f ? 1.f : 0x1p-20f, t = top * down;
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = min(max(__float2int_rn(__fdiv_rn(__fmul_rn(x[j], 127.f * down), t)), -127), 127) + 128;
  }
  auto four = [&](int j) {
    return __byte_perm(__byte_perm(w[j], w[j + 1], 0x0040), __byte_perm(w[j + 2], w[j + 3], 0x0040), 0x5410);
  };
  return make_uint2(four(0), four(4));
}

// Values of four codes.
__device__ __forceinline__ void decode4(uint32_t w, float scale, float* x) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float u = __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7650u | j));  // 2^23 + code + 128
    x[j] = __fmul_rn(__fsub_rn(u, 8388608.f + 128.f), scale);
  }
}

// Eight consecutive elements of a row in float32.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int64_t stride, bool vec, float (&x)[8]) {
  if (vec) {
    if constexpr (sizeof(T) == 2) {
      const uint4 w = *reinterpret_cast<const uint4*>(p);
      const __half2* h = reinterpret_cast<const __half2*>(&w);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(h[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    } else {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(p[i * stride]);
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 2) {
    uint4 w;
    __half2* h = reinterpret_cast<__half2*>(&w);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = w;
  } else {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
  }
}

struct Str3 {
  int64_t b, h, t;
};

struct AppendParams {
  CacheView c;
  const void* src[2];  // k, v
  Str4 st[2];
  int vec[2];          // rows can be read 16 bytes at a time
  const float* phi;
  const float* psi;
  Str3 sphi, spsi;
  const int32_t* table;
  int64_t table_stride;
  int max_pages, n;
  const int32_t* start;
  const int32_t* counts;
};

// T: type of k and v; kInt8: codes and scales, else rows as they are. Four blocks on an SM, three for codes from float32, whose
// registers would spill (16 x 12 pairs of up to 2048 tokens of 64: 50 us with four, 42 with three).
template <typename T, bool kInt8>
__global__ void __launch_bounds__(kMaxThreads, kInt8 && sizeof(T) == 4 ? 3 : 4) append_kernel(const __grid_constant__ AppendParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const CacheView& c = p.c;
  const int h = blockIdx.y, b = blockIdx.z, page = 1 << c.page_shift, threads = blockDim.x;
  const int start = p.start[b];
  const int count = p.counts ? min(max(p.counts[b], 0), p.n) : p.n;
  if (count == 0) return;
  const int64_t cap = int64_t(p.max_pages) << c.page_shift;
  if (start < 0 || start >= cap) {
    if (blockIdx.x == 0 && threadIdx.x == 0) report_bad_page(c.status, kSiteAppend);
    return;
  }
  // This block's page of the sequence and the tokens [i0, i1) that fall into it.
  const int64_t pg = int64_t(start >> c.page_shift) + blockIdx.x;
  const int64_t first = pg << c.page_shift;
  const int i0 = int(max(first - start, int64_t(0))), i1 = int(min(first + page - start, int64_t(count)));
  if (i0 >= i1) return;
  const int pid = pg < p.max_pages ? p.table[b * p.table_stride + pg] : -1;
  const int slot0 = int(start + i0 - first), tokens = i1 - i0;
  // Half of the block takes K, half V: thread (sub, e0) the eight elements from e0 on of tokens sub, sub + rows, ...
  const int lanes = c.D >> 3, rows = threads / 2 / lanes;
  const int which = int(threadIdx.x) >= threads / 2 ? 1 : 0, tid = threadIdx.x - which * (threads / 2);
  const int sub = tid / lanes, e0 = (tid - sub * lanes) * 8;
  const Str4 st = p.st[which];
  const T* src = static_cast<const T*>(p.src[which]) + b * st.b + h * st.h + (i0 + sub) * st.t + e0 * st.d;
  const int64_t step = rows * st.t;
  const bool vec = p.vec[which] != 0;
  float x[kAhead][8];
  auto load_rows = [&](int t0) {
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[a][j] = 0.f;
      if (t0 + a * rows + sub < tokens) load8(src + a * step, st.d, vec, x[a]);
    }
    src += kAhead * step;
  };
  // What does not depend on the page's id travels with it.
  load_rows(0);
  const float* src_phi = p.phi + b * p.sphi.b + h * p.sphi.h;
  const float* src_psi = p.psi + b * p.spsi.b + h * p.spsi.h;
  const bool mine = int(threadIdx.x) < tokens;
  const float phi0 = mine ? src_phi[(i0 + int(threadIdx.x)) * p.sphi.t] : kInf;
  const float psi0 = mine ? src_psi[(i0 + int(threadIdx.x)) * p.spsi.t] : 0.f;
  if (unsigned(pid) >= unsigned(c.n_pages)) {
    if (threadIdx.x == 0) report_bad_page(c.status, kSiteAppend);
    return;
  }
  const int64_t base = (int64_t(pid) * c.H + h) << c.page_shift;  // pool index of the page's slot 0
  // The field, and the page's minimum over the slots up to the last one written.
  float* phi = const_cast<float*>(c.phi) + base;
  float* psi = const_cast<float*>(c.psi) + base + slot0;
  float low = phi0;
  if (mine) {
    phi[slot0 + threadIdx.x] = phi0;
    psi[threadIdx.x] = psi0;
  }
  for (int i = threadIdx.x + threads; i < tokens; i += threads) {
    const float f = src_phi[(i0 + i) * p.sphi.t];
    phi[slot0 + i] = f;
    psi[i] = src_psi[(i0 + i) * p.spsi.t];
    low = fminf(low, f);
  }
  for (int s = threadIdx.x; s < slot0; s += threads) low = fminf(low, phi[s]);
  // Whole warps stay in the loop for the shuffles.
  char* dst = const_cast<char*>(static_cast<const char*>(which ? c.v : c.k)) +
              ((base + slot0 + sub) * c.D + e0) * int(kInt8 ? 1 : sizeof(T));
  float* scales = const_cast<float*>(which ? c.vs : c.ks) + base + slot0 + sub;
  const int dst_step = rows * c.D * int(kInt8 ? 1 : sizeof(T));
  for (int t0 = 0; t0 < tokens; t0 += kAhead * rows) {
    if (t0 > 0) load_rows(t0);
    float top[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      if (t0 + a * rows >= tokens) break;
      const bool ok = t0 + a * rows + sub < tokens;
      if constexpr (kInt8) {
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmax_nan(m, fabsf(x[a][j]));
#pragma unroll
        for (int o = 1; o < 32; o <<= 1)
          if (o < lanes) m = fmax_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
        // Scales stay at or above 2^-90, so that their inverses sum up in float32 (see fpa_decode_mma.cu); a row of
        // zeros takes that smallest scale, so that it does not outweigh small rows there. A row with a NaN or an infinity
        // has no codes: its scale is NaN.
        top[a] = m < kInf ? fmaxf(m, 127.f * 0x1p-90f) : __int_as_float(0x7fffffff);
        const uint2 w = encode8<T>(x[a], top[a]);
        if (ok) *reinterpret_cast<uint2*>(dst + a * dst_step) = w;
      } else if (ok) {
        store8(reinterpret_cast<T*>(dst + a * dst_step), x[a]);
      }
    }
    if constexpr (kInt8) {
      // Lane j of a row's lanes divides for the j-th row (and the rows `lanes` after it).
      for (int a0 = 0; a0 < kAhead; a0 += lanes) {
        const int a = a0 + (e0 >> 3);
        float t = top[0];
#pragma unroll
        for (int j = 1; j < kAhead; ++j)
          if (a == j) t = top[j];
        if (a < kAhead && t0 + a * rows + sub < tokens) scales[a * rows] = __fdiv_rn(t, 127.f);
      }
    }
    dst += kAhead * dst_step;
    scales += kAhead * rows;
  }
  __shared__ float warp_low[kMaxThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
  if ((threadIdx.x & 31) == 0) warp_low[threadIdx.x >> 5] = low;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < threads / 32; ++w) low = fminf(low, warp_low[w]);
    const_cast<float*>(c.pmin)[int64_t(pid) * c.H + h] = low;
  }
}

struct ReadParams {
  CacheView c;
  const int32_t* table;
  int64_t table_stride;
  int max_pages, n;
  const int32_t* start;
  const int32_t* lengths;
  void* k;
  void* v;
  float* phi;
  float* psi;
};

// A block reads a run of kReadRows tokens of one (sequence, head).
constexpr int kReadRows = 64;

template <typename T, bool kInt8>
__global__ void __launch_bounds__(kReadThreads) read_kernel(const __grid_constant__ ReadParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const CacheView& c = p.c;
  const int h = blockIdx.y, b = blockIdx.z, page = 1 << c.page_shift;
  const int i0 = blockIdx.x * kReadRows, i1 = min(i0 + kReadRows, p.n);
  const int64_t start = p.start ? p.start[b] : 0;
  const int64_t cap = int64_t(p.max_pages) << c.page_shift;
  const int64_t len = p.lengths ? min(int64_t(p.lengths[b]), cap) : cap;
  if (threadIdx.x == 0 && blockIdx.x == 0 && (start < 0 || (p.lengths && p.lengths[b] > cap)))
    report_bad_page(c.status, kSiteRead);
  const int64_t out0 = (int64_t(b) * c.H + h) * p.n;
  // Pool index of token i, or -1.
  auto slot = [&](int i) -> int64_t {
    const int64_t s = start + i;
    if (s < 0 || s >= len) return -1;
    const int pid = p.table[b * p.table_stride + (s >> c.page_shift)];
    if (unsigned(pid) >= unsigned(c.n_pages)) {
      report_bad_page(c.status, kSiteRead);
      return -1;
    }
    return ((int64_t(pid) * c.H + h) << c.page_shift) + (s & (page - 1));
  };
  const int lanes = c.D >> 3, rows = kReadThreads / lanes;
  const int sub = threadIdx.x / lanes, e0 = (threadIdx.x - sub * lanes) * 8;
  for (int first = i0 + sub; first < i1; first += kAhead * rows) {
    int64_t at[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) at[a] = first + a * rows < i1 ? slot(first + a * rows) : -1;
    const int64_t to = (out0 + first) * c.D + e0;
    if constexpr (kInt8) {
      uint2 w[2][kAhead];
      float scale[2][kAhead];
#pragma unroll
      for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
          w[which][a] = make_uint2(0x80808080u, 0x80808080u);  // code 0
          scale[which][a] = 0.f;
          if (at[a] >= 0) {
            w[which][a] = __ldcs(reinterpret_cast<const uint2*>(static_cast<const char*>(which ? c.v : c.k) + at[a] * c.D + e0));
            scale[which][a] = (which ? c.vs : c.ks)[at[a]];
          }
        }
#pragma unroll
      for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
          float x[8];
          decode4(w[which][a].x, scale[which][a], x);
          decode4(w[which][a].y, scale[which][a], x + 4);
          if (first + a * rows < i1) store8(static_cast<T*>(which ? p.v : p.k) + to + int64_t(a) * rows * c.D, x);
        }
    } else {
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        float x[kAhead][8];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
#pragma unroll
          for (int j = 0; j < 8; ++j) x[a][j] = 0.f;
          if (at[a] >= 0) load8(static_cast<const T*>(which ? c.v : c.k) + at[a] * c.D + e0, 1, true, x[a]);
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
          if (first + a * rows < i1) store8(static_cast<T*>(which ? p.v : p.k) + to + int64_t(a) * rows * c.D, x[a]);
      }
    }
  }
  for (int i = i0 + threadIdx.x; i < i1; i += kReadThreads) {
    const int64_t at = slot(i);
    p.phi[out0 + i] = at >= 0 ? c.phi[at] : 0.f;
    p.psi[out0 + i] = at >= 0 ? c.psi[at] : 0.f;
  }
}

int invalid(const char* msg) {
  set_last_error(msg);
  return FPA_ERR_INVALID_ARGUMENT;
}

int unsupported(const char* msg) {
  set_last_error(msg);
  return FPA_ERR_UNSUPPORTED;
}

int cuda_result(cudaError_t e, const char* where) {
  if (e == cudaSuccess) return FPA_OK;
  set_last_error(std::string(where) + ": " + cudaGetErrorString(e));
  return FPA_ERR_CUDA;
}

// 16-byte reads of rows of eight elements: unit innermost stride, and everything else a multiple of 16 bytes.
bool rows_aligned(const void* p, const int64_t st[4], int elem) {
  if (reinterpret_cast<uintptr_t>(p) % 16 || st[3] != 1) return false;
  for (int i = 0; i < 3; ++i)
    if (st[i] * elem % 16) return false;
  return true;
}

}  // namespace

int check_cache(const FpaCache* c) {
  if (c == nullptr) return invalid("null cache");
  const bool f16 = c->dtype == FPA_DTYPE_F16;
  if (!f16 && c->dtype != FPA_DTYPE_F32) return invalid("the cache's dtype must be fp16 or fp32");
  if (c->storage != FPA_STORE_I8 && c->storage != (f16 ? FPA_STORE_F16 : FPA_STORE_F32))
    return invalid("the cache's storage must be its dtype or int8");
  if (c->n_pages <= 0 || c->H <= 0) return invalid("the cache needs at least one page and one head");
  if (c->H > 65535) return unsupported("H above 65535 is not supported");
  if (c->page_size != 32 && c->page_size != 64 && c->page_size != 128 && c->page_size != 256)
    return invalid("the page size must be 32, 64, 128 or 256");
  if (c->D != 16 && c->D != 32 && c->D != 64 && c->D != 128 && c->D != 256)
    return invalid("the head dimension must be 16, 32, 64, 128 or 256");
  if (!c->k || !c->v || !c->phi || !c->psi || !c->phi_min || !c->status) return invalid("null cache pointer");
  if (c->storage == FPA_STORE_I8 && (!c->k_scale || !c->v_scale)) return invalid("null cache scale pointer");
  const void* arrays[] = {c->k, c->v, c->phi, c->psi, c->storage == FPA_STORE_I8 ? c->k_scale : nullptr,
                          c->storage == FPA_STORE_I8 ? c->v_scale : nullptr};
  for (const void* a : arrays)
    if (reinterpret_cast<uintptr_t>(a) % 16) return invalid("the cache's arrays must be 16-byte aligned");
  return FPA_OK;
}

}  // namespace fpa

using namespace fpa;

extern "C" FPA_API int fpa_cache_append(const FpaAppendArgs* a, void* stream) {
  if (a == nullptr) return invalid("null argument block");
  if (const int rc = check_cache(a->cache)) return rc;
  if (a->B <= 0 || a->n <= 0) return invalid("fpa_cache_append: B and n must be positive");
  if (a->max_pages <= 0) return invalid("fpa_cache_append: the block table must have at least one column");
  if (!a->k || !a->v || !a->phi || !a->psi || !a->table || !a->start) return invalid("fpa_cache_append: null tensor pointer");
  if (a->B > 65535) return unsupported("fpa_cache_append: B above 65535 is not supported");
  const FpaCache& c = *a->cache;
  const int elem = c.dtype == FPA_DTYPE_F16 ? 2 : 4;
  AppendParams p;
  p.c = cache_view(c);
  p.src[0] = a->k;
  p.src[1] = a->v;
  p.st[0] = str4(a->k_stride);
  p.st[1] = str4(a->v_stride);
  p.vec[0] = rows_aligned(a->k, a->k_stride, elem);
  p.vec[1] = rows_aligned(a->v, a->v_stride, elem);
  p.phi = a->phi;
  p.psi = a->psi;
  p.sphi = Str3{a->phi_stride[0], a->phi_stride[1], a->phi_stride[2]};
  p.spsi = Str3{a->psi_stride[0], a->psi_stride[1], a->psi_stride[2]};
  p.table = a->table;
  p.table_stride = a->table_stride;
  p.max_pages = a->max_pages;
  p.n = a->n;
  p.start = a->start;
  p.counts = a->counts;
  // n tokens touch at most this many pages, wherever they start.
  const dim3 grid(unsigned((int64_t(a->n) + 2 * c.page_size - 2) / c.page_size), c.H, a->B);
  // 256 threads for a page's worth of tokens, 128 for a few: 32 x 12 (sequence, head) pairs of one token take 3.5 us with
  // 128, 4.6 with 256; 16 x 12 of 64 tokens 7.7 and 6.8.
  const bool i8 = c.storage == FPA_STORE_I8;
  auto kernel = c.dtype == FPA_DTYPE_F16 ? (i8 ? append_kernel<__half, true> : append_kernel<__half, false>)
                                         : (i8 ? append_kernel<float, true> : append_kernel<float, false>);
  return cuda_result(launch_pdl(kernel, grid, dim3(a->n > 16 ? kMaxThreads : 128), 0, static_cast<cudaStream_t>(stream), p),
                     "fpa_cache_append");
}

extern "C" FPA_API int fpa_cache_read(const FpaReadArgs* a, void* stream) {
  if (a == nullptr) return invalid("null argument block");
  if (const int rc = check_cache(a->cache)) return rc;
  if (a->B <= 0 || a->n <= 0) return invalid("fpa_cache_read: B and n must be positive");
  if (a->max_pages <= 0) return invalid("fpa_cache_read: the block table must have at least one column");
  if (!a->k || !a->v || !a->phi || !a->psi || !a->table) return invalid("fpa_cache_read: null tensor pointer");
  if (a->B > 65535) return unsupported("fpa_cache_read: B above 65535 is not supported");
  if (reinterpret_cast<uintptr_t>(a->k) % 16 || reinterpret_cast<uintptr_t>(a->v) % 16)
    return invalid("fpa_cache_read: k and v must be 16-byte aligned");
  const FpaCache& c = *a->cache;
  ReadParams p{cache_view(c), a->table, a->table_stride, a->max_pages, a->n, a->start, a->lengths, a->k, a->v, a->phi, a->psi};
  const dim3 grid((unsigned(a->n) + kReadRows - 1) / kReadRows, c.H, a->B);
  const bool i8 = c.storage == FPA_STORE_I8;
  auto kernel = c.dtype == FPA_DTYPE_F16 ? (i8 ? read_kernel<__half, true> : read_kernel<__half, false>)
                                         : (i8 ? read_kernel<float, true> : read_kernel<float, false>);
  return cuda_result(launch_pdl(kernel, grid, dim3(kReadThreads), 0, static_cast<cudaStream_t>(stream), p), "fpa_cache_read");
}
