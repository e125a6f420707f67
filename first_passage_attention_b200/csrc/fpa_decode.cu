// fpa_decode: argument checks, the split rules and the launches (fpa_decode.cuh has the mathematics).
#include "fpa_serve.h"

namespace fpa {

int check_cache(const FpaCache* c);  // fpa_cache.cu

namespace {

int invalid(const char* msg) {
  set_last_error(msg);
  return FPA_ERR_INVALID_ARGUMENT;
}

// The prefix pass runs on tcgen05 for fp16 queries with D = 64 and more than 16 rows in the batch, or D = 128 and more
// than 8; fewer fit one pass of the mma.sync kernel over the prefix. A whole call behind 8192 tokens, 12 heads, us with
// mma.sync / tcgen05: int8 D = 64, 8 rows 13.5 / 17.3, 16 rows 16.5 / 17.6, 17 rows 22.8 / 17.8, 64 rows 30.8 / 21.2; fp16 D =
// 128, 4 rows 16.1 / 17.5, 8 rows 18.2 / 17.9, 12 rows 26.9 / 18.2, 64 rows 58.5 / 27.7.
bool prefix_on_tc(const FpaCache& c, int64_t rows) {
  return c.dtype == FPA_DTYPE_F16 && ((c.D == 64 && rows > 16) || (c.D == 128 && rows > 8));
}

// Parts of the prefix (CTAs that share a row group's or row tile's prefix). tcgen05: one CTA on every SM, two 128-key
// tiles each at least. Otherwise about four CTAs for an SM, two 32-key blocks for each of their four warps at least.
int prefix_chunks(const FpaCache& c, int B, int n, int prefix_len) {
  const int64_t R = int64_t(B) * n;
  const bool tc = prefix_on_tc(c, R);
  const int64_t most = (int64_t(prefix_len) + 255) / 256;
  const int64_t units = (tc ? prefix_tc_row_tiles(R) : (R + 15) / 16) * c.H;
  const int64_t want = tc ? sm_count() / units : (4 * sm_count() + units - 1) / units;
  return int(want < 1 ? 1 : want > most ? most : want);
}

size_t workspace_bytes(const FpaCache& c, int B, int n, int prefix_len, size_t* ml, size_t* o) {
  if (prefix_len <= 0) return 0;
  const size_t rows = size_t(c.H) * B * n, chunks = prefix_chunks(c, B, n, prefix_len);
  *ml = align256(rows * 4);
  *o = *ml + align256(rows * chunks * 8);
  return *o + align256(rows * chunks * c.D * 4);
}

}  // namespace
}  // namespace fpa

using namespace fpa;

extern "C" FPA_API size_t fpa_decode_workspace_bytes(const FpaCache* cache, int B, int n, int prefix_len) {
  if (check_cache(cache) || B <= 0 || n <= 0 || n > kMaxNew || prefix_len > kMaxPositions) return 0;
  size_t ml, o;
  return workspace_bytes(*cache, B, n, prefix_len, &ml, &o);
}

extern "C" FPA_API int fpa_decode(FpaDecodeArgs* a, void* stream) {
  if (a == nullptr) return invalid("null argument block");
  a->kernels_launched = 0;
  if (const int rc = check_cache(a->cache)) return rc;
  const FpaCache& c = *a->cache;
  if (a->B <= 0) return invalid("fpa_decode: B must be positive");
  if (a->n < 1 || a->n > kMaxNew) return invalid("fpa_decode: between 1 and 16 new tokens per call");
  if (a->max_pages <= 0) return invalid("fpa_decode: the block table must have at least one column");
  if (!a->q || !a->o || !a->beta || !a->table || !a->lengths) return invalid("fpa_decode: null tensor pointer");
  if (a->prefix_len < 0 || (a->prefix_len > 0 && (!a->prefix_table || int64_t(a->prefix_pages) * c.page_size < a->prefix_len)))
    return invalid("fpa_decode: the prefix is longer than the pages of its table");
  if (a->prefix_len > kMaxPositions) {
    set_last_error("fpa_decode: prefixes above 2147483392 tokens are not supported");
    return FPA_ERR_UNSUPPORTED;
  }
  // The grids' y and z extents stay below 65536: B, and the row groups of all heads, or of the batch behind a prefix. fp16
  // queries go in groups of at least eight rows.
  auto groups = [&](int64_t rows) {
    const int group = c.dtype == FPA_DTYPE_F16 ? 8 : ffma_group(c.D, rows);
    return (rows + group - 1) / group;
  };
  if (a->B > 65535 || c.H > 32767 || c.H * groups(a->n) > 65535 || (a->prefix_len > 0 && groups(int64_t(a->B) * a->n) > 65535)) {
    set_last_error("fpa_decode: B above 65535, H above 32767 (16383 for float32 with D above 64 and n above 12) or, with a "
                   "prefix, B * n above 524280 (262140 for float32 with D above 64) is not supported");
    return FPA_ERR_UNSUPPORTED;
  }
  DecodeParams p{};
  p.c = cache_view(c);
  p.q = a->q;
  p.sq = str4(a->q_stride);
  p.o = a->o;
  p.so = str4(a->o_stride);
  p.beta = a->beta;
  p.table = a->table;
  p.table_stride = a->table_stride;
  p.max_pages = a->max_pages;
  p.lengths = a->lengths;
  p.prefix_table = a->prefix_table;
  p.prefix_pages = a->prefix_pages;
  p.prefix_len = a->prefix_len;
  p.B = a->B;
  p.n = a->n;
  p.q_pairs = reinterpret_cast<uintptr_t>(a->q) % 4 == 0 && p.sq.d == 1 && p.sq.b % 2 == 0 && p.sq.h % 2 == 0 && p.sq.t % 2 == 0;
  p.scale2 = kLog2e / sqrtf(float(c.D));
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool i8 = c.storage == FPA_STORE_I8, f16 = c.dtype == FPA_DTYPE_F16;
  auto run = f16 ? launch_decode_mma : launch_decode_ffma;
  cudaError_t e;
  int launches = 0;
  if (p.prefix_len > 0) {
    size_t ml, o;
    const size_t need = workspace_bytes(c, p.B, p.n, p.prefix_len, &ml, &o);
    if (a->workspace == nullptr || reinterpret_cast<uintptr_t>(a->workspace) % 256 || a->workspace_bytes < need) {
      set_last_error("fpa_decode: the workspace must be 256-byte aligned and as large as fpa_decode_workspace_bytes says");
      return FPA_ERR_WORKSPACE;
    }
    char* ws = static_cast<char*>(a->workspace);
    p.row_min = reinterpret_cast<float*>(ws);
    p.part_ml = reinterpret_cast<float*>(ws + ml);
    p.part_o = reinterpret_cast<float*>(ws + o);
    p.chunks = prefix_chunks(c, p.B, p.n, p.prefix_len);
    prof_mark(s, "decode_row_min");
    e = launch_row_min(p, s);
    if (e == cudaSuccess) {
      prof_mark(s, "decode_prefix");
      e = prefix_on_tc(c, int64_t(p.B) * p.n) ? launch_prefix_tc(p, i8, s) : run(p, i8, true, s, launches);
    }
    if (e != cudaSuccess) {
      set_last_error(std::string("fpa_decode, prefix: ") + cudaGetErrorString(e));
      return FPA_ERR_CUDA;
    }
    a->kernels_launched = 2;
    launches = 0;
  }
  prof_mark(s, "decode");
  e = run(p, i8, false, s, launches);
  prof_mark(s, nullptr);
  if (e != cudaSuccess) {
    set_last_error(std::string("fpa_decode: ") + cudaGetErrorString(e));
    return FPA_ERR_CUDA;
  }
  a->kernels_launched += launches;
  return FPA_OK;
}
