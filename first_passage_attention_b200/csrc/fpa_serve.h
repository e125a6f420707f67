// Shared by the serving kernels (cache append / read, decode, verification): device views and host-side launchers.
#pragma once

#include "fpa_internal.h"

namespace fpa {

constexpr int kMaxNew = 16;  // newest tokens of one decode call
// Positions of a sequence, or of a prefix, that decode takes: rounding one up to a page or a tile stays within 32 bits.
constexpr int kMaxPositions = INT32_MAX - 255;

// Sites that the cache's status word names next to FPA_ERR_INVALID_ARGUMENT.
enum ServeSite { kSiteAppend = 1, kSiteRead = 2, kSiteDecode = 3 };

struct CacheView {
  const void* k;
  const void* v;
  const float* ks;
  const float* vs;
  const float* phi;
  const float* psi;
  const float* pmin;
  int* status;
  int n_pages, H, page_shift, D;
};

inline int log2_int(int x) {
  int n = 0;
  while ((1 << n) < x) ++n;
  return n;
}

inline CacheView cache_view(const FpaCache& c) {
  return CacheView{c.k, c.v, c.k_scale, c.v_scale, c.phi, c.psi, c.phi_min, c.status, c.n_pages, c.H,
                   log2_int(c.page_size), c.D};
}

__device__ __forceinline__ void report_bad_page(int* status, int site) {
  if (status) atomicCAS(status, 0, (FPA_ERR_INVALID_ARGUMENT << 16) | site);
}

struct DecodeParams {
  CacheView c;
  const void* q;
  Str4 sq;
  void* o;
  Str4 so;
  const float* beta;
  const int32_t* table;
  int64_t table_stride;
  int max_pages;
  const int32_t* lengths;
  const int32_t* prefix_table;
  int prefix_pages, prefix_len;
  int B, n;
  int groups;      // row groups of a (sequence, head) (decode) or of a head (prefix pass)
  int q_pairs;     // q can be read two elements at a time
  float scale2;    // log2(e) / sqrt(D)
  // Prefix: rows are (b, i) in b-major order, R = B * n of them for each head.
  float* row_min;  // [H][R]  minimum of phi over the row's own tokens up to itself
  float* part_ml;  // [H][R][chunks][2]  softmax maximum and sum of each chunk of the prefix
  float* part_o;   // [H][R][chunks][D]  unnormalised output of each chunk
  int chunks;
  // The batch in two launches: the sequences from `first` on; another launch follows; another one went before.
  int first;
  bool followed, follows;
};

// Rows are handled by one CTA in groups of 8 or 16 (tensor cores) or 1, 4 or 8 (FFMA). For FFMA, 8 for D <= 64 and more than 4
// rows. Measured on 8 x 8 (sequence, head) pairs of 4096 tokens, us for groups of 1 / 4 / 8: 8 rows, D = 32 int8 84 / 41 / 38,
// D = 64 147 / 88 / 87, D = 128 246 / 134 / 135; 2000 tokens at D = 256 200 / 100 / 127 (the registers of 8 rows leave fewer
// CTAs); 2 rows, D = 32 29 / 25 / 37.
inline int ffma_group(int D, int64_t rows) { return rows == 1 ? 1 : rows < 5 || D > 64 ? 4 : 8; }
cudaError_t launch_decode_mma(const DecodeParams& p, bool int8, bool prefix, cudaStream_t s, int& launches);
cudaError_t launch_decode_ffma(const DecodeParams& p, bool int8, bool prefix, cudaStream_t s, int& launches);
// The prefix on tcgen05: fp16 queries, D = 64 or 128. p.chunks: CTAs that share a row tile's prefix.
int prefix_tc_row_tiles(int64_t rows);
cudaError_t launch_prefix_tc(const DecodeParams& p, bool int8, cudaStream_t s);
cudaError_t launch_row_min(const DecodeParams& p, cudaStream_t s);

int sm_count();  // fpa_tma.cu

}  // namespace fpa
